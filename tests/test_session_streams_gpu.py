"""Sessions that are closed while work of theirs is queued on a caller's stream."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from test_fork_gpu import prefill  # noqa: E402
from test_llama_gpu import make_engine, small_geo  # noqa: E402

BUSY = 200_000_000  # clocks of a delay in front of the queued work: about a tenth of a second


def queue(e, session, side, kind, base, vocab):
    """Windows or rounds of the session on `side`, behind a delay: none has begun when this returns."""
    import torch

    toks = torch.arange(8, dtype=torch.int32, device="cuda") * 7 % vocab
    out = torch.empty(8, vocab, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(BUSY)
    for _ in range(12):
        if kind == "rounds":
            e.spec_round_device(session, 4, temperature=1.0, seed=3, stream=side.cuda_stream)
        else:
            e.run_window_device(session, base, d_tokens=toks, d_out=out, stream=side.cuda_stream)
            e.abort(session)
    return toks, out


@pytest.mark.parametrize("kind", ["windows", "rounds"])
def test_close_waits_for_work_on_another_stream(ctx, kind):
    """The next session takes the closed one's place and pages: nothing queued for the closed one may write there."""
    import torch

    geo = small_geo("q4_k")
    rng = np.random.default_rng(5)
    first, second = (rng.integers(0, geo.vocab, 70).astype(np.int32) for _ in range(2))
    window = rng.integers(0, geo.vocab, 8).astype(np.int32)
    ref = make_engine(ctx, geo, max_context=256, max_window=16, sessions=1)
    ref.open_session(1)
    prefill(ref, 1, second, 16)
    want = ref.run_window(1, len(second), tokens=window)
    ref.close()
    e = make_engine(ctx, geo, max_context=256, max_window=16, sessions=1)
    side = torch.cuda.Stream()
    for turn in range(3):  # the queued work eager and captured, captured and replayed
        e.open_session(turn)
        if kind == "rounds":
            e.spec_begin(turn, first, 4, temperature=1.0, seed=3)
        else:
            prefill(e, turn, first, 16)
        kept = queue(e, turn, side, kind, len(first), geo.vocab)
        e.close_session(turn)
        assert side.query()
        e.open_session(100 + turn)
        prefill(e, 100 + turn, second, 16)
        np.testing.assert_array_equal(e.run_window(100 + turn, len(second), tokens=window), want)
        assert e.position(100 + turn) == len(second)
        e.close_session(100 + turn)
        del kept
    e.close()
