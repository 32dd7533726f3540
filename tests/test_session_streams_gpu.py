"""Sessions that are closed or forked while work of theirs is queued on a caller's stream."""
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


def test_fork_waits_for_rounds_on_another_stream(ctx):
    """The child continues after the rounds that were queued for its parent when it was forked."""
    import torch

    geo = small_geo("q4_k")
    prompt = np.random.default_rng(6).integers(0, geo.vocab, 60).astype(np.int32)  # the rounds pass a page's end
    side = torch.cuda.Stream()

    def rounds(e, s):
        return [int(t) for _ in range(6) for t in e.spec_round(s, 4, temperature=1.0, seed=3)]

    for turn in range(3):
        e = make_engine(ctx, geo, max_context=256, max_window=16, sessions=3)
        ref = make_engine(ctx, geo, max_context=256, max_window=16, sessions=1)
        for x in (e, ref):
            x.open_session(1)
            x.spec_begin(1, prompt, 4, temperature=1.0, seed=3)
            for _ in range(turn):
                x.spec_round(1, 4, temperature=1.0, seed=3)
        for _ in range(12):
            ref.spec_round(1, 4, temperature=1.0, seed=3)
        kept = queue(e, 1, side, "rounds", 0, geo.vocab)
        e.fork_session(1, 2)
        assert side.query()
        assert e.position(2) == ref.position(1) and e.position(1) == ref.position(1)
        want = rounds(ref, 1)
        assert rounds(e, 2) == want and rounds(e, 1) == want
        e.fork_session(1, 3)  # nothing queued since: the position is the parent's now
        assert e.position(3) == ref.position(1)
        del kept
        e.close()
        ref.close()
