"""A bounded wait of the paged attention that gives up: rows of NaN, an error at an engine's commit, and a context that goes
on.  The limit is set to no polls at all, so that every wait ends at once and nothing is in flight."""
import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu

from test_fork_gpu import prefill  # noqa: E402
from test_kv_cache_gpu import check, make  # noqa: E402
from test_llama_gpu import make_engine, rel, small_geo  # noqa: E402


@pytest.fixture
def limit(ctx):
    from clusterlm_b200 import kv_cache

    yield lambda polls: kv_cache.set_wait_limit(ctx, polls)
    kv_cache.set_wait_limit(ctx)


@pytest.mark.parametrize("n,positions,nh,nkv,hd,pos,shared", [
    (3, 5, 8, 2, 128, [70, 300, 128], None),                # 20 rows a kv head: the tile kernel alone, alternate pages
    (2, 100, 4, 1, 64, [40, 200], None),                    # row tiles of both streams
    (8, 2, 4, 2, 128, [200 + 9 * i for i in range(8)], [(8, 3)]),  # shared pages in the tile kernel, own ones not
])
def test_rows_become_nan_and_the_next_call_is_right(ctx, limit, n, positions, nh, nkv, hd, pos, shared):
    from clusterlm_b200 import kv_cache as kv

    args = make(n, positions, nh, nkv, hd, pos, torch.float16, shared=shared)
    limit(0)
    out = kv.kv_attention(ctx, *args, groups=shared)
    torch.cuda.synchronize()
    assert out.isnan().all()
    limit(2**20)
    check(kv.kv_attention(ctx, *args, groups=shared), *ref.attention(*args))


def test_rows_that_wait_for_nothing_are_right(ctx, limit):
    """Up to 16 rows a kv head without a group take no wait."""
    from clusterlm_b200 import kv_cache as kv

    args = make(3, 2, 8, 2, 128, [70, 300, 128], torch.float16)
    limit(0)
    check(kv.kv_attention(ctx, *args), *ref.attention(*args))


def test_the_commit_of_a_batched_window_of_forks_fails(ctx, limit):
    from clusterlm_b200 import ClmError

    geo = small_geo("q8_0", n_heads=8, n_kv_heads=2, hidden=1024)
    e = make_engine(ctx, geo, max_context=512, max_window=96, sessions=4)
    rng = np.random.default_rng(4)
    e.open_session(1)
    prefill(e, 1, rng.integers(0, geo.vocab, 200).astype(np.int32))
    order = [1, 2, 3, 4]
    for s in order[1:]:
        e.fork_session(1, s)
    toks = rng.integers(0, geo.vocab, (4, 8)).astype(np.int32)
    limit(0)
    assert np.isnan(e.run_batch_window(order, [200] * 4, toks)).any()
    with pytest.raises(ClmError) as err:
        e.commit(1, 8)
    assert err.value.name == "kDeadlineExceeded"
    for s in order[1:]:
        e.abort(s)
    limit(2**20)
    assert [e.position(s) for s in order] == [200] * 4
    for _ in range(3):  # captured with the limit in force now, and replayed
        got = e.run_batch_window(order, [200] * 4, toks)
        for s in order:
            e.abort(s)
        for i, s in enumerate(order):
            alone = e.run_window(s, 200, tokens=toks[i])
            assert rel(got[i], alone) < 2e-2
            e.abort(s)
    for s in order:
        e.run_window(s, 200, tokens=toks[0])
        e.commit(s, 8)
    e.close()
