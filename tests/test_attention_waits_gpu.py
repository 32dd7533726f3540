"""A bounded wait of the paged attention that gives up: rows of NaN, and a context that goes on.  The limit is set to no polls at all, so that every wait ends at once and nothing is in flight."""
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu

from test_kv_cache_gpu import check, make  # noqa: E402


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
