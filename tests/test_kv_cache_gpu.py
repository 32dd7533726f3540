"""The paged-cache operators on the GPU against their 64-bit forms (tests/kv_reference.py)."""
import math

import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAGE = 64


@pytest.fixture(scope="module")
def kv():
    from clusterlm_b200 import kv_cache

    return kv_cache


def make(n, positions, nh, nkv, hd, pos, dtype, seed=0, spare=2, shared=None):
    """Pools of random values, tables over shuffled pages (shared: list of (sequences, pages)), positions."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    need = [max(0, (p + positions - 1) // PAGE + 1) if p >= 0 else 0 for p in pos]
    width = max(need + [1]) + 1
    lead = np.zeros(n, int)
    tables = np.full((n, width), -1, np.int32)
    ids = iter(rng.permutation(sum(need) + spare + 1))
    at = 0
    for count, pages in shared or []:
        common = [next(ids) for _ in range(pages)]
        for b in range(at, at + count):
            tables[b, :pages] = common
            lead[b] = pages
        at += count
    for b in range(n):
        for j in range(lead[b], need[b]):
            tables[b, j] = next(ids)
    pages = int(tables.max()) + 1 + spare
    k = torch.randn(pages, nkv, PAGE, hd, device="cuda", generator=g).to(dtype)
    v = torch.randn(pages, nkv, hd, PAGE, device="cuda", generator=g).to(dtype)
    q = (1.5 * torch.randn(n, positions, nh, hd, device="cuda", generator=g)).to(dtype)
    return k, v, torch.from_numpy(tables).cuda(), torch.tensor(pos, dtype=torch.int64, device="cuda"), q


def tree(rng, p):
    return torch.tensor([-1] + [int(rng.integers(max(-1, i - 4), i)) for i in range(1, p)], dtype=torch.int32).cuda()


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("n,positions,nh,nkv,hd,rot,inter,src,dst,pos,tr", [
    (1, 1, 4, 4, 64, 64, True, F16, F16, [0], False),
    (3, 1, 8, 2, 128, 128, False, BF16, BF16, [63, 64, 1000], False),
    (2, 4, 6, 2, 128, 64, True, F32, F16, [61, 127], False),        # rows cross a page's end
    (2, 64, 7, 1, 64, 32, False, F32, BF16, [0, 3], False),         # whole pages, and the same shifted
    (1, 300, 2, 2, 128, 24, False, F16, F16, [37], False),          # halves of 12: partners not in vectors of 8
    (1, 129, 3, 3, 64, 20, True, F16, BF16, [64], False),
    (4, 9, 4, 2, 128, 128, True, F32, F32, [5, -1, 60, 2_000_000], True),  # a tree; an idle row; a far position
    (2, 16, 2, 1, 64, 0, True, BF16, F16, [7, 8], False),           # nothing rotated
])
def test_append_follows_the_formulas(ctx, kv, n, positions, nh, nkv, hd, rot, inter, src, dst, pos, tr):
    dst = F16 if dst is F32 else dst
    if max(pos) > 10_000:  # a far position needs a table that reaches it: its early entries name no page
        k, v, tables, p, _ = make(n, positions, nh, nkv, hd, [x if x < 10_000 else 70 for x in pos], dst)
        wide = torch.full((n, 2_000_000 // PAGE + 2), -1, dtype=torch.int32, device="cuda")
        wide[:, : tables.shape[1]] = tables
        wide[-1, :] = -1
        wide[-1, 2_000_000 // PAGE:] = k.shape[0] - 1
        tables, p = wide, torch.tensor(pos, dtype=torch.int64, device="cuda")
    else:
        k, v, tables, p, _ = make(n, positions, nh, nkv, hd, pos, dst)
    rng = np.random.default_rng(1)
    qkv = torch.randn(n, positions, nh + 2 * nkv, hd, device="cuda").to(src)
    q, kn, vn = qkv[:, :, :nh], qkv[:, :, nh:nh + nkv], qkv[:, :, nh + nkv:]
    parents = tree(rng, positions) if tr else None
    freqs = torch.from_numpy(kv.rope_frequencies(rot, 10000.0)[0]).cuda() if rot else None
    rope = kv.Rope(freqs, interleaved=inter, scale=1.25) if rot else None
    K, V = k.clone(), v.clone()
    got = kv.kv_append(ctx, K, V, tables, p, q, kn, vn, rope=rope, parents=parents)
    Q, wk, wv = ref.append(k, v, tables.cpu(), p.cpu(), q, kn, vn, freqs, inter, 1.25, parents)
    half = torch.finfo(dst).eps / 2
    # the products' f32 roundings, the sine's and cosine's (2 ulp) and the reduced angle's (2^-24 of pi) on a pair
    pair = 1.25 * 2.0**-20 * 2 * float(qkv.float().abs().max())
    for a, b in ((got, Q), (K, wk)):
        assert bool(((a.double() - b).abs() <= half * b.abs() * 1.01 + pair + 2.0**-25).all())
    assert bool(((V.double() - wv).abs() <= half * wv.abs() + 2.0**-25).all())
    # what no row writes keeps its bits
    same_k, same_v = wk == k.double(), wv == v.double()
    assert bool((K[same_k] == k[same_k]).all()) and bool((V[same_v] == v[same_v]).all())
    changed = (V != v).sum()
    assert changed <= sum(positions for x in pos if x >= 0) * nkv * hd


def test_append_takes_unaligned_and_strided_rows(ctx, kv):
    k, v, tables, pos, _ = make(2, 5, 4, 2, 64, [3, 62], F16)
    freqs = torch.from_numpy(kv.rope_frequencies(64, 10000.0)[0]).cuda()
    rope = kv.Rope(freqs, interleaved=False)
    wide = torch.randn(2 * 5 * 521 + 1, device="cuda", dtype=F16)[1:].view(2, 5, 521)  # rows 521 apart, from an odd element
    q, kn, vn = (wide[:, :, a:b].unflatten(2, (-1, 64)) for a, b in ((1, 257), (257, 385), (385, 513)))
    K, V, K2, V2 = k.clone(), v.clone(), k.clone(), v.clone()
    got = kv.kv_append(ctx, K, V, tables, pos, q, kn, vn, rope=rope)
    want = kv.kv_append(ctx, K2, V2, tables, pos, q.contiguous(), kn.contiguous(), vn.contiguous(), rope=rope)
    assert torch.equal(got, want) and torch.equal(K, K2) and torch.equal(V, V2)
    # without queries only the cache is written
    K3, V3 = k.clone(), v.clone()
    assert kv.kv_append(ctx, K3, V3, tables, pos, None, kn, vn, rope=rope) is None
    assert torch.equal(K3, K) and torch.equal(V3, V)


def test_append_drops_rows_without_a_page(ctx, kv):
    k, v, tables, pos, _ = make(3, 4, 2, 2, 64, [62, 62, 62], F16)
    tables[0, 1] = -1           # its rows 2 and 3 have no page
    tables[1, 0] = k.shape[0]   # an entry behind the pool
    tables = tables[:, :1].contiguous()  # every row past the first page is outside the table
    kn, vn = torch.ones(3, 4, 2, 64, device="cuda", dtype=F16), torch.ones(3, 4, 2, 64, device="cuda", dtype=F16)
    K, V = k.clone(), v.clone()
    kv.kv_append(ctx, K, V, tables, pos, None, kn, vn)
    _, wk, wv = ref.append(k, v, tables.cpu(), pos.cpu(), None, kn, vn)
    assert torch.equal(K.double(), wk) and torch.equal(V.double(), wv)


# ------------------------------------------------------------------------------------------------ forks and moves
@pytest.mark.parametrize("pos,layers,nkv,hd,dtype", [(0, 1, 1, 64, F16), (1, 3, 2, 64, BF16), (64, 2, 1, 128, F16),
                                                     (130, 5, 8, 128, F16), (255, 2, 3, 64, F16), (256, 2, 3, 64, F16)])
def test_fork_shares_and_copies(ctx, kv, pos, layers, nkv, hd, dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn(layers, 12, nkv, PAGE, hd, device="cuda", generator=g).to(dtype)
    v = torch.randn(layers, 12, nkv, hd, PAGE, device="cuda", generator=g).to(dtype)
    tables = torch.full((6, 4), -7, dtype=torch.int32, device="cuda")
    tables[2] = torch.tensor([3, 9, 4, 1])
    tables[4] = torch.tensor([8, 2, 6, 0])
    p = torch.tensor([11, 12, pos, 13, pos, 14], dtype=torch.int64, device="cuda")
    K, V, T, P = k.clone(), v.clone(), tables.clone(), p.clone()
    parents, children, new = [2, 4, 2], [0, 1, 5], [5, 7, 10]
    kv.kv_fork(ctx, K, V, T, P, parents, children, new)
    for a, c, page in zip(parents, children, new):
        full = pos // PAGE
        tables[c, :full] = tables[a, :full]
        if full < 4:
            if pos % PAGE:
                k[:, page], v[:, page] = k[:, int(tables[a, full])], v[:, int(tables[a, full])]
            tables[c, full] = page
        p[c] = pos
    assert torch.equal(T, tables) and torch.equal(P, p) and torch.equal(K, k) and torch.equal(V, v)


def test_fork_of_an_idle_sequence_and_of_a_missing_page(ctx, kv):
    k = torch.randn(1, 6, 1, PAGE, 64, device="cuda", dtype=F16)
    v = torch.randn(1, 6, 1, 64, PAGE, device="cuda", dtype=F16)
    tables = torch.tensor([[0, 1], [2, -1], [3, 3], [4, 4]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([-1, 70, 5, 6], dtype=torch.int64, device="cuda")
    K, V = k.clone(), v.clone()
    kv.kv_fork(ctx, K, V, tables, pos, [0, 1], [2, 3], [5, 4])
    assert torch.equal(K, k) and torch.equal(V, v)  # nothing to copy
    assert tables.tolist() == [[0, 1], [2, -1], [3, 3], [2, 4]] and pos.tolist() == [-1, 70, -1, 70]


@pytest.mark.parametrize("moves,layers,nkv,hd", [(1, 1, 1, 64), (7, 3, 2, 128), (300, 2, 1, 64)])
def test_copy_pages_moves_pages_and_entries(ctx, kv, moves, layers, nkv, hd):
    g = torch.Generator(device="cuda").manual_seed(5)
    pages = 2 * moves + 5
    k = torch.randn(layers, pages, nkv, PAGE, hd, device="cuda", generator=g).to(BF16)
    v = torch.randn(layers, pages, nkv, hd, PAGE, device="cuda", generator=g).to(BF16)
    ids = np.random.default_rng(5).permutation(pages)
    src, dst = ids[:moves].tolist(), ids[moves:2 * moves].tolist()
    tables = torch.from_numpy(np.random.default_rng(6).integers(-1, pages, (9, 33)).astype(np.int32)).cuda()
    K, V, T = k.clone(), v.clone(), tables.clone()
    kv.kv_copy_pages(ctx, K, V, src, dst)
    assert torch.equal(T, tables)
    k[:, dst], v[:, dst] = k[:, src].clone(), v[:, src].clone()
    assert torch.equal(K, k) and torch.equal(V, v)
    kv.kv_copy_pages(ctx, K, V, src, dst, tables=T)
    to = dict(zip(src, dst))
    assert T.cpu().tolist() == [[to.get(x, x) for x in row] for row in tables.cpu().tolist()]
    assert torch.equal(K, k) and torch.equal(V, v)


# ------------------------------------------------------------------------------------------------ attention
def check(out, want, bound):
    nan = want.isnan()
    assert torch.equal(out.isnan(), nan)
    err = (out.double() - want).abs()
    assert bool((err <= bound)[~nan].all()), f"worst {float((err / bound)[~nan].max())} of the bound"


@pytest.mark.parametrize("n,positions,nh,nkv,hd,pos,dtype,shared", [
    (1, 1, 1, 1, 64, [0], F16, None),                                  # one position, which is its own row
    (1, 1, 8, 1, 128, [63], BF16, None),
    (1, 1, 8, 1, 128, [64], F16, None),
    (3, 2, 4, 2, 128, [0, 127, 700], F16, None),
    (2, 5, 6, 2, 64, [33, 64], BF16, None),                            # 15 rows: one tile of 16
    (1, 16, 8, 2, 128, [200], F16, None),                              # 64 rows: four tiles
    (1, 17, 7, 1, 64, [1], F16, None),                                 # 119 rows: eight tiles
    (1, 256, 2, 1, 64, [321], F16, None),                              # 512 rows: four row tiles
    (2, 100, 3, 3, 128, [0, 190], BF16, None),
    (4, 1, 4, 1, 128, [64, 65, 130, 500], F16, [(4, 1)]),              # one shared page, one sequence right at its end
    (6, 3, 4, 2, 128, [256, 300, 257, 280, 5, 90], F16, [(4, 4)]),     # two sequences outside the group
    (5, 2, 8, 4, 64, [640, 700, 130, 128, 129], BF16, [(2, 10), (3, 2)]),
    (33, 4, 4, 1, 128, [128 + 3 * i for i in range(33)], F16, [(33, 2)]),  # 528 shared rows: five row tiles
    (40, 1, 1, 1, 64, [i for i in range(40)], F16, None),
    (1, 1, 8, 8, 128, [30000], F16, None),                             # one long row: split over every CTA
    (2, 1, 16, 1, 128, [20000, 20003], BF16, [(2, 312)]),
])
def test_attention_against_64_bits(ctx, kv, n, positions, nh, nkv, hd, pos, dtype, shared):
    k, v, tables, p, q = make(n, positions, nh, nkv, hd, pos, dtype, shared=shared)
    out = kv.kv_attention(ctx, k, v, tables, p, q, groups=shared)
    check(out, *ref.attention(k, v, tables, p, q))
    # without the groups the same pages are read once per sequence: the same rows within the same bound
    if shared:
        check(kv.kv_attention(ctx, k, v, tables, p, q), *ref.attention(k, v, tables, p, q))


@pytest.mark.parametrize("n,positions,nh,nkv,pos,shared", [(1, 16, 4, 1, [100], None), (3, 31, 2, 2, [64, 70, 200], [(3, 1)]),
                                                           (1, 200, 2, 1, [50], None)])
def test_attention_over_a_tree(ctx, kv, n, positions, nh, nkv, pos, shared):
    k, v, tables, p, q = make(n, positions, nh, nkv, 128, pos, F16, shared=shared)
    parents = tree(np.random.default_rng(2), positions)
    check(kv.kv_attention(ctx, k, v, tables, p, q, groups=shared, parents=parents),
          *ref.attention(k, v, tables, p, q, parents))
    parents[positions // 2] = positions - 1  # not an earlier node: a root
    parents[positions - 1] = -9
    check(kv.kv_attention(ctx, k, v, tables, p, q, groups=shared, parents=parents),
          *ref.attention(k, v, tables, p, q, parents))


def test_attention_of_idle_sequences_and_missing_pages(ctx, kv):
    k, v, tables, p, q = make(5, 2, 4, 2, 128, [300, -1, 200, 90, -5], F16)
    tables[0, 2] = -1
    tables[2, 1] = k.shape[0] + 5
    tables[3, :] = -1  # nothing of it is in the cache: its rows see nothing
    room = torch.full((7, 2, 4, 128), 9.0, device="cuda", dtype=F16)
    out = kv.kv_attention(ctx, k, v, tables, p, q, out=room[1:6])
    want, bound = ref.attention(k, v, tables, p, q)
    check(out, want, bound)
    for b in (1, 3, 4):
        assert not out[b].any()
    assert bool((room[0] == 9).all()) and bool((room[6] == 9).all())  # rows before and behind stay as they are


def test_positions_behind_every_table(ctx, kv):
    """The largest positions: their rows have no page, are given back all the same, and see every page of the table."""
    k, v, tables, p, q = make(3, 4, 4, 2, 64, [130, 200, 100], F16)
    table = tables[:, :2].contiguous()
    for far in (2**63 - 1, 2**63 - 3, 2**62, 2**40):
        p[:] = torch.tensor([far, 2**63 - 64, far], device="cuda")
        K, V = k.clone(), v.clone()
        kn = torch.randn(3, 4, 2, 64, device="cuda", dtype=F16)
        room = torch.full((3, 4, 4, 64), math.nan, device="cuda", dtype=F16)
        assert torch.equal(kv.kv_append(ctx, K, V, table, p, q, kn, kn, out=room), q)
        assert torch.equal(K, k) and torch.equal(V, v)
        near = torch.full((3,), 128, dtype=torch.int64, device="cuda")  # as many positions as the tables hold
        for x in (q, torch.randn(3, 40, 4, 64, device="cuda", dtype=F16)):
            check(kv.kv_attention(ctx, k, v, table, p, x), *ref.attention(k, v, table, near, x))


@pytest.mark.parametrize("positions,nh", [(1, 2), (1, 16), (6, 8), (3, 64)])  # 1, 8, 24 and 96 rows per kv head of a sequence
def test_attention_of_a_group_whose_first_sequences_are_idle(ctx, kv, positions, nh):
    """The group's pages come from the table of a sequence that is not idle; the idle ones' tables name other pages, or none."""
    shared = [(8, 3), (3, 1)]
    pos = [200, 330, 192, 250, 400, 193, 300, 201, 64, 70, 65]
    k, v, tables, p, q = make(11, positions, nh, 2, 128, pos, F16, shared=shared)
    graph = None
    for idle in ([0], [0, 1, 2], [0, 3, 8, 9], [1, 10], list(range(8)), [0], list(range(11))):
        live, entries = p.clone(), tables.clone()
        for b in idle:
            live[b] = -1
            entries[b] = -1 if b % 2 else 0
        want, bound = ref.attention(k, v, entries, live, q)
        out = kv.kv_attention(ctx, k, v, entries, live, q, groups=shared)
        check(out, want, bound)
        assert not out[idle].any()
        if graph is None:
            held, named = live.clone(), entries.clone()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                again = kv.kv_attention(ctx, k, v, named, held, q, groups=shared)
        held.copy_(live)
        named.copy_(entries)
        graph.replay()
        assert torch.equal(again, out)


@pytest.mark.parametrize("hd,dtype,shared", [(64, F16, None), (128, BF16, None), (128, F16, [(3, 2)])])
def test_attention_ignores_what_is_not_seen(ctx, kv, hd, dtype, shared):
    """Infinities and NaN behind the last row, and in a row of the window: only rows that see them are touched."""
    k, v, tables, p, q = make(3, 4, 4, 2, hd, [130, 191, 128], dtype, shared=shared)
    ki, vi = (x.cuda() for x in ref.page_index(hd))
    for b in range(3):
        end = int(p[b]) + 4
        for slot in range(end, -(-end // PAGE) * PAGE):
            page = int(tables[b, slot // PAGE])
            k[page].view(2, -1)[:, ki[slot % PAGE]] = math.nan
            v[page].view(2, -1)[:, vi[slot % PAGE]] = math.inf if slot % 2 else math.nan
    want, bound = ref.attention(k, v, tables, p, q)
    assert not want.isnan().any()
    check(kv.kv_attention(ctx, k, v, tables, p, q, groups=shared), want, bound)
    slot = int(p[1]) + 2  # row 2 of sequence 1's window: rows 0 and 1 do not see it
    page = int(tables[1, slot // PAGE])
    v[page].view(2, -1)[0, vi[slot % PAGE][5]] = math.nan
    want, bound = ref.attention(k, v, tables, p, q)
    nan = want.isnan()
    assert nan[1, 2:, :2, 5].all() and int(nan.sum()) == 4
    check(kv.kv_attention(ctx, k, v, tables, p, q, groups=shared), want, bound)


@pytest.mark.parametrize("hd,dtype,nh,positions,shared,tr", [
    (128, F16, 4, 3, None, False),       # 6 rows a kv head: the stream kernel
    (64, BF16, 8, 4, None, True),        # 16
    (128, BF16, 16, 4, None, False),     # 32 and more: the tile kernel, alternate pages of a row tile
    (64, F16, 16, 20, None, True),       # 160: both streams' rows
    (128, F16, 16, 40, None, False),     # 320: two row tiles
    (128, F16, 4, 3, [(3, 2)], False),   # shared pages in the tile kernel, own ones in the stream kernel
    (64, BF16, 16, 4, [(2, 1)], False),
])
def test_attention_of_values_that_are_not_finite(ctx, kv, hd, dtype, nh, positions, shared, tr):
    """Infinities of either sign and NaN in a full page, in the last page's committed part and in the window: each row that
    sees one gets it, whichever kernel has the row."""
    base = [150, 200, 141]
    k, v, tables, p, q = make(3, positions, nh, 2, hd, base, dtype, shared=shared)
    parents = tree(np.random.default_rng(12), positions) if tr else None
    sees = ref.ancestors(parents, positions)
    ki, vi = (x.cuda() for x in ref.page_index(hd))
    odd = torch.zeros(3, positions, 2, hd, dtype=torch.float64, device="cuda")  # what the rows of a kv head see
    bad = v.clone()
    for b in range(3):
        full, partial = 70 + b, base[b] - 2  # of its own full page (a shared one for a group of two pages), and the last page
        marks = [(full, 3, math.inf), (full, 4, -math.inf), (full, 5, math.nan), (full, 6, math.inf), (full + 1, 6, -math.inf),
                 (partial, 7, math.inf), (partial, 8, -math.inf), (partial, 9, math.nan), (partial, 10, math.inf)]
        for j in {1, positions - 1}:
            slot = base[b] + j
            marks += [(slot, 11 + j % 3, math.inf), (slot, 14, -math.inf), (slot, 15, math.nan), (slot, 10, -math.inf), (slot, 3, math.inf)]
        if shared and b < shared[0][0] and shared[0][1] * PAGE > full:
            marks = [m for m in marks if m[0] > full + 1] if b else marks  # the group's page is marked once
        for slot, dim, value in marks:
            page, at = int(tables[b, slot // PAGE]), slot % PAGE
            k[page].view(2, -1)[:, ki[at]] = 0  # a score of 0: its weight is far from rounding to 0
            for h in range(2):
                d = dim + 20 * h
                bad[page, h].view(-1)[vi[at, d]] = value
                v[page, h].view(-1)[vi[at, d]] = 0
                for other in range(3):  # (a shared page is seen by every sequence that names it)
                    if int(tables[other, slot // PAGE]) != page:
                        continue
                    for i in range(positions):
                        if slot < base[other] or sees[i, slot - base[other]]:
                            odd[other, i, h, d] += value
    want, bound = ref.attention(k, v, tables, p, q, parents)
    want = want + odd.repeat_interleave(nh // 2, dim=2)
    assert want.isinf().any() and want.isnan().any()
    out = kv.kv_attention(ctx, k, bad, tables, p, q, groups=shared, parents=parents).double()
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out[want.isinf()], want[want.isinf()])
    finite = want.isfinite()
    assert out[finite].isfinite().all() and bool(((out - want).abs() <= bound)[finite].all())


@pytest.mark.parametrize("positions,nh,hd", [(33, 1, 64), (33, 2, 128), (20, 7, 64), (70, 4, 128)])
def test_attention_of_an_infinity_next_to_pages_that_are_not_seen(ctx, kv, positions, nh, hd):
    """The window begins in one page and ends in others, so that its first rows see nothing of these: an infinity in the first
    page reaches them as such, whichever warps have the other pages (enough sequences that a CTA takes several pages)."""
    n, nkv = 48, 4
    base = [(57, 2, 63, 50)[b % 4] for b in range(n)]
    k, v, tables, p, q = make(n, positions, nh * nkv, nkv, hd, base, BF16)
    ki, vi = (x.cuda() for x in ref.page_index(hd))
    bad, odd = v.clone(), torch.zeros(n, positions, nkv, hd, dtype=torch.float64, device="cuda")
    for b in range(n):
        for slot, d, value in ((base[b], 3, math.inf), (base[b] + 4, 5, -math.inf), (1, 7, math.inf), (base[b] + 1, 7, -math.inf),
                               (base[b] + positions - 1, 9, math.inf), (0, 11, math.nan)):
            page, at = int(tables[b, slot // PAGE]), slot % PAGE
            k[page].view(nkv, -1)[:, ki[at]] = 0
            v[page].view(nkv, -1)[:, vi[at, d]] = 0
            bad[page].view(nkv, -1)[:, vi[at, d]] = value
            odd[b, max(0, slot - base[b]):, :, d] += value
    want, bound = ref.attention(k, v, tables, p, q)
    want = want + odd.repeat_interleave(nh, dim=2)
    out = kv.kv_attention(ctx, k, bad, tables, p, q).double()
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out[want.isinf()], want[want.isinf()])
    finite = want.isfinite()
    assert bool(((out - want).abs() <= bound)[finite].all())


def test_attention_with_large_scores_and_another_scale(ctx, kv):
    k, v, tables, p, q = make(2, 3, 4, 2, 64, [100, 200], BF16)
    q = q * 40  # a softmax that is nearly one-hot
    check(kv.kv_attention(ctx, k, v, tables, p, q, scale=0.5), *ref.attention(k, v, tables, p, q, scale=0.5))
    check(kv.kv_attention(ctx, k, v, tables, p, q, scale=0.0), *ref.attention(k, v, tables, p, q, scale=0.0))


def test_attention_of_strided_queries(ctx, kv):
    k, v, tables, p, q = make(2, 3, 4, 2, 64, [100, 200], F16)
    wide = torch.randn(2, 3, 8, 64, device="cuda", dtype=F16)
    wide[:, :, 2:6] = q
    assert torch.equal(kv.kv_attention(ctx, k, v, tables, p, wide[:, :, 2:6]), kv.kv_attention(ctx, k, v, tables, p, q))


def test_attention_repeats_to_the_bit_and_on_two_streams(ctx, kv):
    a = make(9, 3, 8, 2, 128, [700 + 13 * i for i in range(9)], F16, shared=[(9, 10)])
    b = make(4, 16, 4, 1, 64, [900, 1, 64, 333], BF16, seed=9)
    want_a, want_b = kv.kv_attention(ctx, *a, groups=[(9, 10)]), kv.kv_attention(ctx, *b)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(one):
            x = kv.kv_attention(ctx, *a, groups=[(9, 10)])
        with torch.cuda.stream(two):
            y = kv.kv_attention(ctx, *b)
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, want_a) and torch.equal(y, want_b)


def test_attention_in_two_graphs_reads_current_tables_and_positions(ctx, kv):
    n, positions = 3, 2
    k, v, tables, p, q = make(n, positions, 4, 2, 128, [400, 500, 390], F16, shared=[(3, 6)])
    k2, v2, tables2, p2, q2 = make(2, 1, 4, 2, 128, [800, 5], F16, seed=4)
    kv.kv_attention(ctx, k, v, tables, p, q, groups=[(3, 6)])
    kv.kv_attention(ctx, k2, v2, tables2, p2, q2)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = kv.kv_attention(ctx, k, v, tables, p, q, groups=[(3, 6)])
    with torch.cuda.graph(g2):
        o2 = kv.kv_attention(ctx, k2, v2, tables2, p2, q2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for pos in ([400, 500, 390], [384, -1, 450], [511, 386, 400]):
        p.copy_(torch.tensor(pos))
        p2.copy_(torch.tensor([pos[2], 60]))
        q.normal_()
        tables[0, 6], tables[2, 6] = tables[2, 6].clone(), tables[0, 6].clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
        torch.cuda.synchronize()
        check(o1, *ref.attention(k, v, tables, p, q))
        check(o2, *ref.attention(k2, v2, tables2, p2, q2))


# ------------------------------------------------------------------------------------------------ refusals
def test_python_refusals(ctx, kv):
    k, v, tables, p, q = make(2, 3, 4, 2, 64, [10, 20], F16)
    ok = (k, v, tables, p, q)

    def swapped(i, x):
        return (*ok[:i], x, *ok[i + 1:])

    for bad in (swapped(0, k.cpu()), swapped(0, k.float()), swapped(0, k[:, :, :32].contiguous()),
                swapped(1, v.bfloat16()), swapped(2, tables.long()),
                swapped(2, tables[0]), swapped(2, tables[:, ::2]), swapped(3, p.int()), swapped(3, p[:1]),
                swapped(4, q.bfloat16()), swapped(4, q[..., :32]), swapped(4, q[0]), swapped(4, q.transpose(2, 3)),
                swapped(4, q[:, ::2])):
        with pytest.raises(ValueError):
            kv.kv_attention(ctx, *bad)
    for kw in (dict(groups=[(-1, 2)]), dict(parents=torch.zeros(2, dtype=torch.int32, device="cuda")),
               dict(parents=torch.zeros(3, device="cuda")), dict(out=torch.empty_like(q)[:1]),
               dict(out=torch.empty_like(q).float())):
        with pytest.raises(ValueError):
            kv.kv_attention(ctx, *ok, **kw)
    from clusterlm_b200._native import ClmError

    with pytest.raises(ClmError):
        kv.kv_attention(ctx, *ok, groups=[(3, 1)])
    with pytest.raises(ClmError):
        kv.kv_attention(ctx, *swapped(4, q[:, :, :3].contiguous()))
    k1, v1, t1, p1, q1 = make(2, 3, 4, 2, 128, [10, 20], F16)
    with pytest.raises(ValueError):  # (with 64 dims the two layouts of a page have one shape)
        kv.kv_attention(ctx, k1, v1.transpose(2, 3).contiguous(), t1, p1, q1)
    kn = torch.zeros(2, 3, 2, 64, device="cuda", dtype=F16)
    for args in ((q, kn, kn.float()), (q, kn, kn[:1]), (q.float(), kn, kn), (q[:1], kn, kn), (q, kn[:, :, :1], kn),
                 (q, kn.expand(2, 3, 2, 64)[:, :, :, ::2], kn)):
        with pytest.raises(ValueError):
            kv.kv_append(ctx, k, v, tables, p, *args)
    with pytest.raises(ValueError):
        kv.Rope(torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        kv.kv_append(ctx, k, v, tables, p, q, kn, kn, rope=kv.Rope(torch.ones(4, dtype=torch.float64)))
    with pytest.raises(ValueError):
        kv.kv_fork(ctx, k, v, tables, p, [0], [1], [0])  # a layer's pool where all layers are expected
    with pytest.raises(ValueError):
        kv.kv_fork(ctx, k[None], v[None], tables, p, [0], [1, 2], [0])
    with pytest.raises(ValueError):
        kv.kv_copy_pages(ctx, k[None], v[None], [0], [1, 2])
    with pytest.raises(ValueError):
        kv.kv_copy_pages(ctx, k[None], v[None], [0.5], [1])
