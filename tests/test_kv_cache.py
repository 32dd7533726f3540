"""Host side of the paged-cache operators and of sampling from logits: the page ledger against a model of it, rotary
frequencies against their formulas, and every refusal of the C ABI (checked before a device is touched, so without a
GPU)."""
import ctypes as C
import math
import random

import numpy as np
import pytest

from clusterlm_b200 import _native
from clusterlm_b200._native import ClmError
from clusterlm_b200.kv_cache import Pages, _Pool, _Rope, _Seqs, rope_frequencies

INVALID, RANGE, NOT_FOUND, EXHAUSTED, UNIMPLEMENTED = 1, 2, 3, 6, 18


# ------------------------------------------------------------------------------------------------ page ledger
def test_pages_follow_a_model_of_them():
    rng = random.Random(7)
    pages = Pages(40)
    refs = [0] * 40
    for _ in range(3000):
        what = rng.random()
        live = [i for i in range(40) if refs[i]]
        if what < 0.35:
            n = rng.randrange(0, 9)
            free = [i for i in range(40) if not refs[i]]
            if n > len(free):
                with pytest.raises(ClmError) as err:
                    pages.alloc(n)
                assert err.value.code == EXHAUSTED
            else:
                got = pages.alloc(n)
                assert got == free[:n]
                for i in got:
                    refs[i] = 1
        elif what < 0.5 and live:
            some = [rng.choice(live) for _ in range(rng.randrange(1, 5))]
            pages.retain(some)
            for i in some:
                refs[i] += 1
        elif what < 0.9 and live:
            some = [rng.choice(live) for _ in range(rng.randrange(1, 5))]
            short = any(some.count(i) > refs[i] for i in some)
            if short:
                with pytest.raises(ClmError) as err:
                    pages.release(some)
                assert err.value.code == NOT_FOUND
            else:
                pages.release(some)
                for i in some:
                    refs[i] -= 1
        elif what > 0.97:
            src, dst = pages.compact()
            n = len(live)
            assert src == [i for i in live if i >= n] and dst == [i for i in range(n) if not refs[i]]
            for s, d in zip(src, dst):
                refs[d], refs[s] = refs[s], 0
            assert all(refs[i] for i in range(n)) and not any(refs[n:])
        assert pages.free() == refs.count(0)
        i = rng.randrange(40)
        assert pages.holders(i) == refs[i]


def test_pages_refuse():
    with pytest.raises(ClmError):
        Pages(0)
    pages = Pages(4)
    for bad in ([4], [-1], [0]):  # outside the pool, or not in use
        with pytest.raises(ClmError) as err:
            pages.release(bad)
        assert err.value.code == NOT_FOUND
        with pytest.raises(ClmError):
            pages.retain(bad)
    with pytest.raises(ClmError):
        pages.holders(4)
    a = pages.alloc(3)
    with pytest.raises(ClmError):  # the third release of page 0 is one too many: nothing is released
        pages.release([a[0], a[1], a[0]])
    assert [pages.holders(i) for i in range(4)] == [1, 1, 1, 0] and pages.free() == 1
    with pytest.raises(ValueError):
        pages.release([1.5])
    with pytest.raises(ValueError):
        pages.retain([2**40])
    assert pages.compact() == ([], [])
    pages.close()
    with pytest.raises(ClmError):
        pages.alloc(1)


# ------------------------------------------------------------------------------------------------ rotary frequencies
def test_rope_frequencies_follow_their_formulas():
    theta, rot, factor, ctx = 500000.0, 128, 8.0, 8192.0
    plain = np.array([theta ** (-2 * j / rot) for j in range(rot // 2)])
    f, scale = rope_frequencies(rot, theta)
    np.testing.assert_allclose(f, plain, rtol=1e-14)
    assert scale == 1.0
    f, _ = rope_frequencies(rot, theta, "linear", factor)
    np.testing.assert_allclose(f, plain / factor, rtol=1e-14)
    f, scale = rope_frequencies(rot, theta, "bands", factor, 1.0, 4.0, ctx)
    for j, x in enumerate(f):
        turns = ctx * plain[j] / (2 * math.pi)
        want = plain[j] if turns >= 4 else plain[j] / factor if turns <= 1 else \
            ((turns - 1) / 3) * plain[j] + (1 - (turns - 1) / 3) * plain[j] / factor
        assert x == pytest.approx(want, rel=1e-13)
    assert scale == 1.0
    f, scale = rope_frequencies(rot, 10000.0, "yarn", 16.0, 1.0, 32.0, 4096.0)
    assert scale == pytest.approx(0.1 * math.log(16.0) + 1.0, rel=1e-6)
    plain = np.array([10000.0 ** (-2 * j / rot) for j in range(rot // 2)])
    first = math.floor(rot * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    last = math.ceil(rot * math.log(4096 / (1 * 2 * math.pi)) / (2 * math.log(10000.0)))
    ramp = np.clip((np.arange(rot // 2) - first) / (last - first), 0, 1)
    np.testing.assert_allclose(f, plain * (1 - ramp) + plain / 16 * ramp, rtol=1e-12)
    assert f[0] == 1.0 and f[-1] == pytest.approx(plain[-1] / 16)


@pytest.mark.parametrize("args", [(0, 1e4), (7, 1e4), (8, 1.0), (8, float("nan")), (8, 1e4, "linear", 0.5),
                                  (8, 1e4, "linear", float("inf")), (8, 1e4, "bands", 2.0, 4.0, 1.0),
                                  (8, 1e4, "bands", 2.0, 0.0, 1.0), (8, 1e4, "yarn", 2.0, 1.0, 32.0, 0.0)])
def test_rope_frequencies_refuse(args):
    with pytest.raises(ClmError) as err:
        rope_frequencies(*args)
    assert err.value.code == INVALID


def test_rope_frequencies_refuse_an_unknown_kind():
    with pytest.raises(ValueError):
        rope_frequencies(8, 1e4, "cubic")


# ------------------------------------------------------------------------------------------------ refusals
# Every check comes before the first CUDA call: a zeroed context (device 0) and made-up aligned addresses suffice, and
# nothing is launched because each call differs from a valid one in one argument that is refused.
FAKE = C.create_string_buffer(4096)
CTX = C.cast(FAKE, C.c_void_p)
A = 1 << 20  # an aligned "device address"


def vp(x):
    return C.c_void_p(x)


def pool(**kw):
    d = dict(k=A, v=A, layers=2, pages=10, n_kv_heads=2, head_dim=128, dtype=1)
    d.update(kw)
    return _Pool(*(d[k] for k in ("k", "v", "layers", "pages", "n_kv_heads", "head_dim", "dtype")))


def seqs(**kw):
    d = dict(d_tables=A, d_pos=A, rows=4, max_pages=8)
    d.update(kw)
    return _Seqs(*(d[k] for k in ("d_tables", "d_pos", "rows", "max_pages")))


BAD_POOLS = [(dict(k=0), INVALID), (dict(v=0), INVALID), (dict(layers=0), INVALID), (dict(pages=0), INVALID),
             (dict(pages=2**31), RANGE), (dict(n_kv_heads=0), INVALID), (dict(n_kv_heads=70000), RANGE),
             (dict(head_dim=96), UNIMPLEMENTED), (dict(dtype=0), UNIMPLEMENTED), (dict(dtype=7), UNIMPLEMENTED),
             (dict(k=A + 2), INVALID)]
BAD_SEQS = [(dict(d_tables=0), INVALID), (dict(d_pos=0), INVALID), (dict(rows=0), INVALID),
            (dict(max_pages=0), INVALID), (dict(max_pages=2**26), INVALID)]


def append(ctx=CTX, p=None, layer=0, s=None, n=2, positions=3, heads=4, src=1, q=A, ld_q=1024, k=A, ld_k=1024, v=A,
           ld_v=1024, rope=None, parents=0, out=A):
    p, s = pool() if p is None else p, seqs() if s is None else s
    return _native.lib.clm_b200_kv_append(ctx, C.byref(p), layer, C.byref(s), n, positions, heads, src, vp(q), ld_q, vp(k),
                                          ld_k, vp(v), ld_v, None if rope is None else C.byref(rope), vp(parents), vp(out),
                                          None)


APPEND = [(dict(ctx=None), INVALID), (dict(layer=2), RANGE), (dict(n=5), RANGE), (dict(heads=3), INVALID),
          (dict(src=3), INVALID), (dict(src=-1), INVALID), (dict(k=0), INVALID), (dict(v=0), INVALID),
          (dict(out=0), INVALID), (dict(heads=0), INVALID), (dict(out=A + 8), INVALID), (dict(ld_k=255), INVALID),
          (dict(ld_v=255), INVALID), (dict(ld_q=511), INVALID), (dict(ld_q=2**41), INVALID),
          (dict(positions=2**25), RANGE), (dict(positions=257, parents=A), RANGE),
          (dict(rope=_Rope(2, 64, A, 1.0)), INVALID), (dict(rope=_Rope(0, 63, A, 1.0)), INVALID),
          (dict(rope=_Rope(0, 130, A, 1.0)), INVALID), (dict(rope=_Rope(0, 64, 0, 1.0)), INVALID)]


@pytest.mark.parametrize("kw,code", APPEND + [(dict(p=pool(**p)), c) for p, c in BAD_POOLS]
                         + [(dict(s=seqs(**s)), c) for s, c in BAD_SEQS])
def test_append_refuses(kw, code):
    assert append(**kw) == code


@pytest.mark.parametrize("q,out,ld_q,src", [(A, A, 1024, 1), (A, A + 8192, 1024, 1), (A + 6128, A, 512, 1), (A, A + 22512, 1024, 0)])
def test_append_refuses_to_rotate_in_place(q, out, ld_q, src):
    """Six rows of 512 elements: the rows from q on (5 strides and a row), the result's 6,144 bytes."""
    assert append(q=q, out=out, ld_q=ld_q, src=src) == INVALID
    assert b"overlap" in _native.lib.clm_b200_last_error()


def attention(ctx=CTX, p=None, layer=0, s=None, n=3, positions=2, heads=4, q=A, ld_q=512, groups=(), parents=0, out=A,
              work=A, work_bytes=1 << 40, null_groups=False, scale=0.1):
    p, s = pool() if p is None else p, seqs() if s is None else s
    counts = (C.c_uint32 * 80)(*[g[0] for g in groups])
    pages = (C.c_uint32 * 80)(*[g[1] for g in groups])
    return _native.lib.clm_b200_kv_attention(ctx, C.byref(p), layer, C.byref(s), n, positions, heads, vp(q), ld_q,
                                             len(groups) or int(null_groups), None if null_groups else counts,
                                             None if null_groups else pages, vp(parents), scale, vp(out), vp(work),
                                             work_bytes, None)


ATTENTION = [(dict(ctx=None), INVALID), (dict(layer=2), RANGE), (dict(n=5), RANGE), (dict(n=513, s=seqs(rows=600)), RANGE),
             (dict(positions=257), RANGE), (dict(heads=3), INVALID), (dict(heads=0), INVALID), (dict(heads=2048), RANGE),
             (dict(q=0), INVALID), (dict(out=0), INVALID), (dict(work=0), INVALID), (dict(ld_q=504), INVALID),
             (dict(ld_q=513), INVALID), (dict(q=A + 2), INVALID), (dict(out=A + 8), INVALID), (dict(work=A + 8), INVALID),
             (dict(groups=[(2, 1), (2, 1)]), INVALID), (dict(groups=[(0, 1)] * 65), RANGE),
             (dict(scale=-0.1), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
             (dict(null_groups=True), INVALID), (dict(groups=[(2**32 - 1, 1), (2, 1)]), INVALID)]


@pytest.mark.parametrize("kw,code", ATTENTION + [(dict(p=pool(**p)), c) for p, c in BAD_POOLS]
                         + [(dict(s=seqs(**s)), c) for s, c in BAD_SEQS])
def test_attention_refuses(kw, code):
    assert attention(**kw) == code


def fork(ctx=CTX, p=None, s=None, forks=((0, 1, 5), (0, 2, 6)), n=None):
    p, s = pool() if p is None else p, seqs() if s is None else s
    a = [np.array([f[i] for f in forks], t) for i, t in enumerate((np.uint32, np.uint32, np.int32))]
    return _native.lib.clm_b200_kv_fork(ctx, C.byref(p), C.byref(s), len(forks) if n is None else n,
                                        *(x.ctypes.data_as(C.c_void_p) for x in a), None)


FORK = [(dict(ctx=None), INVALID), (dict(forks=[(4, 1, 5)]), RANGE), (dict(forks=[(0, 4, 5)]), RANGE),
        (dict(forks=[(0, 1, 10)]), RANGE), (dict(forks=[(0, 1, -1)]), RANGE), (dict(forks=[(0, 1, 5), (2, 1, 6)]), INVALID),
        (dict(forks=[(0, 0, 5)]), INVALID), (dict(forks=[(0, 1, 5), (1, 2, 6)]), INVALID),
        (dict(forks=[(0, 1, 5), (0, 2, 5)]), INVALID), (dict(n=257), RANGE), (dict(s=seqs(rows=70000)), RANGE)]


@pytest.mark.parametrize("kw,code", FORK + [(dict(p=pool(**p)), c) for p, c in BAD_POOLS]
                         + [(dict(s=seqs(**s)), c) for s, c in BAD_SEQS])
def test_fork_refuses(kw, code):
    assert fork(**kw) == code


def copy(ctx=CTX, p=None, pairs=((1, 2), (3, 4)), tables=0):
    p = pool() if p is None else p
    a = [np.array([x[i] for x in pairs], np.int32) for i in range(2)]
    return _native.lib.clm_b200_kv_copy_pages(ctx, C.byref(p), len(pairs), *(x.ctypes.data_as(C.c_void_p) for x in a),
                                              vp(tables), 8, None)


COPY = [(dict(ctx=None), INVALID), (dict(pairs=[(10, 1)]), RANGE), (dict(pairs=[(1, 10)]), RANGE),
        (dict(pairs=[(-1, 1)]), RANGE), (dict(pairs=[(1, -2)]), RANGE), (dict(pairs=[(1, 2), (3, 2)]), INVALID),
        (dict(pairs=[(1, 1)]), INVALID), (dict(pairs=[(1, 2), (2, 3)]), INVALID),
        (dict(pairs=[(1, 2), (1, 3)], tables=A), INVALID)]


@pytest.mark.parametrize("kw,code", COPY + [(dict(p=pool(**p)), c) for p, c in BAD_POOLS])
def test_copy_refuses(kw, code):
    assert copy(**kw) == code


def sample(ctx=CTX, logits=A, dtype=0, rows=3, vocab=100, ld=100, u=A, out=A):
    return _native.lib.clm_b200_sample_logits(ctx, vp(logits), dtype, rows, vocab, ld, None, None, None, None, vp(u),
                                              vp(out), None, None)


@pytest.mark.parametrize("kw,code", [(dict(ctx=None), INVALID), (dict(vocab=0), INVALID),
                                     (dict(vocab=385025, ld=385025), RANGE), (dict(ld=99), INVALID),
                                     (dict(dtype=3), INVALID), (dict(dtype=-1), INVALID), (dict(logits=0), INVALID),
                                     (dict(u=0), INVALID), (dict(out=0), INVALID), (dict(rows=2**30), RANGE)])
def test_sample_refuses(kw, code):
    assert sample(**kw) == code


def test_empty_calls_touch_nothing():
    assert append(n=0) == 0 and append(positions=0) == 0
    assert attention(n=0) == 0 and attention(positions=0) == 0
    assert fork(forks=()) == 0 and copy(pairs=()) == 0 and sample(rows=0) == 0
    need = C.c_uint64(9)
    assert _native.lib.clm_b200_kv_attention_workspace(CTX, 0, 4, 8, 8, 128, 0, None, None, C.byref(need)) == 0
    assert need.value == 0


def test_wait_limit_refuses():
    from clusterlm_b200.kv_cache import set_wait_limit

    class Ctx:
        h = None

    with pytest.raises(ClmError) as err:
        set_wait_limit(Ctx())
    assert err.value.code == INVALID
    for polls in (-1, 2**32):
        with pytest.raises(ValueError):
            set_wait_limit(Ctx(), polls)


def test_counts_that_no_32_bits_hold():
    """ctypes keeps the low bits of an integer: such counts must not become other, valid ones."""
    with pytest.raises(ValueError):
        Pages(2**32 + 5)
    with pytest.raises(ValueError):
        Pages(-1)
    pages = Pages(5)
    assert pages.alloc(2) == [0, 1]
    for call, x in ((pages.alloc, 2**32 + 1), (pages.alloc, -1), (pages.holders, 2**32)):
        with pytest.raises(ValueError):
            call(x)
    for page in (-1, -2**32, -2**32 + 1):
        with pytest.raises(ClmError) as err:
            pages.holders(page)
        assert err.value.code == RANGE
    assert pages.free() == 3
    for rot in (2**32 + 2, 2**21):
        with pytest.raises(ValueError):
            rope_frequencies(rot, 1e4)
    with pytest.raises(ClmError) as err:
        rope_frequencies(-2**32 + 4, 1e4)
    assert err.value.code == INVALID


@pytest.mark.parametrize("k,v,out", [(A, A + 2**16, A + 2047), (A, A + 2**16, A + 2**16 - 6144 + 16), (A + 2**16, A, A + 16),
                                     (A + 2**16, A, A + 2**16 + 5 * 512 + 512 - 16)])
def test_append_refuses_queries_over_keys_or_values(k, v, out):
    """Six rows of two kv heads of 128 in 16 bits, 256 elements apart: 3,072 bytes each; the result's 6,144 bytes."""
    assert append(q=A + 2**20, k=k, v=v, out=out & ~15, ld_q=512, ld_k=256, ld_v=256) == INVALID
    assert b"overlap" in _native.lib.clm_b200_last_error()


def test_append_refuses_rows_beyond_any_memory():
    assert append(n=4, positions=2**24, ld_k=2**39, out=A + 2**40) == RANGE
    assert append(n=4, positions=2**24, q=0, heads=0, ld_v=2**39) == RANGE
