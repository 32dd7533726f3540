"""Paged KV-cache operators: rows in, attention, forks, page moves, and the host ledger of a pool's pages.

Python face of clm_b200_kv_* / clm_b200_pages_* over torch tensors that the caller owns:

  k_pool  (pages, n_kv_heads, 64, head_dim)   one layer's keys    (a whole cache: one more leading dim, layers)
  v_pool  (pages, n_kv_heads, head_dim, 64)   one layer's values
  tables  (rows, max_pages) int32             page of each sequence's positions 64 j .. 64 j + 63
  pos     (rows,) int64                       committed positions (negative: an idle sequence)

The pages' 16-byte chunks are permuted inside (include/clm_b200.h): kv_append writes them, kv_attention reads them.
Every call runs on torch's current stream of the context's device and can be captured into a CUDA graph; tables and
positions are read on the device, so a replay uses their current contents.  No reference counterpart: the reference's
sequence state is private to a domain (runtime/domain/src/reference_domain.cpp:297-329).
"""
from __future__ import annotations

import ctypes as C
from array import array

import numpy as np
import torch

from ._native import call, check, lib
from .runtime import DTYPES, Context, _operand, _stream_on

_vp = C.c_void_p
PAGE_TOKENS = 64
_POOL_TYPES = {torch.float16: 1, torch.bfloat16: 2}  # CLM_DTYPE_*


class _Pool(C.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("layers", C.c_uint32), ("pages", C.c_uint32), ("n_kv_heads", C.c_uint32),
                ("head_dim", C.c_uint32), ("dtype", C.c_int)]


class _Seqs(C.Structure):
    _fields_ = [("d_tables", _vp), ("d_pos", _vp), ("rows", C.c_uint32), ("max_pages", C.c_uint32)]


class _Rope(C.Structure):
    _fields_ = [("layout", C.c_int), ("rot", C.c_uint32), ("d_inv_freq", _vp), ("scale", C.c_float)]


def _pool(ctx: Context, k: torch.Tensor, v: torch.Tensor, layers: bool) -> _Pool:
    kp = _operand(ctx, "k_pool", k)
    dtype, shape = _POOL_TYPES.get(k.dtype), k.shape
    if dtype is None:
        raise ValueError("k_pool: expected float16 or bfloat16")
    if len(shape) != 4 + layers or shape[-2] != PAGE_TOKENS:
        raise ValueError(f"k_pool: expected {'(layers, ' if layers else '('}pages, n_kv_heads, 64, head_dim)")
    *lead, pages, heads, _, hd = shape
    vp = _operand(ctx, "v_pool", v, k.dtype, (*lead, pages, heads, hd, PAGE_TOKENS))
    return _Pool(kp, vp, lead[0] if layers else 1, pages, heads, hd, dtype)


def _seqs(ctx: Context, tables: torch.Tensor, pos: torch.Tensor) -> _Seqs:
    tp = _operand(ctx, "tables", tables, torch.int32)
    if tables.dim() != 2:
        raise ValueError("tables: expected (rows, max_pages)")
    rows, width = tables.shape
    return _Seqs(tp, _operand(ctx, "pos", pos, torch.int64, (rows,)), rows, width)


def _rows(ctx: Context, name: str, t: torch.Tensor, heads, head_dim: int):
    """(address, n, positions, heads, row stride) of rows (n, positions, heads, head_dim): the heads of a row are
    contiguous, and consecutive rows lie a fixed number of elements apart (a slice of a fused projection)."""
    p = _operand(ctx, name, t, contiguous=False)
    shape = t.shape
    if len(shape) != 4 or shape[3] != head_dim or (heads is not None and shape[2] != heads):
        raise ValueError(f"{name}: expected (n, positions, {heads or 'heads'}, {head_dim}), got {tuple(shape)}")
    n, positions, h, d = shape
    s0, s1, s2, s3 = t.stride()
    if n == 0 or positions == 0 or h == 0:
        return p, n, positions, h, h * d
    if s3 != 1 or (h > 1 and s2 != d):
        raise ValueError(f"{name}: a row's heads must be contiguous")
    ld = s1 if positions > 1 else (s0 if n > 1 else h * d)
    if ld < h * d or (n > 1 and positions > 1 and s0 != positions * ld):
        raise ValueError(f"{name}: rows must lie a fixed distance apart")
    return p, n, positions, h, ld


def _result(ctx: Context, out, dtype, like: torch.Tensor, shape):
    """The caller's output tensor, or a new one, and its address."""
    if out is not None:
        return out, _operand(ctx, "out", out, dtype, shape)
    out = torch.empty_like(like) if like.dtype is dtype and like.is_contiguous() else like.new_empty(shape, dtype=dtype)
    return out, out.data_ptr()


def _parents(ctx: Context, parents, positions: int):
    return None if parents is None else _operand(ctx, "parents", parents, torch.int32, (positions,))


def _count(name: str, x, most: int = 2**32 - 1) -> int:
    """A count as the C ABI takes it (ctypes would drop the bits above its type)."""
    if not 0 <= x <= most:
        raise ValueError(f"{name}: expected 0 to {most}")
    return x


ROPE_KINDS = {"plain": 0, "linear": 1, "bands": 2, "yarn": 3}


def rope_frequencies(rot: int, theta: float, kind: str = "plain", factor: float = 1.0, low: float = 1.0,
                     high: float = 4.0, original: float = 8192.0) -> tuple[np.ndarray, float]:
    """(frequencies float64 (rot / 2,), scale) of rotary positions: theta^(-2j / rot) as they are ("plain"), divided by
    `factor` ("linear"), kept above `high` turns in the `original` context, divided below `low` and blended between
    ("bands"), or blended over the pair index with the scale 0.1 ln(factor) + 1 ("yarn")."""
    if kind not in ROPE_KINDS:
        raise ValueError(f"unknown frequency scaling {kind!r}: one of {', '.join(ROPE_KINDS)}")
    rot = _count("rot", max(0, rot), 2**20)
    out, scale = np.empty(rot // 2, np.float64), C.c_float()
    call("clm_b200_rope_frequencies", ROPE_KINDS[kind], rot, theta, factor, low, high, original,
         out.ctypes.data_as(_vp), C.byref(scale))
    return out, scale.value


class Rope:
    """Rotary positions of the leading 2 * len(inv_freq) dims of a head: inv_freq float64 on the device (see
    rope_frequencies), pairs (2j, 2j + 1) when interleaved, else (j, j + rot / 2); `scale` multiplies the rotated part."""

    def __init__(self, inv_freq: torch.Tensor, interleaved: bool = True, scale: float = 1.0):
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1 or inv_freq.dtype != torch.float64:
            raise ValueError("inv_freq: expected a float64 vector")
        self.inv_freq, self.interleaved, self.scale = inv_freq, bool(interleaved), float(scale)

    def _c(self, ctx: Context) -> _Rope:
        return _Rope(0 if self.interleaved else 1, 2 * self.inv_freq.numel(), _operand(ctx, "inv_freq", self.inv_freq),
                     self.scale)


def kv_append(ctx: Context, k_pool, v_pool, tables, pos, q, k, v, rope: Rope | None = None, parents=None, out=None):
    """Puts rows k, v (n, positions, n_kv_heads, head_dim) of sequences 0..n-1 into the cache at pos[b] + i, k rotated,
    and returns q (n, positions, heads, head_dim) rotated, in the cache's type (None for q = None).  q, k and v have one
    type (f32, f16 or bf16) and may be slices of one tensor.  parents int32 (positions,): a tree window, node i at slot
    pos[b] + i and rotated at pos[b] + its depth.  pos is not advanced."""
    pool, seqs = _pool(ctx, k_pool, v_pool, False), _seqs(ctx, tables, pos)
    hd, nkv = pool.head_dim, pool.n_kv_heads
    kp, n, positions, _, ldk = _rows(ctx, "k", k, nkv, hd)
    vp, vn, vpos, _, ldv = _rows(ctx, "v", v, nkv, hd)
    if (vn, vpos) != (n, positions) or v.dtype != k.dtype or k.dtype not in DTYPES:
        raise ValueError("k and v: expected the same shape and type (float32, float16 or bfloat16)")
    qp, heads, ldq, op = None, 0, 0, None
    if q is not None:
        qp, qn, qpos, heads, ldq = _rows(ctx, "q", q, None, hd)
        if (qn, qpos) != (n, positions) or q.dtype != k.dtype:
            raise ValueError("q: expected the rows and type of k")
        out, op = _result(ctx, out, k_pool.dtype, q, (n, positions, heads, hd))
    r = rope._c(ctx) if rope is not None else None
    check(lib.clm_b200_kv_append(ctx.h, C.byref(pool), 0, C.byref(seqs), n, positions, heads, DTYPES[k.dtype], qp, ldq, kp,
                                 ldk, vp, ldv, None if r is None else C.byref(r), _parents(ctx, parents, positions), op,
                                 _stream_on(ctx.device)))
    return out if q is not None else None


def kv_attention(ctx: Context, k_pool, v_pool, tables, pos, q, groups=None, scale: float | None = None, parents=None,
                 out=None):
    """Attention of rows q (n, positions <= 256, heads, head_dim) of sequences 0..n-1 over the cache that kv_append
    filled: row i of sequence b sees the positions below pos[b] and window rows 0..i (with parents: its ancestors and
    itself).  groups [(sequences, pages), ...]: consecutive sequences whose first `pages` table entries are the same
    (or which are idle: their tables are not read); these pages are read once for the group.  scale: 1 / sqrt(head_dim) by default.  Returns the outputs in q's type."""
    pool, seqs = _pool(ctx, k_pool, v_pool, False), _seqs(ctx, tables, pos)
    hd = pool.head_dim
    qp, n, positions, heads, ldq = _rows(ctx, "q", q, None, hd)
    if q.dtype is not k_pool.dtype:
        raise ValueError(f"q: expected {k_pool.dtype}, got {q.dtype}")
    g, counts, pages = 0, None, None
    if groups:
        g = len(groups)
        for c, p in groups:
            if not (0 <= c < 2**32 and 0 <= p < 2**32):
                raise ValueError("groups: expected (sequences, pages) of zero or more")
        counts, pages = (C.c_uint32 * g)(*[c for c, _ in groups]), (C.c_uint32 * g)(*[p for _, p in groups])
    out, op = _result(ctx, out, q.dtype, q, (n, positions, heads, hd))
    need = C.c_uint64()
    check(lib.clm_b200_kv_attention_workspace(ctx.h, n, positions, heads, pool.n_kv_heads, hd, g, counts, pages,
                                              C.byref(need)))
    need = need.value
    work = torch.empty(need, dtype=torch.uint8, device=q.device)  # this call's own: captured graphs keep theirs
    check(lib.clm_b200_kv_attention(ctx.h, C.byref(pool), 0, C.byref(seqs), n, positions, heads, qp, ldq, g, counts, pages,
                                    _parents(ctx, parents, positions), hd**-0.5 if scale is None else scale, op,
                                    work.data_ptr(), need, _stream_on(ctx.device)))
    return out


def set_wait_limit(ctx: Context, polls: int = 2**20) -> None:
    """Polls after which a device wait inside kv_attention gives up and leaves NaN rows, for later calls of the context
    and later windows of its engines (whose commit then fails); captured ones keep theirs."""
    call("clm_b200_kv_attention_wait_limit", ctx.h, _count("polls", polls))


def _ints(name: str, a, dtype):
    """(address, entries, their owner) of integers: a list, or an array that is copied unless it has the type."""
    if isinstance(a, (list, tuple, range)):
        try:
            a = array("I" if dtype is np.uint32 else "i", a)
            return a.buffer_info()[0], len(a), a
        except (TypeError, OverflowError):
            pass  # (said below)
    a = np.asarray(a)
    if a.dtype == dtype and a.ndim == 1 and a.flags.c_contiguous:
        return a.ctypes.data, a.size, a
    if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
        raise ValueError(f"{name}: expected a list of integers")
    lim = np.iinfo(dtype)
    if a.size and (int(a.min()) < lim.min or int(a.max()) > lim.max):
        raise ValueError(f"{name}: an entry is out of range")
    a = np.ascontiguousarray(a, dtype=dtype)
    return a.ctypes.data, a.size, a


def kv_fork(ctx: Context, k_pools, v_pools, tables, pos, parents, children, new_pages) -> None:
    """Row children[i] of the tables becomes a continuation of row parents[i]: the full pages shared, the last page
    copied into new_pages[i] in every layer (pools with a leading layers dim), the position taken over."""
    pool, seqs = _pool(ctx, k_pools, v_pools, True), _seqs(ctx, tables, pos)
    (p, n, _p), (c, nc, _c), (g, ng, _g) = (_ints("parents", parents, np.uint32), _ints("children", children, np.uint32),
                                            _ints("new_pages", new_pages, np.int32))
    if not n == nc == ng:
        raise ValueError("parents, children and new_pages: expected one entry per fork")
    check(lib.clm_b200_kv_fork(ctx.h, C.byref(pool), C.byref(seqs), n, p, c, g, _stream_on(ctx.device)))


def kv_copy_pages(ctx: Context, k_pools, v_pools, src, dst, tables=None) -> None:
    """Copies page src[i] to dst[i] in every layer (pools with a leading layers dim); with tables, entries that name
    src[i] then name dst[i]."""
    pool = _pool(ctx, k_pools, v_pools, True)
    (s, n, _s), (d, nd, _d) = _ints("src", src, np.int32), _ints("dst", dst, np.int32)
    if n != nd:
        raise ValueError("src and dst: expected one entry per page")
    tp = None if tables is None else _operand(ctx, "tables", tables, torch.int32)
    check(lib.clm_b200_kv_copy_pages(ctx.h, C.byref(pool), n, s, d, tp, 0 if tables is None else tables.numel(),
                                     _stream_on(ctx.device)))


class Pages:
    """Host ledger of a pool's pages: free ones, and how many sequences hold each."""

    def __init__(self, pages: int):
        self.h = None
        h = _vp()
        call("clm_b200_pages_create", _count("pages", pages), C.byref(h))
        self.h, self.pages = h, pages

    def close(self) -> None:
        if self.h:
            call("clm_b200_pages_destroy", self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def alloc(self, n: int) -> list[int]:
        """The n lowest free pages, one holder each (none is taken when fewer are free)."""
        ids = np.empty(_count("n", n, 2**31 - 1), np.int32)
        call("clm_b200_pages_alloc", self.h, n, ids.ctypes.data_as(_vp))
        return ids.tolist()

    def retain(self, ids) -> None:
        a, n, _a = _ints("ids", ids, np.int32)
        call("clm_b200_pages_retain", self.h, n, a)

    def release(self, ids) -> None:
        a, n, _a = _ints("ids", ids, np.int32)
        call("clm_b200_pages_release", self.h, n, a)

    def holders(self, page: int) -> int:
        r = C.c_uint32()
        call("clm_b200_pages_info", self.h, _count("page", page, 2**31 - 1) if page >= 0 else -1, C.byref(r), None)
        return r.value

    def free(self) -> int:
        f = C.c_uint32()
        call("clm_b200_pages_info", self.h, 0, None, C.byref(f))
        return f.value

    def compact(self) -> tuple[list[int], list[int]]:
        """(src, dst) of the moves that pack the live pages into the lowest ones, for kv_copy_pages; the ledger counts
        them as done."""
        cap = self.pages - self.free()
        src, dst, n = np.empty(cap, np.int32), np.empty(cap, np.int32), C.c_uint32()
        call("clm_b200_pages_compact", self.h, cap, src.ctypes.data_as(_vp), dst.ctypes.data_as(_vp), C.byref(n))
        return src[: n.value].tolist(), dst[: n.value].tolist()
