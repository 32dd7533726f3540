"""Plain 64-bit forms of the paged-cache operators and of sampling from logits, for the tests."""
from __future__ import annotations

import math
from fractions import Fraction

import numpy as np
import torch

PAGE = 64


def page_index(hd: int):
    """Offsets in a stored page: K (position, dim) and V (position, dim)."""
    pos, dim = torch.arange(PAGE).view(-1, 1), torch.arange(hd).view(1, -1)
    c = dim // 8
    k = pos * hd + 8 * (c ^ torch.where(c >= 8, 2, 0) ^ (pos % 2)) + dim % 8
    v = dim * PAGE + 8 * ((pos // 8) ^ (dim % 2)) + pos % 8
    return k, v


def unpack(pool: torch.Tensor, hd: int, values: bool) -> torch.Tensor:
    """(pages, heads, 64, hd) of a layer's pool in position order."""
    at = page_index(hd)[1 if values else 0].to(pool.device)
    return pool.reshape(pool.shape[0], pool.shape[1], -1)[:, :, at.reshape(-1)].view(*pool.shape[:2], PAGE, hd)


def ancestors(parents, positions: int) -> torch.Tensor:
    """sees[i, j]: window row i sees window row j.  A parent that is not an earlier node ends the chain."""
    sees = torch.zeros(positions, positions, dtype=torch.bool)
    for i in range(positions):
        at = i
        while True:
            sees[i, at] = True
            up = at - 1 if parents is None else int(parents[at])
            if up < 0 or up >= at:
                break
            at = up
    return sees


def append(k_pool, v_pool, tables, pos, q, k, v, freqs=None, interleaved=True, scale=1.0, parents=None):
    """(q rotated, K pool, V pool) in float64; elements that no row writes keep their values."""
    n, p, nkv, hd = k.shape
    K, V = k_pool.double().clone(), v_pool.double().clone()
    depth = ancestors(parents, p).sum(1) - 1
    ki, vi = (x.to(k.device) for x in page_index(hd))

    def turn(x, at):
        x = x.double().clone()
        if freqs is None or len(freqs) == 0:
            return x
        rot = 2 * len(freqs)
        a = float(at) * freqs.double().cpu()
        c, s = (scale * torch.cos(a)).to(x.device), (scale * torch.sin(a)).to(x.device)
        one, two = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        u, w = x[..., one].clone(), x[..., two].clone()
        x[..., one], x[..., two] = u * c - w * s, u * s + w * c
        return x

    Q = None if q is None else torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b in range(n):
        base = int(pos[b])
        if base < 0:
            continue
        for i in range(p):
            if q is not None:
                Q[b, i] = turn(q[b, i], base + int(depth[i]))
            slot = base + i
            page = int(tables[b, slot // PAGE]) if slot // PAGE < tables.shape[1] else -1
            if not 0 <= page < k_pool.shape[0]:
                continue
            K[page].view(nkv, -1)[:, ki[slot % PAGE]] = turn(k[b, i], base + int(depth[i]))
            V[page].view(nkv, -1)[:, vi[slot % PAGE]] = v[b, i].double()
    return Q, K, V


def attention(k_pool, v_pool, tables, pos, q, parents=None, scale=None):
    """(outputs, bound): float64 outputs, and for each the error that one rounding of every weight and of the output to
    the operands' type, f32 products, sums and exponentials allow."""
    n, p, nh, hd = q.shape
    nkv, pages = k_pool.shape[1], k_pool.shape[0]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    K, V = unpack(k_pool, hd, False).double(), unpack(v_pool, hd, True).double()
    sees = ancestors(parents, p).to(q.device)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    half = torch.finfo(q.dtype).eps / 2
    for b in range(n):
        base = int(pos[b])
        if base < 0:
            continue
        length = min(base + p, tables.shape[1] * PAGE)
        ids = tables[b, : -(-length // PAGE)].long()
        real = (ids >= 0) & (ids < pages)
        at = torch.arange(length, device=q.device)
        seen = (at.view(1, -1) < base) | (sees[:, (at - base).clamp(0, p - 1)] & (at >= base) & (at - base < p))
        seen = seen & real[at // PAGE]
        use = ids.clamp(0, pages - 1)
        k = K[use].transpose(1, 2).reshape(-1, nkv, hd)[:length]
        v = V[use].transpose(1, 2).reshape(-1, nkv, hd)[:length]
        for h in range(nh):
            kk, vv, qq = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)], q[b, :, h].double()
            x = (qq @ torch.nan_to_num(kk).T) * scale
            x = x.masked_fill(~seen, -math.inf)
            m = x.amax(1, keepdim=True)
            w = torch.where(seen, torch.exp(x - torch.where(m.isinf(), 0.0, m)), 0.0)
            l = w.sum(1, keepdim=True)
            clean = torch.where(vv.isfinite(), vv, 0.0)
            o = torch.where(l > 0, w @ clean / l, 0.0)
            # outputs that a value which is not finite reaches, from a position that the row sees
            hit = (seen.double() @ (~vv.isfinite()).double()) > 0
            out[b, :, h] = torch.where(hit, math.nan, o)
            # the exponent's error: f32 sums of hd products (truncated adds count double), the scale's two roundings,
            # the exponential's own; every weight carries it, numerator and denominator
            size = (qq.abs() @ torch.nan_to_num(kk).abs().T * scale * seen).amax(1, keepdim=True)
            delta = 2.0**-24 * (2 * hd + 16) * size + 2.0**-18
            spread = torch.where(l > 0, w @ clean.abs() / l, 0.0)  # sum p |v| / l
            tiny = 2.0**-25 * clean.abs().sum(0) if q.dtype == torch.float16 else 0.0  # f16 weights below 2^-14
            bound[b, :, h] = spread * (half + 2 * delta + 2 * length * 2.0**-24) + tiny + half * o.abs() * 1.01 + 2.0**-25
    return out, bound


def sample(logits: np.ndarray, u: float, temp: float, top_k: int, top_p: float, min_p: float):
    """(token, probability) of one row, float64 masses in the order's own definition; integers where they tie."""
    x = logits.astype(np.float32) + np.float32(0)
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float32)
    top = x.max()
    if top == -np.inf:
        return -1, 0.0
    if not temp > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore"):
        d = np.where(x == top, np.float32(0), x - top).astype(np.float32)
        e = np.where(np.isinf(d), 0.0, np.exp(np.where(np.isinf(d), 0.0, d.astype(np.float64)) / float(temp)))
    e = np.where(e < 2.0**-45, 0.0, e)
    order = np.lexsort((np.arange(len(x)), -d))
    count = len(x)
    if 0 < top_k < count:
        count = top_k
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(e[order])[:-1]])
        count = min(count, max(1, int(np.count_nonzero(before < max(top_p, 0.0) * e.sum()))))
    keep = np.zeros(len(x), bool)
    keep[order[:count]] = True
    if min_p > 0:
        keep &= e >= min(min_p, 1.0)
    keep &= e > 0
    index = np.flatnonzero(keep)
    mass = e[index]
    if np.all(mass == mass[0]):  # equal masses: the walk in exact arithmetic
        r = Fraction(min(max(u, 0.0), 1.0)) * len(index)
        at = min(int(r), len(index) - 1)
    else:
        cum = np.cumsum(mass)
        at = min(int(np.searchsorted(cum, u * cum[-1], side="right")), len(index) - 1)
    return int(index[at]), float(mass[at] / mass.sum())
