"""Measured cases of the paged KV-cache operators and of sampling from logits.

`run` computes one pass of an operator: in its plain form (elementary torch operations) where `own` is false, through
the framework's public calls where it is true.  The inputs are the same on both sides: cache pools in the stored page
layout, page tables, positions, activations, logits, uniforms.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64  # positions per cache page
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


# --------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one session draws its next token from the 8B shape's vocabulary with everyday settings
        {"name": "sample-1x128256", "op": "sample", "rows": 1, "vocab": 128256, "pad": 0, "dtype": "f32", "temp": 0.8,
         "top_k": 50, "top_p": 0.95, "min_p": 0.0, "mixed": False, "masked": 0.0},
        # nucleus sampling of a batch at the acceptance workload's vocabulary
        {"name": "sample-64x151936-nucleus", "op": "sample", "rows": 64, "vocab": 151936, "pad": 0, "dtype": "f32",
         "temp": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "mixed": False, "masked": 0.0},
        # a serving batch: every row its own settings, some greedy, some unrestricted; padded rows; a grammar's mask
        {"name": "sample-256x128256-mixed", "op": "sample", "rows": 256, "vocab": 128256, "pad": 64, "dtype": "f32",
         "temp": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": True, "masked": 0.3},
        # the rows of 16 verify windows of 4 tokens enter the cache (8B shape)
        {"name": "append-16x4", "op": "append", "n": 16, "positions": 4, "nh": 32, "nkv": 8, "hd": 128, "ctx": 4096,
         "rot": 128, "interleaved": True, "src": "f16", "dtype": "f16", "tree": False},
        # a long prompt enters the cache from f32 activations (70B shape), half layout, part of the head rotated
        {"name": "append-1x4096-prompt", "op": "append", "n": 1, "positions": 4096, "nh": 64, "nkv": 8, "hd": 128,
         "ctx": 4000, "rot": 64, "interleaved": False, "src": "f32", "dtype": "bf16", "tree": False},
        # eight answers to one prompt: the sessions share its pages, each gets a copy of the last one (8B shape)
        {"name": "fork-8-of-4131", "op": "fork", "children": 8, "pos": 4131, "layers": 32, "nkv": 8, "hd": 128,
         "pages": 160, "dtype": "f16"},
        # a fragmented cache is packed: live pages move to the front and the tables follow
        {"name": "move-384-pages", "op": "move", "moves": 384, "layers": 10, "nkv": 8, "hd": 128, "pages": 1024,
         "seqs": 8, "dtype": "f16"},
        # four short forks decode one token each: latency
        {"name": "attend-4x1-1024", "op": "attend", "n": 4, "positions": 1, "nh": 32, "nkv": 8, "hd": 128,
         "groups": 1, "shared": 1024, "lo": 1, "hi": 90, "dtype": "f16", "tree": False},
        # eight sessions verify a 16-node draft tree each over one 4096-token prompt
        {"name": "attend-8x16-tree-4096", "op": "attend", "n": 8, "positions": 16, "nh": 32, "nkv": 8, "hd": 128,
         "groups": 1, "shared": 4096, "lo": 20, "hi": 300, "dtype": "f16", "tree": True},
        # 64 sessions with windows of 4 over a long common document, ragged own histories
        {"name": "attend-64x4-16384", "op": "attend", "n": 64, "positions": 4, "nh": 32, "nkv": 8, "hd": 128,
         "groups": 1, "shared": 16384, "lo": 100, "hi": 900, "dtype": "f16", "tree": False},
        # a chunk of 256 prompt rows against its own 8192-token context, nothing shared (70B shape)
        {"name": "attend-1x256-8192", "op": "attend", "n": 1, "positions": 256, "nh": 64, "nkv": 8, "hd": 128,
         "groups": 0, "shared": 0, "lo": 8100, "hi": 8200, "dtype": "bf16", "tree": False},
        # two prompts with 16 answers each, one token at a time, small heads
        {"name": "attend-2x16x1-hd64", "op": "attend", "n": 32, "positions": 1, "nh": 16, "nkv": 4, "hd": 64,
         "groups": 2, "shared": 8192, "lo": 33, "hi": 1500, "dtype": "bf16", "tree": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "append", "fork", "move", "attend", "attend"])
    if op == "sample":
        vocab = rng.choice([_log(rng, 300, 150000), 128256, 151936])
        rows = min(_log(rng, 1, 256), 30_000_000 // vocab)
        return {"op": op, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, 5, 64]),
                "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "temp": round(rng.uniform(0.3, 1.6), 3),
                "top_k": rng.choice([0, 0, _log(rng, 1, 2000)]), "top_p": rng.choice([1.0, round(rng.uniform(0.05, 0.99), 3)]),
                "min_p": rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), "mixed": rng.random() < 0.4,
                "masked": rng.choice([0.0, 0.5, 0.97])}
    if op == "append":
        hd = rng.choice([64, 128])
        positions = _log(rng, 1, 2048)
        n = max(1, min(_log(rng, 1, 64), 4096 // positions))
        nkv = rng.choice([1, 2, 4, 8])
        return {"op": op, "n": n, "positions": positions, "nh": nkv * rng.choice([1, 2, 4, 7, 8]), "nkv": nkv, "hd": hd,
                "ctx": _log(rng, 1, 200000 // n), "rot": rng.choice([hd, hd // 2, 24]),
                "interleaved": rng.random() < 0.5, "src": rng.choice(["f32", "f16", "bf16"]),
                "dtype": rng.choice(["f16", "bf16"]), "tree": positions <= 64 and rng.random() < 0.3}
    if op == "fork":
        return {"op": op, "children": _log(rng, 1, 32), "pos": _log(rng, 1, 6000), "layers": _log(rng, 1, 24),
                "nkv": rng.choice([1, 2, 8]), "hd": rng.choice([64, 128]), "pages": 160,
                "dtype": rng.choice(["f16", "bf16"])}
    if op == "move":
        return {"op": op, "moves": _log(rng, 1, 300), "layers": _log(rng, 1, 10), "nkv": rng.choice([1, 2, 8]),
                "hd": rng.choice([64, 128]), "pages": 640 + rng.randrange(200), "seqs": 1 + rng.randrange(12),
                "dtype": rng.choice(["f16", "bf16"])}
    groups = rng.choice([0, 1, 1, 2, 3])
    per = _log(rng, 1, 32)
    n = per * max(1, groups)
    positions = rng.choice([1, 1, 2, 4, 8, 1 + rng.randrange(16), _log(rng, 1, 256 // n) if n <= 256 else 1])
    nkv = rng.choice([1, 2, 4, 8])
    hi = _log(rng, 40, 6000 if groups == 0 and n <= 8 else 1200)
    return {"op": "attend", "n": n, "positions": positions, "nh": nkv * rng.choice([1, 3, 4, 8]), "nkv": nkv,
            "hd": rng.choice([64, 128, 128]), "groups": groups, "shared": PAGE * _log(rng, 1, 128) if groups else 0,
            "lo": rng.choice([0, hi // 3]), "hi": hi, "dtype": rng.choice(["f16", "bf16"]), "tree": rng.random() < 0.25}


# --------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _pools(g, layers, pages, nkv, hd, dtype):
    """K pages [64][hd] and V pages [hd][64] of every layer and kv head, in the stored layout (random values)."""
    k = torch.randn(layers, pages, nkv, PAGE, hd, generator=g, device=DEV, dtype=dtype)
    v = torch.randn(layers, pages, nkv, hd, PAGE, generator=g, device=DEV, dtype=dtype)
    return k, v


def _layout(hd):
    """Where the stored page keeps an element: K (position, dim) and V (position, dim) -> offset in the page."""
    pos = torch.arange(PAGE, device=DEV).view(PAGE, 1)
    dim = torch.arange(hd, device=DEV).view(1, hd)
    c = dim // 8
    kat = pos * hd + 8 * (c ^ (((c >> 3) & 1) << 1) ^ (pos & 1)) + dim % 8
    vat = dim * PAGE + 8 * ((pos // 8) ^ (dim & 1)) + pos % 8
    return kat, vat


def _tree(rng, p):
    return np.array([-1] + [int(rng.integers(max(-1, i - 5), i)) for i in range(1, p)], np.int32)


def _freqs(rot):
    """Rotary frequencies of a long-context model: the slow ones divided by 8, the middle ones blended."""
    f = 500000.0 ** (-np.arange(rot // 2) * 2.0 / rot)
    wave = 2 * math.pi / f
    smooth = np.clip((8192 / wave - 1.0) / (4.0 - 1.0), 0.0, 1.0)
    return (1 - smooth) * f / 8 + smooth * f


def prepare(case, seed):
    g, rng, op = _gen(seed), np.random.default_rng(seed), case["op"]
    s = {"case": case}
    if own:
        from clusterlm_b200.runtime import Context

        s["ctx"] = _context(Context)
    if op == "sample":
        rows, vocab, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
        full = _randn(g, rows, vocab + case["pad"], scale=3.0)
        if case["masked"]:
            full.masked_fill_(torch.rand(full.shape, generator=g, device=DEV) < case["masked"], -math.inf)
        full[:, min(3, vocab - 1)] = 2.5  # a token that every mask allows
        s["logits"] = full.to(dt)[:, :vocab]
        s["uniforms"] = torch.rand(rows, generator=g, device=DEV, dtype=torch.float64)
        temp, top_k = np.full(rows, case["temp"], np.float32), np.full(rows, case["top_k"], np.int32)
        top_p, min_p = np.full(rows, case["top_p"], np.float32), np.full(rows, case["min_p"], np.float32)
        if case["mixed"]:
            temp = rng.choice(np.array([0.0, 0.6, 0.8, 1.0, 1.3], np.float32), rows)
            top_k = rng.choice(np.array([0, 0, 1, 20, 50, 1000], np.int32), rows)
            top_p = rng.choice(np.array([1.0, 1.0, 0.5, 0.9, 0.95, 0.99], np.float32), rows)
            min_p = rng.choice(np.array([0.0, 0.0, 0.02, 0.1], np.float32), rows)
        for key, a in (("temp", temp), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
            s[key] = torch.from_numpy(a).to(DEV)
        return s
    dt = DTYPES[case["dtype"]]
    if op in ("fork", "move"):
        pages = case["pages"]
        s["k"], s["v"] = _pools(g, case["layers"], pages, case["nkv"], case["hd"], dt)
        ids = rng.permutation(pages)
        if op == "fork":
            need, c = case["pos"] // PAGE + 1, case["children"]
            tables = np.full((c + 2, need + 3), -1, np.int32)
            tables[1, :need] = ids[:need]
            pos = np.zeros(c + 2, np.int64)
            pos[1] = case["pos"]
            s["children"] = [i for i in range(c + 2) if i != 1][:c]
            s["new"] = [int(x) for x in ids[need:need + c]]
        else:
            m, n = case["moves"], case["seqs"]
            src, dst = np.sort(ids[:m]), np.sort(ids[m:2 * m])
            live = np.concatenate([src, ids[2 * m:]])
            tables = rng.choice(live, (n, 3 + pages // n)).astype(np.int32)
            tables[:, -2:] = -1
            pos = np.zeros(n, np.int64)
            s["src"], s["dst"] = [int(x) for x in src], [int(x) for x in dst]
        s["tables"], s["pos"] = torch.from_numpy(tables).to(DEV), torch.from_numpy(pos).to(DEV)
        return s
    n, p, nh, nkv, hd = (case[k] for k in ("n", "positions", "nh", "nkv", "hd"))
    if op == "append":
        pos = np.maximum(0, case["ctx"] - rng.integers(0, 70, n))
        shared, groups = 0, 0
    else:
        groups, shared = case["groups"], case["shared"] // PAGE
        pos = case["shared"] + rng.integers(case["lo"], case["hi"] + 1, n)
    last = (pos + p - 1) // PAGE  # the last page of each sequence
    first = pos // PAGE if op == "append" else np.full(n, shared)  # an append touches the pages of its rows only
    own_pages = last - first + 1
    total = n * ((p - 2) // PAGE + 2) + 3 if op == "append" else int(groups * shared + own_pages.sum()) + 3
    ids = rng.permutation(total).astype(np.int32)
    width = int(last.max()) + 2
    tables = np.full((n, width), -1, np.int32)
    at = groups * shared
    for b in range(n):
        if groups:
            k = b // (n // groups)
            tables[b, :shared] = ids[k * shared:(k + 1) * shared]
        tables[b, first[b]:last[b] + 1] = ids[at:at + own_pages[b]]
        at += int(own_pages[b])
    k, v = _pools(g, 1, total, nkv, hd, dt)
    s["k"], s["v"] = k[0], v[0]
    s["tables"], s["pos"] = torch.from_numpy(tables).to(DEV), torch.from_numpy(pos.astype(np.int64)).to(DEV)
    s["parents"] = torch.from_numpy(_tree(rng, p)).to(DEV) if case["tree"] else None
    if op == "append":
        src = DTYPES[case["src"]]
        qkv = _randn(g, n, p, nh + 2 * nkv, hd, dtype=src)  # one fused projection's output
        s["q"], s["kn"], s["vn"] = qkv[:, :, :nh], qkv[:, :, nh:nh + nkv], qkv[:, :, nh + nkv:]
        s["freqs"] = torch.from_numpy(_freqs(case["rot"])).to(DEV)
        if own:
            from clusterlm_b200.kv_cache import Rope

            s["rope"] = Rope(s["freqs"], interleaved=case["interleaved"], scale=1.1)
    else:
        s["q"] = _randn(g, n, p, nh, hd, dtype=dt, scale=1.5)
        s["groups"] = [(n // groups, shared)] * groups if groups else None
    return s


_kept = []


def _context(make):
    """The program's one context."""
    if not _kept:
        _kept.append(make(torch.cuda.current_device()))
    return _kept[0]


# --------------------------------------------------------------------------------------------------- plain forms
def _depths(parents, p):
    """Depth of every window row and which rows it sees: its ancestors and itself (a chain without parents)."""
    if parents is None:
        i = torch.arange(p, device=DEV)
        return i, i.view(p, 1) >= i.view(1, p)
    par = parents.long()
    up = torch.zeros(p + 1, p + 1, device=DEV)  # up[i, j]: j is i's parent; node p stands for "none"
    up[torch.arange(p, device=DEV), torch.where(par < 0, p, par)] = 1.0
    # (1 + up)^p has an entry wherever a chain of at most p steps leads from i to j
    sees = torch.linalg.matrix_power(torch.eye(p + 1, device=DEV, dtype=torch.float64) + up.double(), p)[:p, :p] > 0
    return sees.sum(1) - 1, sees


def _plain_sample(s):
    l = s["logits"].float()
    m = l.amax(1, keepdim=True)
    d = l - m
    t = s["temp"].double().view(-1, 1)
    e = torch.exp(d.double() / torch.where(t > 0, t, 1.0))
    order = torch.sort(d, dim=1, descending=True, stable=True).indices
    es = e.gather(1, order)
    cum = es.cumsum(1)
    rank = torch.arange(l.shape[1], device=DEV).view(1, -1)
    k = torch.where(s["top_k"] > 0, s["top_k"], l.shape[1]).view(-1, 1)
    k = torch.where(t > 0, k, 1)
    p = torch.where(s["top_p"] < 1, s["top_p"].double(), 2.0).view(-1, 1)
    keep = (rank < k) & (cum - es < p * cum[:, -1:]) & (es >= s["min_p"].double().clamp(max=1.0).view(-1, 1))
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    w = torch.where(kept, e, 0.0)
    cw = w.cumsum(1)
    r = s["uniforms"].view(-1, 1) * cw[:, -1:]
    past = (cw > r) & (w > 0)
    index = rank.expand_as(past)
    first = torch.where(past, index, l.shape[1]).amin(1)
    final = torch.where(w > 0, index, -1).amax(1)
    token = torch.where(first < l.shape[1], first, final)
    prob = w.gather(1, token.clamp(min=0).view(-1, 1)) / cw[:, -1:]
    return token.int(), prob.view(-1).float()


def _plain_append(s):
    case = s["case"]
    n, p, hd, rot = case["n"], case["positions"], case["hd"], case["rot"]
    depth, _ = _depths(s["parents"], p)
    at = (s["pos"].view(n, 1) + depth.view(1, p)).double()
    angle = at.view(n, p, 1, 1) * s["freqs"].view(1, 1, 1, rot // 2)
    cos, sin = (torch.cos(angle) * 1.1).float(), (torch.sin(angle) * 1.1).float()
    j = torch.arange(rot // 2, device=DEV)
    one, two = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + rot // 2)

    def turn(x):
        x = x.float()
        y = x.clone()
        y[..., one] = x[..., one] * cos - x[..., two] * sin
        y[..., two] = x[..., one] * sin + x[..., two] * cos
        return y.to(s["k"].dtype)

    q, k, v = turn(s["q"]), turn(s["kn"]), s["vn"].to(s["v"].dtype)
    slot = s["pos"].view(n, 1) + torch.arange(p, device=DEV)
    page = s["tables"].long().gather(1, slot // PAGE)
    kat, vat = _layout(hd)
    nkv = case["nkv"]
    head = (page.view(n, p, 1) * nkv + torch.arange(nkv, device=DEV)) * (PAGE * hd)
    inside = slot % PAGE
    s["k"].view(-1)[head.view(n, p, nkv, 1) + kat[inside].view(n, p, 1, hd)] = k
    s["v"].view(-1)[head.view(n, p, nkv, 1) + vat[inside].view(n, p, 1, hd)] = v
    return q, s["k"], s["v"]


def _plain_fork(s):
    kids = torch.tensor(s["children"], device=DEV)
    new = torch.tensor(s["new"], device=DEV)
    tables, pos = s["tables"], s["pos"]
    full = pos[1] // PAGE
    col = torch.arange(tables.shape[1], device=DEV).view(1, -1)
    row = torch.where(col < full, tables[1].view(1, -1), tables[kids])
    tables[kids] = torch.where(col == full, new.int().view(-1, 1), row)
    pos[kids] = pos[1].clone()
    last = tables[1].gather(0, full.view(1)).long()
    source = torch.where(pos[1] % PAGE > 0, last, new)
    s["k"][:, new] = s["k"][:, source]
    s["v"][:, new] = s["v"][:, source]
    return s["k"], s["v"], tables, pos


def _plain_move(s):
    src, dst = torch.tensor(s["src"], device=DEV), torch.tensor(s["dst"], device=DEV)
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    to = torch.arange(s["k"].shape[1], device=DEV, dtype=torch.int32)
    to[src] = dst.int()
    tables = s["tables"]
    return s["k"], s["v"], torch.where(tables >= 0, to[tables.clamp(min=0).long()], tables)


def _plain_attend(s):
    case = s["case"]
    n, p, nh, nkv, hd = (case[k] for k in ("n", "positions", "nh", "nkv", "hd"))
    kat, vat = _layout(hd)
    tables = s["tables"].clamp(min=0).long()
    length = tables.shape[1] * PAGE
    k = s["k"].view(-1, nkv, PAGE * hd)[:, :, kat.view(-1)].view(-1, nkv, PAGE, hd)[tables].float()
    v = s["v"].view(-1, nkv, PAGE * hd)[:, :, vat.view(-1)].view(-1, nkv, PAGE, hd)[tables].float()
    k = k.transpose(1, 2).reshape(n, nkv, length, hd)
    v = v.transpose(1, 2).reshape(n, nkv, length, hd)
    q = s["q"].float().view(n, p, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, hd)
    scores = (q @ k.transpose(2, 3)).view(n, nkv, -1, p, length) / math.sqrt(hd)
    _, sees = _depths(s["parents"], p)
    at = torch.arange(length, device=DEV).view(1, 1, length) - s["pos"].view(n, 1, 1)  # < 0: committed
    inside = sees.expand(n, p, p).gather(2, at.clamp(0, p - 1).expand(n, p, length))
    visible = (at < 0) | (inside & (at < p))
    scores = scores.masked_fill(~visible.view(n, 1, 1, p, length), -math.inf)
    scores = scores - scores.amax(-1, keepdim=True)
    w = torch.exp(scores)
    w = w / w.sum(-1, keepdim=True)
    o = (w.view(n, nkv, -1, length) @ v).view(n, nkv, nh // nkv, p, hd)
    return o.permute(0, 3, 1, 2, 4).reshape(n, p, nh, hd).to(s["q"].dtype)


def _no_tf32(f, s):
    """f(s) with float32 products in 32 bits."""
    before = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        return f(s)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = before


_PLAIN = {"sample": _plain_sample, "append": _plain_append, "fork": _plain_fork, "move": _plain_move,
          "attend": _plain_attend}


def run(state):
    op = state["case"]["op"]
    if not own:
        return _no_tf32(_PLAIN[op], state)
    s = state
    if op == "sample":
        from clusterlm_b200.runtime import sample_logits

        return sample_logits(s["ctx"], s["logits"], s["uniforms"], temperature=s["temp"], top_k=s["top_k"],
                             top_p=s["top_p"], min_p=s["min_p"], with_probs=True)
    from clusterlm_b200 import kv_cache

    if op == "append":
        q = kv_cache.kv_append(s["ctx"], s["k"], s["v"], s["tables"], s["pos"], s["q"], s["kn"], s["vn"],
                               rope=s["rope"], parents=s["parents"])
        return q, s["k"], s["v"]
    if op == "fork":
        kv_cache.kv_fork(s["ctx"], s["k"], s["v"], s["tables"], s["pos"], [1] * len(s["children"]), s["children"],
                         s["new"])
        return s["k"], s["v"], s["tables"], s["pos"]
    if op == "move":
        kv_cache.kv_copy_pages(s["ctx"], s["k"], s["v"], s["src"], s["dst"], tables=s["tables"])
        return s["k"], s["v"], s["tables"]
    return kv_cache.kv_attention(s["ctx"], s["k"], s["v"], s["tables"], s["pos"], s["q"], groups=s["groups"],
                                 parents=s["parents"])


# --------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZES[case["dtype"]] + case["rows"] * 32, "flops": 4 * n}
    hd = case["hd"]
    page = case["nkv"] * PAGE * hd * 2
    if op == "fork":
        copied = case["children"] if case["pos"] % PAGE else 0
        return {"bytes": 2 * 2 * case["layers"] * copied * page + case["children"] * (case["pos"] // PAGE + 3) * 8,
                "flops": 0}
    if op == "move":
        return {"bytes": 2 * 2 * case["layers"] * case["moves"] * page + 8 * (case["pages"] + 3 * case["seqs"]), "flops": 0}
    rows, nh, nkv = case["n"] * case["positions"], case["nh"], case["nkv"]
    if op == "append":
        values = rows * (nh + 2 * nkv) * hd
        return {"bytes": values * (SIZES[case["src"]] + 2), "flops": 3 * rows * (nh + nkv) * case["rot"]}
    private = (case["lo"] + case["hi"]) / 2 + (case["positions"] + 1) / 2
    seen = case["shared"] + private
    cached = case["groups"] * case["shared"] + case["n"] * private
    return {"bytes": 2 * 2 * nkv * hd * cached + 2 * 2 * rows * nh * hd, "flops": 4 * hd * nh * rows * seen}


# --------------------------------------------------------------------------------------------------- 64 bits
def _page_rows(pool, hd, transposed):
    """A pool's pages as (page, head, position, dim), read element by element from the stored layout, in 64 bits."""
    at = np.empty((PAGE, hd), np.int64)
    for pos in range(PAGE):
        for dim in range(hd):
            if transposed:
                at[pos, dim] = dim * PAGE + 8 * ((pos >> 3) ^ (dim & 1)) + (pos & 7)
            else:
                chunk = dim >> 3
                at[pos, dim] = pos * hd + 8 * (chunk ^ (2 if chunk >= 8 else 0) ^ (pos & 1)) + (dim & 7)
    return pool.reshape(pool.shape[0], pool.shape[1], -1)[..., torch.from_numpy(at).to(DEV).view(-1)].view(
        pool.shape[0], pool.shape[1], PAGE, hd), at


def _walk(parents, p):
    """Every window row's chain of window rows, itself first."""
    chains = []
    for i in range(p):
        chain = [i]
        while True:
            up = chain[-1] - 1 if parents is None else int(parents[chain[-1]])
            if up < 0:
                break
            chain.append(up)
        chains.append(chain)
    return chains


def _exact_sample(s):
    logits = s["logits"].float().cpu().numpy()
    u, temp, top_k, top_p, min_p = (s[k].cpu().numpy() for k in ("uniforms", "temp", "top_k", "top_p", "min_p"))
    tokens, probs = np.empty(len(u), np.int32), np.empty(len(u), np.float64)
    for r in range(len(u)):
        row = logits[r]
        top = row.max()
        d = row - top
        if temp[r] <= 0:
            tokens[r], probs[r] = int(np.argmax(row)), 1.0
            continue
        e = np.exp(d.astype(np.float64) / float(temp[r]))
        keep = e >= min(float(min_p[r]), 1.0)
        if top_k[r] > 0 or top_p[r] < 1:
            order = np.argsort(-d, kind="stable")
            count = len(row) if top_k[r] <= 0 else min(len(row), int(top_k[r]))
            if top_p[r] < 1:
                mass = np.cumsum(e[order])
                count = min(count, int(np.searchsorted(mass, float(top_p[r]) * mass[-1])) + 1)
            among = np.zeros(len(row), bool)
            among[order[:count]] = True
            keep &= among
        index = np.flatnonzero(keep & (e > 0))
        mass = np.cumsum(e[index])
        at = min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), len(index) - 1)
        tokens[r], probs[r] = index[at], e[index[at]] / mass[-1]
    return tokens, probs


def _exact_append(s):
    case = s["case"]
    n, p, hd, rot, nkv = case["n"], case["positions"], case["hd"], case["rot"], case["nkv"]
    chains = None if s["parents"] is None else _walk(s["parents"].cpu().numpy(), p)
    depth = np.arange(p) if chains is None else np.array([len(c) - 1 for c in chains])
    at = s["pos"].cpu().numpy()[:, None] + depth[None]
    angle = torch.from_numpy(at[..., None].astype(np.float64) * s["freqs"].cpu().numpy()).to(DEV)
    turn = torch.polar(torch.full_like(angle, 1.1), angle)[:, :, None, :]

    def rotated(x):
        x = x.double()
        part = x[..., :rot]
        if case["interleaved"]:
            z = torch.view_as_complex(part.reshape(*part.shape[:-1], rot // 2, 2).contiguous()) * turn
            part = torch.view_as_real(z).reshape(part.shape)
        else:
            z = torch.complex(part[..., :rot // 2], part[..., rot // 2:]) * turn
            part = torch.cat([z.real, z.imag], -1)
        return torch.cat([part, x[..., rot:]], -1)

    q, k, v = rotated(s["q"]), rotated(s["kn"]), s["vn"].double()
    _, kat = _page_rows(s["k"][:1], hd, False)
    _, vat = _page_rows(s["v"][:1], hd, True)
    kat, vat = torch.from_numpy(kat).to(DEV), torch.from_numpy(vat).to(DEV)
    out_k = s["k"].double().view(s["k"].shape[0], nkv, -1)
    out_v = s["v"].double().view(s["v"].shape[0], nkv, -1)
    tables, pos = s["tables"].cpu().numpy(), s["pos"].cpu().numpy()
    for b in range(n):
        slots = pos[b] + np.arange(p)
        for page in np.unique(slots // PAGE):
            rows = np.flatnonzero(slots // PAGE == page)
            inside = torch.from_numpy(slots[rows] % PAGE).to(DEV)
            out_k[int(tables[b, page])][:, kat[inside]] = k[b, rows[0]:rows[-1] + 1].transpose(0, 1)
            out_v[int(tables[b, page])][:, vat[inside]] = v[b, rows[0]:rows[-1] + 1].transpose(0, 1)
    return q, out_k.view(s["k"].shape), out_v.view(s["v"].shape)


def _exact_attend(s):
    case = s["case"]
    n, p, nh, nkv, hd = (case[k] for k in ("n", "positions", "nh", "nkv", "hd"))
    chains = _walk(None if s["parents"] is None else s["parents"].cpu().numpy(), p)
    mask = torch.zeros(p, p, dtype=torch.bool)
    for i, chain in enumerate(chains):
        mask[i, chain] = True
    mask = mask.to(DEV)
    kp, vp = _page_rows(s["k"], hd, False)[0], _page_rows(s["v"], hd, True)[0]
    pos, out = s["pos"].tolist(), torch.empty(n, p, nh, hd, dtype=torch.float64, device=DEV)
    for b in range(n):
        length = pos[b] + p
        pages = s["tables"][b, :-(-length // PAGE)].long()
        k = kp[pages].double().permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :length]
        v = vp[pages].double().permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :length]
        see = torch.cat([torch.ones(p, pos[b], dtype=torch.bool, device=DEV), mask], 1)
        for h in range(nh):
            kv = h // (nh // nkv)
            x = (s["q"][b, :, h].double() @ k[kv].T) / math.sqrt(hd)
            out[b, :, h] = torch.softmax(x.masked_fill(~see, -math.inf), -1) @ v[kv]
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "sample":
        return _exact_sample(s)
    if op == "append":
        return _exact_append(s)
    if op == "attend":
        return _exact_attend(s)
    return None  # forks and moves copy bits: nothing is computed
