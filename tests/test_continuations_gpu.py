"""The paged-cache operators and sampling together, as a decoder uses them: a prompt enters the cache, several continuations
are forked from it, each step appends a row, attends with the prompt's pages shared, and draws the next token."""
import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
PAGE, NH, NKV, HD, LAYERS, VOCAB = 64, 4, 2, 64, 2, 1000
PROMPT, CHILDREN, STEPS, PAGES = 150, 4, 60, 40


def mm(x, w):
    """x @ w by elementary operations, whose order does not depend on where they run."""
    return (x.unsqueeze(-1) * w).sum(-2)


class Decoder:
    """Two layers of projections around the operators; sequence 0 is the prompt, 1.. its continuations."""

    def __init__(self, ctx, kv, sample):
        g = torch.Generator(device="cuda").manual_seed(11)
        h = NH * HD

        def mat(*shape, scale):
            return torch.randn(*shape, device="cuda", generator=g) * scale

        self.ctx, self.kv, self.sample = ctx, kv, sample
        self.embed, self.head = mat(VOCAB, h, scale=1.0), mat(h, VOCAB, scale=0.2)
        self.qkv = [mat(h, (NH + 2 * NKV) * HD, scale=h**-0.5) for _ in range(LAYERS)]
        self.wo = [mat(h, h, scale=h**-0.5) for _ in range(LAYERS)]
        freqs, factor = kv.rope_frequencies(HD, 10000.0)
        self.rope = kv.Rope(torch.from_numpy(freqs).cuda(), interleaved=False, scale=factor)
        self.k = torch.zeros(LAYERS, PAGES, NKV, PAGE, HD, device="cuda", dtype=F16)
        self.v = torch.zeros(LAYERS, PAGES, NKV, HD, PAGE, device="cuda", dtype=F16)
        self.tables = torch.full((1 + CHILDREN, 8), -1, dtype=torch.int32, device="cuda")
        self.pos = torch.full((1 + CHILDREN,), -1, dtype=torch.int64, device="cuda")
        self.ledger = kv.Pages(PAGES)
        self.prompt = torch.randint(0, VOCAB, (PROMPT,), device="cuda", generator=g)
        self.uniforms = torch.rand(STEPS + 1, CHILDREN, device="cuda", dtype=torch.float64, generator=g)
        self.settings = dict(temperature=torch.tensor([0.7, 1.0, 0.0, 1.3], device="cuda"),
                             top_k=torch.tensor([0, 40, 0, 5], dtype=torch.int32, device="cuda"),
                             top_p=torch.tensor([0.9, 1.0, 1.0, 0.8], device="cuda"),
                             min_p=torch.tensor([0.0, 0.02, 0.0, 0.0], device="cuda"))

    def layers(self, rows, tables, pos, groups, verify):
        """Logits (n, VOCAB) of the last of each sequence's rows (n, p)."""
        x = self.embed[rows]
        n, p, h = x.shape
        for li in range(LAYERS):
            qkv = mm(x, self.qkv[li]).half().view(n, p, NH + 2 * NKV, HD)
            q, k, v = qkv[:, :, :NH], qkv[:, :, NH:NH + NKV], qkv[:, :, NH + NKV:]
            if verify:
                _, K, V = ref.append(self.k[li], self.v[li], tables.cpu(), pos.cpu(), None, k, v, self.rope.inv_freq, False,
                                     self.rope.scale)
            q = self.kv.kv_append(self.ctx, self.k[li], self.v[li], tables, pos, q, k, v, rope=self.rope)
            o = self.kv.kv_attention(self.ctx, self.k[li], self.v[li], tables, pos, q, groups=groups)
            if verify:
                # one rounding to fp16, and four f32 roundings of terms below 16
                assert bool(((self.k[li].double() - K).abs() <= K.abs() * 2**-11 + 2**-18).all())
                assert torch.equal(self.v[li].double(), V)
                want, bound = ref.attention(self.k[li], self.v[li], tables, pos, q)
                assert bool(((o.double() - want).abs() <= bound).all())
            x = x + mm(o.float().view(n, p, h), self.wo[li])
        return mm(x[:, -1], self.head)

    def draw(self, logits, u, verify):
        tok = self.sample(self.ctx, logits, u, **self.settings)
        if verify:
            s = {n: t.cpu().numpy() for n, t in self.settings.items()}
            for r in range(CHILDREN):
                want, _ = ref.sample(logits[r].cpu().numpy(), float(u[r]), float(s["temperature"][r]), int(s["top_k"][r]),
                                     float(s["top_p"][r]), float(s["min_p"][r]))
                assert int(tok[r]) == want
        return tok

    def start(self, verify=False):
        """The prompt, the forks, and the continuations' first tokens; every page that the run needs is in the tables."""
        need = PROMPT // PAGE + 1
        own = self.ledger.alloc(need)
        self.tables[0, :need] = torch.tensor(own, dtype=torch.int32)
        self.pos[0] = 0
        logits = self.layers(self.prompt.view(1, -1), self.tables[:1], self.pos[:1], None, verify)
        self.pos[0] = PROMPT
        full, last = PROMPT // PAGE, (PROMPT + STEPS) // PAGE
        pages = self.ledger.alloc(CHILDREN)
        for _ in range(CHILDREN):
            self.ledger.retain(own[:full])
        self.kv.kv_fork(self.ctx, self.k, self.v, self.tables, self.pos, [0] * CHILDREN, range(1, 1 + CHILDREN), pages)
        self.held = [own[:full] + [page] for page in pages]
        for c in range(CHILDREN):
            more = self.ledger.alloc(last - full)
            self.tables[1 + c, full + 1:last + 1] = torch.tensor(more, dtype=torch.int32)
            self.held[c] += more
        self.groups = [(CHILDREN, full)]
        self.tokens = self.draw(logits.expand(CHILDREN, -1).contiguous(), self.uniforms[0], verify).long()

    def step(self, u, verify=False):
        logits = self.layers(self.tokens.view(-1, 1), self.tables[1:], self.pos[1:], self.groups, verify)
        self.pos[1:].add_((self.pos[1:] >= 0).long())
        self.tokens.copy_(self.draw(logits, u, verify))


@pytest.fixture(scope="module")
def parts():
    from clusterlm_b200 import kv_cache
    from clusterlm_b200.runtime import sample_logits

    return kv_cache, sample_logits


def run(d, hook=None):
    out = [d.tokens.tolist()]
    for i in range(1, STEPS + 1):
        d.step(d.uniforms[i])
        if hook:
            hook(i)
        out.append(d.tokens.tolist())
    return out


def test_each_step_follows_the_formulas(ctx, parts):
    d = Decoder(ctx, *parts)
    d.start(verify=True)
    for i in range(1, STEPS + 1):
        d.step(d.uniforms[i], verify=True)
    assert d.pos.tolist() == [PROMPT] + [PROMPT + STEPS] * CHILDREN


def test_replayed_steps_equal_eager_ones(ctx, parts):
    a, b = Decoder(ctx, *parts), Decoder(ctx, *parts)
    a.start(), b.start()
    want = run(a)
    assert len({tuple(row) for row in zip(*want)}) > 1  # the continuations part
    u = b.uniforms[1].clone()
    k, v, pos, tokens = b.k.clone(), b.v.clone(), b.pos.clone(), b.tokens.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step(u)  # (the first call sets the kernels' attributes)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step(u)
    b.k.copy_(k), b.v.copy_(v), b.pos.copy_(pos), b.tokens.copy_(tokens)
    got = [b.tokens.tolist()]
    for i in range(1, STEPS + 1):
        u.copy_(b.uniforms[i])
        graph.replay()
        got.append(b.tokens.tolist())
    assert got == want
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.pos, b.pos)


def test_moved_pages_change_nothing(ctx, parts):
    a, b = Decoder(ctx, *parts), Decoder(ctx, *parts)
    a.start(), b.start()
    want = run(a)

    def hook(i):
        if i == 7:  # a continuation ends, its pages come back, and the others move down
            b.pos[2] = -1
            b.ledger.release(b.held[1])
            src, dst = b.ledger.compact()
            assert len(src) > 0
            b.kv.kv_copy_pages(ctx, b.k, b.v, src, dst, tables=b.tables)

    got = run(b, hook)
    keep = [0, 2, 3]
    assert [[row[c] for c in keep] for row in got] == [[row[c] for c in keep] for row in want]
    assert b.pos.tolist() == [PROMPT, PROMPT + STEPS, -1, PROMPT + STEPS, PROMPT + STEPS]


def test_a_captured_fork_reads_positions_and_tables_when_it_runs(ctx, parts):
    kv, _ = parts
    k = torch.randn(LAYERS, 12, NKV, PAGE, HD, device="cuda").half()
    v = torch.randn(LAYERS, 12, NKV, HD, PAGE, device="cuda").half()
    tables = torch.tensor([[0, 1, 2], [9, 9, 9], [9, 9, 9]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([70, 0, 0], device="cuda")
    kv.kv_fork(ctx, k, v, tables, pos, [0], [1], [5])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.kv_fork(ctx, k, v, tables, pos, [0, 0], [1, 2], [5, 6])
        kv.kv_copy_pages(ctx, k, v, [6], [7], tables=tables)
    for p, page in ((70, 1), (130, 2), (64, 1)):
        pos[0] = p
        tables[0] = torch.tensor([3, 4, 8]) if p == 130 else torch.tensor([0, 1, 2])
        source = int(tables[0, p // PAGE])
        k.normal_(), v.normal_()
        K, V = k.clone(), v.clone()
        graph.replay()
        if p % PAGE:
            for to in (5, 6):
                K[:, to], V[:, to] = K[:, source], V[:, source]
        K[:, 7], V[:, 7] = K[:, 6], V[:, 6]
        assert torch.equal(k, K) and torch.equal(v, V)
        assert pos.tolist() == [p] * 3
        n = p // PAGE
        assert tables[1, :n + 1].tolist() == tables[0, :n].tolist() + [5]
        assert tables[2, :n + 1].tolist() == tables[0, :n].tolist() + [7]


def test_pools_past_32_bit_offsets(ctx, parts):
    """Pages whose elements lie past 2^32 (and 2^32 bytes), and the last page of the widest table."""
    kv, _ = parts
    nkv, hd = 8, 128
    pages = 2**32 // (nkv * PAGE * hd) + 40
    if torch.cuda.mem_get_info()[0] < 5 * pages * nkv * PAGE * hd:
        pytest.skip("needs 22 GB of device memory")
    k = torch.empty(1, pages, nkv, PAGE, hd, device="cuda", dtype=F16)
    v = torch.empty(1, pages, nkv, hd, PAGE, device="cuda", dtype=F16)
    ids = [pages - 1 - i for i in range(8)]
    k[0, ids], v[0, ids] = (torch.randn(8, *t.shape[2:], device="cuda").half() for t in (k, v))

    def small():  # the same pages as a small pool: entry i is page ids[i]
        return k[0, ids].clone(), v[0, ids].clone()

    tables = torch.tensor([[ids[0], ids[1], ids[2]], [ids[0], ids[3], -1]], dtype=torch.int32, device="cuda")
    local = torch.tensor([[0, 1, 2], [0, 3, -1]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([140, 80], device="cuda")
    q, kn, vn = (torch.randn(2, 3, h, hd, device="cuda").half() for h in (16, nkv, nkv))
    K, V = small()
    kv.kv_append(ctx, K, V, local, pos, None, kn, vn)
    kv.kv_append(ctx, k[0], v[0], tables, pos, None, kn, vn)
    assert torch.equal(k[0, ids], K) and torch.equal(v[0, ids], V)
    for rows in (1, 3):  # 2 rows per kv head: the stream kernel; 54: the tile kernel
        qq = q[:, :rows].repeat(1, 1, rows * rows, 1)
        want = kv.kv_attention(ctx, K, V, local, pos, qq, groups=[(2, 1)])
        got = kv.kv_attention(ctx, k[0], v[0], tables, pos, qq, groups=[(2, 1)])
        assert torch.equal(got, want)
        out, bound = ref.attention(K, V, local, pos, qq)
        assert bool(((got.double() - out).abs() <= bound).all())
    t2, p2 = torch.full((2, 3), -1, dtype=torch.int32, device="cuda"), torch.tensor([140, 0], device="cuda")
    t2[0] = tables[0]
    kv.kv_fork(ctx, k, v, t2, p2, [0], [1], [ids[5]])
    kv.kv_copy_pages(ctx, k, v, [ids[1]], [ids[6]], tables=t2)
    assert torch.equal(k[0, ids[5]], K[2]) and torch.equal(v[0, ids[5]], V[2])
    assert torch.equal(k[0, ids[6]], K[1]) and torch.equal(v[0, ids[6]], V[1])
    assert t2.tolist() == [[ids[0], ids[6], ids[2]], [ids[0], ids[6], ids[5]]]
    # the widest table's last page
    far = 2**31 - PAGE + 5
    wide = torch.full((1, far // PAGE + 1), -1, dtype=torch.int32, device="cuda")
    wide[0, -1] = ids[7]
    kv.kv_append(ctx, k[0], v[0], wide, torch.tensor([far], device="cuda"), None, kn[:1, :1], vn[:1, :1])
    K, V = small()
    assert torch.equal(ref.unpack(K, hd, False)[7, :, far % PAGE], kn[0, 0])
    assert torch.equal(ref.unpack(V, hd, True)[7, :, far % PAGE], vn[0, 0])


def test_append_and_fork_on_another_stream(ctx, parts):
    """Operands that a side stream still computes, and results that it reads."""
    kv, _ = parts
    k, v = (torch.zeros(1, 4, 1, PAGE, PAGE, device="cuda", dtype=F16) for _ in range(2))
    tables = torch.tensor([[0, 1], [2, 2]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([60, 0], device="cuda")
    rows = torch.zeros(1, 8, 1, PAGE, device="cuda", dtype=F16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        busy = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            busy = busy @ busy * 1e-2
        rows.copy_(torch.arange(PAGE, device="cuda").expand(1, 8, 1, PAGE))
        kv.kv_append(ctx, k[0], v[0], tables[:1], pos[:1], None, rows, rows)
        pos[0] += 8
        kv.kv_fork(ctx, k, v, tables, pos, [0], [1], [3])
        K, V, T, P = k.clone(), v.clone(), tables.clone(), pos.clone()
    side.synchronize()
    want = torch.arange(PAGE, device="cuda").half().expand(4, PAGE)
    for page in (1, 3):
        assert torch.equal(ref.unpack(K[0], PAGE, False)[page, 0, :4], want)
        assert torch.equal(ref.unpack(V[0], PAGE, True)[page, 0, :4], want)
    assert torch.equal(ref.unpack(K[0], PAGE, False)[0, 0, 60:], want)
    assert T.tolist() == [[0, 1], [0, 3]] and P.tolist() == [68, 68]
