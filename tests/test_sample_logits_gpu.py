"""sample_logits on the GPU against the 64-bit form of its definition (tests/kv_reference.py)."""
import math

import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def sample():
    from clusterlm_b200.runtime import sample_logits

    return sample_logits


def check(ctx, sample, logits, u, temp=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = logits.shape[0]

    def column(x, dtype):
        return torch.as_tensor(np.broadcast_to(np.asarray(x), (rows,)).copy()).to(dtype).cuda()

    settings = dict(temperature=column(temp, F32), top_k=column(top_k, torch.int32), top_p=column(top_p, F32),
                    min_p=column(min_p, F32))
    tok, prob = sample(ctx, logits, u, with_probs=True, **settings)
    x, us = logits.float().cpu().numpy(), u.cpu().numpy()
    t, k, p, m = (settings[n].cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p"))
    for r in range(rows):
        want, pw = ref.sample(x[r], float(us[r]), float(t[r]), int(k[r]), float(p[r]), float(m[r]))
        assert int(tok[r]) == want, (r, int(tok[r]), want)
        # the f32 rounding of the probability, and the masses' (2^-45 of the largest each, 1e-12 relative)
        assert abs(float(prob[r]) - pw) <= pw * (2.0**-24 + 2e-12) + x.shape[1] * 2.0**-45 * pw + 1e-38, r
    return tok


def uniforms(rows, seed=0):
    return torch.rand(rows, dtype=torch.float64, generator=torch.Generator().manual_seed(seed)).cuda()


def gaussian(rows, vocab, seed=0, scale=3.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(rows, vocab, device="cuda", generator=g)).to(dtype)


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 64, 512, 1000, 4099, 32000, 128256, 151936])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=5), dict(top_p=0.8), dict(min_p=0.05),
                                dict(temp=0.7, top_k=40, top_p=0.95, min_p=0.01), dict(temp=0.0)])
def test_settings_over_vocabularies(ctx, sample, vocab, kw):
    rows = 12 if vocab < 10000 else 4
    check(ctx, sample, gaussian(rows, vocab, vocab), uniforms(rows, vocab), **kw)


def test_every_row_has_its_own_settings(ctx, sample):
    rng = np.random.default_rng(3)
    rows = 96
    check(ctx, sample, gaussian(rows, 5003, 3), uniforms(rows, 3), temp=rng.choice([0.0, 0.5, 1.0, 2.0], rows),
          top_k=rng.choice([-1, 0, 1, 3, 100, 4000, 10**6], rows), top_p=rng.choice([0.0, 1e-6, 0.3, 0.9, 0.999, 1.0, 2.0], rows),
          min_p=rng.choice([0.0, -1.0, 1e-4, 0.2, 1.0, 3.0], rows))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=300), dict(top_p=0.5), dict(top_p=0.97, top_k=20000), dict(temp=3.0, top_p=0.9)])
def test_16_bit_logits_tie(ctx, sample, dtype, kw):
    """Thousands of equal logits at the cut: the lowest indices stay."""
    check(ctx, sample, gaussian(3, 50001, 5, 2.0, dtype), uniforms(3, 5), **kw)


@pytest.mark.parametrize("vocab", [5, 2048, 30011])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=1), dict(top_k=2000), dict(top_p=0.3), dict(min_p=1.0), dict(temp=1e30, top_p=0.6)])
def test_equal_logits(ctx, sample, vocab, kw):
    """A flat row: the walk at exact fractions of the mass."""
    u = torch.tensor([0.0, 0.5, 1 / 3, 1 - 2.0**-53, 2.0**-1060, 0.1], dtype=torch.float64, device="cuda")
    logits = torch.full((6, vocab), -3.25, device="cuda")
    tok = check(ctx, sample, logits, u, **kw)
    assert int(tok[0]) == 0


def test_flat_rows_bisect_the_keys(ctx, sample):
    """More than a thousand distinct logits within one histogram bin."""
    g = torch.Generator(device="cuda").manual_seed(8)
    logits = 5.0 + 1e-3 * torch.rand(4, 60000, device="cuda", generator=g)
    logits[2:] = torch.round(logits[2:] * 2**14) / 2**14  # and with ties among them
    for kw in (dict(top_k=30000), dict(top_p=0.37), dict(top_k=20000, top_p=0.5, temp=0.8), dict(top_k=1), dict(top_p=1e-7)):
        check(ctx, sample, logits, uniforms(4, 8), **kw)


def test_one_entry_outweighs_thousands(ctx, sample):
    """The cut lies among entries whose whole mass is a rounding of the first one's: bounds on masses cannot find it."""
    g = torch.Generator(device="cuda").manual_seed(21)
    logits = torch.rand(5, 40000, device="cuda", generator=g) - 20.0
    logits[:, 17] = 0.0
    rest = float(torch.exp(logits[0].double()).sum() - 1.0)
    for part in (0.1, 0.5, 0.9, 0.999):
        p = np.float32((1.0 + part * rest) / (1.0 + rest))
        assert p < 1
        check(ctx, sample, logits, torch.tensor([0.0, 0.5, 1 - 1e-6, 1 - 1e-7, 1 - 2.0**-53], dtype=torch.float64).cuda(), top_p=p)


@pytest.mark.parametrize("rows", [1, 5, 64])
@pytest.mark.parametrize("spread", ["first eighth", "last sixteenth", "everywhere"])
def test_halving_with_uneven_slices(ctx, sample, rows, spread):
    """One entry outweighs thousands, several levels are halved by exact sums, and the parts of a row have unlike work: all the
    others in one part, so that the rest of the row's CTAs run ahead of it.  Every repetition gives the same tokens."""
    vocab = 48000
    first, last = {"first eighth": (0, vocab // 8), "last sixteenth": (vocab - vocab // 16, vocab), "everywhere": (0, vocab)}[spread]
    g = torch.Generator(device="cuda").manual_seed(31)
    logits = torch.full((rows, vocab), -math.inf, device="cuda")
    logits[:, first:last] = torch.rand(rows, last - first, device="cuda", generator=g) - 20.0
    logits[:, first + 11] = 0.0
    rest = float(torch.exp(logits[0].double()).sum() - 1.0)
    u = uniforms(rows, 31)
    u[::2] = 1 - 2.0**-53 * (1 + torch.arange(len(u[::2]), dtype=torch.float64, device="cuda"))
    for part in (0.03, 0.5, 0.98):
        p = np.float32((1.0 + part * rest) / (1.0 + rest))
        want = check(ctx, sample, logits, u, top_p=p)
        top_p = torch.full((rows,), float(p), device="cuda")
        for _ in range(50):
            assert torch.equal(sample(ctx, logits, u, top_p=top_p), want)


def test_masks_infinities_and_nan(ctx, sample):
    logits = gaussian(9, 3001, 6)
    logits[0] = -math.inf                       # nothing left
    logits[1] = math.nan
    logits[2] = -math.inf
    logits[2, 2999] = -80.0                     # one entry left
    logits[3] = torch.finfo(F32).min            # the type's lowest value everywhere
    logits[4] = torch.finfo(F32).min
    logits[4, [7, 70]] = 1.0                    # masked by the lowest value
    logits[5, [5, 500]] = math.inf              # only these count
    logits[6, ::2] = math.nan
    logits[7, 1::3] = -math.inf
    logits[8, :2000] = -math.inf
    for kw in (dict(), dict(top_k=2), dict(top_p=0.9), dict(min_p=0.1, top_k=50, top_p=0.9), dict(temp=0.0), dict(temp=1e-40),
               dict(temp=1e38, top_k=100)):
        tok = check(ctx, sample, logits, uniforms(9, 6), **kw)
        assert tok[:2].tolist() == [-1, -1]


def test_denormal_logits_at_a_denormal_temperature(ctx, sample):
    """Differences below 2^-126 with weights of every size, and more of them than a row ranks at once."""
    g = torch.Generator().manual_seed(3)
    steps = torch.randint(0, 4000, (3, 9000), generator=g)
    steps[:, :3000] %= 5  # thousands of equal ones near the top
    logits = (-steps.double() * 2.0**-149).float().cuda()
    for kw in (dict(temp=1e-42), dict(temp=1e-42, top_p=0.5), dict(temp=1e-42, top_p=0.9, top_k=4000), dict(temp=1e-43, top_p=0.99),
               dict(temp=1e-42, min_p=0.5, top_k=1500)):
        check(ctx, sample, logits, uniforms(3, 8), **kw)


def test_zeros_of_both_signs_are_one_value(ctx, sample):
    logits = torch.zeros(2, 100, device="cuda")
    logits[:, ::2] = -0.0
    for kw in (dict(temp=0.0), dict(top_k=3), dict()):
        check(ctx, sample, logits, torch.tensor([0.2, 0.7], dtype=torch.float64, device="cuda"), **kw)


def test_settings_that_are_not_numbers(ctx, sample):
    """NaN: temperature picks the maximum, top-p and min-p are off; uniforms outside [0, 1) take the first and last."""
    logits = gaussian(6, 700, 12)
    u = torch.tensor([0.3, 0.3, 0.3, math.nan, 1.5, -0.5], dtype=torch.float64, device="cuda")
    nan = float("nan")
    tok = sample(ctx, logits, u, temperature=torch.tensor([nan, 1, 1, 1, 1, 1.0]).cuda(),
                 top_p=torch.tensor([1, nan, 1, 1, 1, 1.0]).cuda(), min_p=torch.tensor([0, 0, nan, 0, 0, 0.0]).cuda())
    plain = sample(ctx, logits, u)
    assert int(tok[0]) == int(logits[0].argmax()) and tok[1:].tolist() == plain[1:].tolist()
    assert int(tok[3]) == int(tok[4] * 0 + 699) and int(tok[4]) == 699 and int(tok[5]) == 0


def test_views_with_padding_and_odd_starts(ctx, sample):
    for dtype in (F32, F16, BF16):
        wide = gaussian(5, 2003, 4, dtype=dtype)
        for view in (wide[:, :2000], wide[:, 1:1999], wide[1:, 3:]):
            u = uniforms(view.shape[0], 4)
            a = sample(ctx, view, u, top_p=0.9, with_probs=True)
            b = sample(ctx, view.contiguous(), u, top_p=0.9, with_probs=True)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        check(ctx, sample, wide[:, 1:1999], uniforms(5, 4), top_p=0.9, top_k=77)


def test_a_row_does_not_depend_on_its_batch(ctx, sample):
    logits, u = gaussian(300, 20000, 9), uniforms(300, 9)
    whole, pw = sample(ctx, logits, u, top_p=0.92, top_k=500, temperature=0.9, with_probs=True)
    for r in (0, 17, 150, 299):
        one, po = sample(ctx, logits[r:r + 1], u[r:r + 1], top_p=0.92, top_k=500, temperature=0.9, with_probs=True)
        assert int(one) == int(whole[r]) and float(po) == float(pw[r])


@pytest.mark.parametrize("vocab", [1, 130, 3001, 128256])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=7), dict(top_p=0.8), dict(min_p=0.03), dict(top_k=900, top_p=0.97),
                                dict(temperature=0.0), dict(temperature=2.5, top_p=0.99)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_rows_and_many_agree(ctx, sample, vocab, kw, dtype):
    """Rows alone, whose parts are halves of those that rows of a batch have."""
    logits, u = gaussian(24, vocab, 21, dtype=dtype), uniforms(24, 21)
    tok, prob = sample(ctx, logits, u, with_probs=True, **kw)
    for r in range(0, 24, 5):
        one, p = sample(ctx, logits[r:r + 2], u[r:r + 2], with_probs=True, **kw)
        assert torch.equal(one, tok[r:r + 2]) and torch.equal(p, prob[r:r + 2])
    check(ctx, sample, logits, u, **{"temp" if k == "temperature" else k: x for k, x in kw.items()})


def test_frequencies_follow_the_distribution(ctx, sample):
    """100,000 draws of a 12-token row: every token within 5 standard deviations of its share."""
    row = torch.tensor([[2.0, 1.5, 1.0, 0.5, 0.0, -0.5, -1.0, -2.0, -3.0, 1.9, 1.4, 0.9]], device="cuda")
    n = 100_000
    tok = sample(ctx, row.expand(n, 12).contiguous(), uniforms(n, 1), top_p=0.95, temperature=0.8)
    e = np.exp(row[0].double().cpu().numpy() / float(np.float32(0.8)))
    order = np.argsort(-e)
    count = int(np.count_nonzero(np.concatenate([[0], np.cumsum(e[order])[:-1]]) < float(np.float32(0.95)) * e.sum()))
    share = np.zeros(12)
    share[order[:count]] = e[order[:count]] / e[order[:count]].sum()
    got = np.bincount(tok.cpu().numpy(), minlength=12)
    assert np.all(np.abs(got - n * share) <= 5 * np.sqrt(n * share * (1 - share)))


def test_agrees_with_distribution_and_sample_from(ctx, sample):
    """The framework's two calls in one, where the uniform is not within a probability's f32 rounding of a border."""
    from clusterlm_b200.runtime import distribution, sample_from

    logits, u = gaussian(64, 4096, 2), uniforms(64, 2)
    for kw in (dict(), dict(top_k=30), dict(top_p=0.9)):
        probs = distribution(ctx, logits, 0.9, kw.get("top_k", 0), kw.get("top_p", 1.0))
        cum = torch.cumsum(probs.double(), 1)
        near = ((cum - u.view(-1, 1) * cum[:, -1:]).abs().amin(1) < 4096 * 2.0**-25)
        want = sample_from(ctx, probs, u)
        got = sample(ctx, logits, u, temperature=0.9, **kw)
        assert bool(((got == want) | near).all()) and int(near.sum()) < 16


def test_captured_and_on_two_streams(ctx, sample):
    logits, u = gaussian(20, 9000, 1), uniforms(20, 1)
    temp = torch.full((20,), 0.8, device="cuda")
    want = sample(ctx, logits, u, temperature=temp, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample(ctx, logits, u, temperature=temp, top_p=0.9)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    logits.copy_(gaussian(20, 9000, 2))
    temp.fill_(1.2)
    graph.replay()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = sample(ctx, logits, u, temperature=temp, top_p=0.9)
    torch.cuda.synchronize()
    assert torch.equal(got, again) and not torch.equal(got, want)


def test_refusals(ctx, sample):
    logits, u = gaussian(3, 100), uniforms(3)
    for args, kw in (((logits[0], u), {}), ((logits.double(), u), {}), ((logits.cpu(), u), {}), ((logits[:, ::2], u), {}),
                     ((logits.T, u), {}), ((logits, u.float()), {}), ((logits, u[:2]), {}), ((logits[:1].expand(3, 100), u), {}),
                     ((logits, u), dict(temperature=torch.ones(3, dtype=F16, device="cuda"))),
                     ((logits, u), dict(top_k=torch.ones(3, device="cuda"))),
                     ((logits, u), dict(top_p=torch.ones(2, device="cuda"))), ((logits, u), dict(min_p=torch.ones(3)))):
        with pytest.raises(ValueError):
            sample(ctx, *args, **kw)
    from clusterlm_b200._native import ClmError

    with pytest.raises(ClmError):
        sample(ctx, torch.zeros(1, 385025, device="cuda"), u[:1])
    assert sample(ctx, logits[:0], u[:0]).numel() == 0
