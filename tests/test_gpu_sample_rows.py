"""Row sampling from given random numbers against its definition in binary64:
the same token for every row (weights are exact to 2^-43 of the largest, the
seeded uniforms keep farther from every border), and its probability to two
units of f32."""
import numpy as np
import pytest

import ferrite_b200 as fb
from tree_reference import fb_type, rounded, sample, torch_type

pytestmark = pytest.mark.gpu


def run(torch, ctx, x, kind, t=None, k=None, p=None, m=None, u=None, stride=None, start=0):
    rows, vocab = x.shape
    stride = stride or vocab
    flat = np.full(start + rows * stride, 100.0)  # what lies between the rows is above every logit
    for r in range(rows):
        flat[start + r * stride:start + r * stride + vocab] = x[r]
    d, held = rounded(torch, flat, kind)
    held = np.stack([held[start + r * stride:start + r * stride + vocab] for r in range(rows)])

    def arr(a, dtype):
        return None if a is None else torch.from_numpy(np.broadcast_to(np.asarray(a, dtype), (rows,)).copy()).cuda()
    td, kd, pd, md, ud = arr(t, np.float32), arr(k, np.int32), arr(p, np.float32), arr(m, np.float32), arr(u, np.float32)
    tok = torch.full((rows + 1,), -9, dtype=torch.int32, device="cuda")
    prob = torch.full((rows + 1,), -9.0, device="cuda")
    ptr = lambda a: 0 if a is None else a.data_ptr()  # noqa: E731
    fb.sample_rows(ctx, fb_type(fb, kind), d.data_ptr() + start * d.element_size(), stride, rows, vocab, ptr(td), ptr(kd),
                   ptr(pd), ptr(md), ptr(ud), tok.data_ptr(), prob.data_ptr())
    torch.cuda.synchronize()
    assert int(tok[rows]) == -9 and float(prob[rows]) == -9.0
    assert ctx.error_word() == 0
    one = lambda a, r, off: off if a is None else float(a[r])  # noqa: E731
    want = [sample(held[r], one(td, r, 1.0), int(one(kd, r, 0)), one(pd, r, 1.0), one(md, r, 0.0), float(ud[r]))
            for r in range(rows)]
    return tok[:rows].cpu().numpy(), prob[:rows].cpu().numpy().astype(np.float64), want


def check(tok, prob, want):
    assert tok.tolist() == [w[0] for w in want]
    # 2^-149: the spacing of f32 next to zero, where a probability below 2^-126 is rounded by up to half of it
    np.testing.assert_allclose(prob, [w[1] for w in want], rtol=2.0 ** -22, atol=2.0 ** -149)


SETTINGS = [dict(), dict(p=0.9, m=0.05, t=0.7), dict(k=40), dict(p=0.95), dict(m=0.1, t=1.3), dict(k=100, p=0.8, m=0.02, t=1.5),
            dict(k=1), dict(t=0.0), dict(p=0.5, k=3, t=0.5), dict(k=10 ** 9, p=2.0, m=-1.0), dict(m=1.0), dict(m=7.0), dict(p=0.0),
            dict(p=-1.0), dict(t=0.004), dict(t=1e4), dict(t=np.inf), dict(p=0.999, t=2.0)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (5, 128256), (3, 4097), (2, 37), (4, 1), (40, 1001)])
def test_settings(fbctx, torch_cuda, kind, rows, vocab):
    rng = np.random.default_rng(rows + vocab)
    for s in SETTINGS:
        x = 2.5 * rng.normal(0, 1, (rows, vocab))
        x[rng.random((rows, vocab)) < 0.2] = -np.inf
        x[:, rng.integers(0, vocab)] = 3.0
        check(*run(torch_cuda, fbctx, x, kind, u=rng.random(rows), **s))


def test_settings_of_their_own(fbctx, torch_cuda):
    """A batch whose rows differ in every setting, NaN ones among them (off)."""
    rng = np.random.default_rng(1)
    rows = 64
    x = 2 * rng.normal(0, 1, (rows, 20000))
    t = rng.uniform(0.3, 2, rows).astype(np.float32)
    t[::5] = 0
    k = rng.integers(-2, 300, rows)
    p = rng.uniform(0.1, 1.3, rows).astype(np.float32)
    m = rng.uniform(-0.05, 0.3, rows).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    tok, prob, want = run(torch_cuda, fbctx, x, "f32", t, k, p, m, u)
    check(tok, prob, want)
    t[1], p[2], m[3], u[4] = np.nan, np.nan, np.nan, np.nan
    t2, p2, m2, u2 = t.copy(), p.copy(), m.copy(), u.copy()
    t2[1], p2[2], m2[3], u2[4] = 1.0, 1.0, 0.0, 0.0
    a, ap, _ = run(torch_cuda, fbctx, x, "f32", t, k, p, m, u)
    b, bp, _ = run(torch_cuda, fbctx, x, "f32", t2, k, p2, m2, u2)
    assert np.array_equal(a, b) and np.array_equal(ap, bp)


@pytest.mark.parametrize("vocab", [11, 3000, 151936])
def test_ties_and_ends(fbctx, torch_cuda, vocab):
    """Equal logits at the cut go to the lowest indices; u at both ends of its range and outside it."""
    rng = np.random.default_rng(vocab)
    x = np.round(rng.normal(0, 1, (1, vocab)))  # a handful of values
    flat = np.zeros((1, vocab))
    flat[0, 1::2] = -0.0
    for rows in (x, flat):
        for s in (dict(k=7), dict(p=0.3), dict(k=5, p=0.5), dict(p=0.2, m=0.5), dict(), dict(k=max(1, vocab // 2))):
            for u in (0.0, 0.37, 0.99999994, 1.0, 1.5, -0.5):
                check(*run(torch_cuda, fbctx, rows, "f32", u=u, **s))


def test_unusual_logits(fbctx, torch_cuda):
    torch = torch_cuda
    inf, nan = np.inf, np.nan
    base = np.random.default_rng(3).normal(0, 1, 500)
    rows = np.stack([base] * 8)
    rows[0, 100] = nan
    rows[1, ::2] = nan
    rows[2, [7, 300]] = inf
    rows[3, :] = -inf
    rows[4, :] = nan
    rows[5, :] = -inf
    rows[5, 77] = -3e38
    rows[6, [3, 4]] = [3.4e38, -3.4e38]
    rows[7, :] = nan
    rows[7, 499] = -inf
    for s in (dict(), dict(k=3, p=0.9), dict(t=0.0), dict(m=0.2), dict(t=0.01)):
        for u in (0.0, 0.6, 0.9999):
            check(*run(torch, fbctx, rows, "f32", u=u, **s))


@pytest.mark.parametrize("kind,start,gap", [("f32", 1, 0), ("f32", 0, 3), ("bf16", 1, 2), ("f16", 3, 1), ("f32", 0, 1000)])
def test_strides_and_alignment(fbctx, torch_cuda, kind, start, gap):
    rng = np.random.default_rng(start + gap)
    x = 2 * rng.normal(0, 1, (5, 7777))
    check(*run(torch_cuda, fbctx, x, kind, t=0.8, p=0.9, k=500, u=rng.random(5), stride=7777 + gap, start=start))


def test_largest_vocab(fbctx, torch_cuda):
    rng = np.random.default_rng(5)
    x = rng.normal(0, 1, (2, 1 << 19))
    for s in (dict(), dict(p=0.97), dict(k=30000), dict(p=0.5, t=3.0)):
        check(*run(torch_cuda, fbctx, x, "f32", u=rng.random(2), **s))


def test_frequencies_follow_the_weights(fbctx, torch_cuda):
    """Uniforms on a grid: each token's share of them is its probability, to one grid step."""
    torch = torch_cuda
    n, vocab = 4096, 50
    x = np.tile(np.linspace(-2, 2, vocab), (n, 1))
    u = (np.arange(n) + 0.5) / n
    tok, _, _ = run(torch, fbctx, x, "f32", u=u)
    p = np.exp(x[0].astype(np.float32).astype(np.float64))
    p /= p.sum()
    assert np.abs(np.bincount(tok, minlength=vocab) / n - p).max() <= 1.0 / n + 1e-7


def test_without_probabilities_and_in_a_graph(fbctx, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(6)
    x = torch.from_numpy(rng.normal(0, 2, (9, 30000)).astype(np.float32)).cuda()
    u = torch.from_numpy(rng.random(9).astype(np.float32)).cuda()
    p = torch.full((9,), 0.9, device="cuda")
    a = torch.zeros(9, dtype=torch.int32, device="cuda")
    b = torch.zeros(9, dtype=torch.int32, device="cuda")
    fb.sample_rows(fbctx, fb.F32, x.data_ptr(), 30000, 9, 30000, 0, 0, p.data_ptr(), 0, u.data_ptr(), a.data_ptr())
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    ctx = fb.Context(0, s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        fb.sample_rows(ctx, fb.F32, x.data_ptr(), 30000, 9, 30000, 0, 0, p.data_ptr(), 0, u.data_ptr(), b.data_ptr())
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, b) and (a >= 0).all()


@pytest.mark.parametrize("rows,vocab", [(6, 5000), (500, 3001)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_top_p_close_to_a_border(fbctx, torch_cuda, kind, rows, vocab):
    """top_p within 10^-6 of what the leading logits hold, on either side: an approximate mass cannot tell the cut."""
    torch = torch_cuda
    rng = np.random.default_rng(vocab)
    x = 2 * rng.normal(0, 1, (rows, vocab))
    x[:, ::7] = 2 * x[:, ::7] + rng.random((rows, 1))
    t = rng.uniform(0.5, 1.5, rows).astype(np.float32)
    _, held = rounded(torch, x, kind)
    p = np.empty(rows, np.float32)
    for r in range(rows):
        w = np.sort(np.exp((held[r] - held[r].max()) / float(t[r])))[::-1]
        at = int(rng.integers(2, 30))
        while w[at] == w[at + 1]:
            at += 1
        p[r] = np.float32(np.cumsum(w)[at] / w.sum() * (1 + (1e-6 if r % 2 else -1e-6)))
    for k in (50, None):
        check(*run(torch, fbctx, x, kind, t=t, k=k, p=p, u=np.full(rows, 0.9999)))


@pytest.mark.parametrize("size,t", [(4000.0, 0.1), (30000.0, 1.0), (3e8, 1e6), (1e30, 1e-8)])
def test_large_logits(fbctx, torch_cuda, size, t):
    """Logits far from zero in units of the temperature: what f32 loses of x / T must not move the cut."""
    rng = np.random.default_rng(7)
    x = size + 20 * t * rng.random((12, 3000))
    for s in (dict(k=40, p=0.9), dict(p=0.7), dict(p=0.99, k=200)):
        check(*run(torch_cuda, fbctx, x, "f32", t=t, u=rng.random(12), **s))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t", [1.0, 0.25, 1e-6])
def test_masks_of_the_lowest_value_and_infinities(fbctx, torch_cuda, kind, t):
    """Masked by the type's lowest value (whole threads' logits, or all but NaN and -inf), several infinite logits."""
    torch = torch_cuda
    lowest = torch.finfo(torch_type(torch, kind)).min
    rng = np.random.default_rng(8)
    x = 3 * rng.normal(0, 1, (6, 20011))
    x[0, 300:] = lowest
    x[1, :19000] = lowest
    x[2, :] = lowest
    x[3, :] = lowest
    x[3, ::3] = -np.inf
    x[3, 1::3] = np.nan
    x[4, [5, 600, 601, 9000, 20010]] = np.inf
    x[5, rng.random(20011) < 0.9] = lowest
    for s in (dict(k=40, p=0.9), dict(p=0.7), dict(p=0.35, k=400), dict(p=0.5, m=0.01)):
        check(*run(torch, fbctx, x, kind, t=t, u=rng.random(6), **s))


def test_equal_weights_share_a_border(fbctx, torch_cuda):
    """top_p times a number of equal logits that is whole keeps that many: few, many, infinite ones."""
    torch = torch_cuda
    for vocab, equal, value in ((64, 10, 5.0), (5000, 40, 1e3), (5000, 3000, 2.0), (200000, 1000, 7.0), (9000, 600, np.inf),
                                (9000, 4, np.inf)):
        x = np.full((3, vocab), -np.inf)
        x[:, np.random.default_rng(vocab).permutation(vocab)[:equal]] = value
        for s in (dict(p=0.5), dict(p=0.25, k=40), dict(p=0.75, m=0.5)):
            check(*run(torch, fbctx, x, "f32", u=[0.0, 0.5, 0.99999994], **s))


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (30, 20000), (500, 3001), (3, 700)])
def test_top_k_among_many_survivors_of_min_p(fbctx, torch_cuda, rows, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 1, (rows, vocab))
    x[:, ::5] = -np.inf
    x[rows // 2, 1:] = 0.25  # equal ones
    for s in (dict(k=1, m=0.02), dict(k=50, m=0.01, t=2.0), dict(k=256, m=1e-4), dict(k=257, m=0.001), dict(k=40, m=0.3, t=3.0),
              dict(k=20, m=0.01, p=0.5)):
        check(*run(torch_cuda, fbctx, x, "bf16", u=rng.random(rows), **s))
