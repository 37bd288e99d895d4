"""Row sampling where neighbouring f32 logits lie hundreds of temperatures apart,
and at temperatures beyond every difference: the weights of exp((x - max) / T)
all the same.

A kept weight counts in whole units of 2^-43, rounded up by one at most, so the
masses of N kept tokens are off by N 2^-43 at most: the token is one whose share
of the mass reaches u, allowing that on either side, and its probability is its
weight over the mass, within that and two units of f32."""
import numpy as np
import pytest

from test_gpu_sample_rows import run
from tree_reference import rounded

pytestmark = pytest.mark.gpu

SETTINGS = [dict(), dict(p=0.9), dict(k=40, p=0.9), dict(k=700), dict(m=0.01), dict(k=3, m=0.2), dict(p=0.8, m=0.01)]


def kept_weights(x, t, k=0, p=1.0, m=0.0):
    """Weights of a row by index, 0 for what is not kept (settings as f32 values)."""
    t, p, m = (float(np.float32(a)) for a in (t, p, m))
    w = np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / t))
    order = np.argsort(-x, kind="stable")
    down = w[order]
    n = int((x > -np.inf).sum())
    if m > 0:
        n = int((down >= m).sum())
    if p < 1:
        mass = np.cumsum(down[:n])
        n = min(n, int((mass < p * mass[-1]).sum()) + 1)
    if k:
        n = min(n, k)
    out = np.zeros_like(w)
    out[order[:n]] = down[:n]
    return out, n


def check(torch, ctx, x, kind, t, u, **s):
    tok, prob, _ = run(torch, ctx, x, kind, t=t, u=u, **s)
    _, held = rounded(torch, x, kind)
    for r in range(x.shape[0]):
        w, n = kept_weights(held[r], t, **s)
        mass, slack = np.cumsum(w), (n + 1) * 2.0 ** -43
        i, place = int(tok[r]), float(np.float32(u if np.isscalar(u) else u[r])) * w.sum()
        assert 0 <= i < w.size and w[i] > 0, (s, r, i)
        assert mass[i] - w[i] <= place + slack and mass[i] + slack >= place, (s, r, i, place, mass[i])
        np.testing.assert_allclose(prob[r], w[i] / mass[-1], rtol=2.0 ** -22 + slack, atol=2.0 ** -149)


@pytest.mark.parametrize("size", [1e6, 2.0 ** 20, -1e6, 2e9])
@pytest.mark.parametrize("gap", [20.0, 80.0, 100.0, 400.0, 700.0, 745.05, 800.0, 1600.0])
def test_neighbours_many_temperatures_apart(fbctx, torch_cuda, size, gap):
    """The largest logits and the f32 numbers next below them, `gap` temperatures away."""
    rng = np.random.default_rng(int(gap))
    top = np.float32(size)
    below = np.nextafter(top, np.float32(-np.inf))
    x = np.full((4, 3000), float(below))
    x[0, [5, 2000]] = float(top)
    x[1, rng.permutation(3000)[:300]] = float(top)
    x[2, 2999] = float(top)
    x[3, rng.random(3000) < 0.5] = float(np.nextafter(below, np.float32(-np.inf)))
    x[3, 77] = float(top)
    t = float(np.float32((float(top) - float(below)) / gap))
    for s in SETTINGS:
        for u in (0.0, 0.5, 0.9999):
            check(torch_cuda, fbctx, x, "f32", t, u, **s)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("t", [1e28, 2e30, 3e33, 1e36, 3.4e38])
def test_temperatures_beyond_the_logits(fbctx, torch_cuda, kind, t):
    """Logits over the type's whole range (masks of its lowest value among them) and over a little of it."""
    torch = torch_cuda
    rng = np.random.default_rng(3)
    lowest = float(torch.finfo(torch.float32 if kind == "f32" else torch.bfloat16).min)
    x = rng.uniform(-3.3e38, 3.3e38, (5, 2500))
    x[1] = 3e36 * rng.normal(0, 1, 2500)
    x[2, 10:] = lowest
    x[3] = rng.normal(0, 1, 2500)
    x[3, ::2] = lowest
    x[4, ::3] = -np.inf
    for s in SETTINGS:
        check(torch, fbctx, x, kind, t, rng.random(5), **s)


@pytest.mark.parametrize("t", [1e-38, 1e-33, 1e-25])
def test_smallest_logits_and_temperatures(fbctx, torch_cuda, t):
    rng = np.random.default_rng(4)
    x = 5 * t * rng.normal(0, 1, (3, 2500))
    x[1, ::2] = -3.0
    x[2, 1::2] = -np.inf
    for s in SETTINGS:
        check(torch_cuda, fbctx, x, "f32", t, rng.random(3), **s)
