"""min-p thresholds that lie next to 0, or where the weights near the maximum all
round to 1: the lowest logit whose weight reaches min_p, in binary64."""
import numpy as np
import pytest

from test_gpu_sample_rows import check, run
from tree_reference import rounded, sample

pytestmark = pytest.mark.gpu


def test_threshold_next_to_zero(fbctx, torch_cuda):
    """max + T ln(min_p) is 1.3e-15: its terms' rounding is a million f32 numbers there."""
    mx, t, m = 1.3482060432434082, 0.785749077796936, 0.17981573939323425
    assert abs(mx + t * np.log(m)) < 2e-15
    rng = np.random.default_rng(1)
    for vocab in (50, 3000, 60000):
        x = rng.choice([1e-3, -1e-3, 0.7, -2.0], (4, vocab))
        x[:, vocab // 3] = mx
        x[2, ::2] = -np.inf
        for s in (dict(), dict(k=20), dict(p=0.9), dict(k=300, p=0.99)):
            for u in (0.0, 0.4, 0.99999):
                check(*run(torch_cuda, fbctx, x, "f32", t=t, m=m, u=u, **s))


@pytest.mark.parametrize("t", [1e16, 1e20, 1e30, 3e38])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_weights_that_round_to_one(fbctx, torch_cuda, kind, t):
    """min_p within a rounding of the weights, which are 1 - d / T: exp in binary64 is off by one unit of 2^-53 of it at
    most on either side, so a logit whose weight lies within two of min_p may be kept or not.  The kept ones are the first n
    of the sorted row for some n that this allows, and everything else follows from n."""
    torch = torch_cuda
    rng = np.random.default_rng(2)
    x = rng.normal(0, 1, (3, 2000))
    x[1, ::3] = -np.inf
    if kind == "f32":
        x[2, ::5] = -1e36  # (weighs 1 at the highest of these temperatures only to 2^-9, nothing at the others)
    for s in (dict(m=1.0), dict(m=0.99999994), dict(m=1.0, k=700), dict(m=1.0, p=0.31)):
        u = rng.random(3)
        tok, prob, _ = run(torch, fbctx, x, kind, t=t, u=u, **s)
        _, held = rounded(torch, x, kind)
        for r in range(3):
            row, m = held[r], float(np.float32(s["m"]))
            w = np.exp((row - row.max()) / float(np.float32(t)))
            fewest, most = (int((w >= m * (1 + d * 2.0 ** -52)).sum()) for d in (1, -1))
            order = np.argsort(-row, kind="stable")
            allowed = []
            for n in range(max(fewest, 1), most + 1):
                kept = np.full_like(row, -np.inf)
                kept[order[:n]] = row[order[:n]]
                allowed.append(sample(kept, float(np.float32(t)), s.get("k", 0), float(np.float32(s.get("p", 1.0))), 0.0,
                                      float(np.float32(u[r]))))
            assert any(tok[r] == a and abs(prob[r] - b) <= 2.0 ** -22 * b for a, b in allowed), (s, r, tok[r], prob[r])
