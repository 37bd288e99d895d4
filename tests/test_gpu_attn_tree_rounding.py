"""Tree attention of 16-bit types is off by its results' rounding and little else.

Before the rounding a result is as f32's, 4e-6 in the 2-norm, plus what the tensor
core truncates of its sums (2^-25 of them at each of 8 instructions a block of 64
keys, half of that on average over a growing sum): 1.9e-6 for the 16 blocks here,
D = 6e-6 together.  An element that is off by d before the rounding lands on the
other side of it with probability d / step, and then a step away: the rounded
results differ from the rounded exact ones by sum(step d) in the squared 2-norm, at
most 2 half-steps D of the results' own squares.  1.5 times its root is allowed (a
probability of 11 bits alone makes it some 3 times).

bf16 calls keep 11 bits of a probability: 2^-11 of it at most, as independent errors
0.42 of that (the error of a rounding, uniform over a step and its place in the
binade), an eighth of the results' own 0.42 of 2^-8: together sqrt(1 + 2^-6) = 1.008
times those.  1.015 times is allowed."""
import math

import numpy as np
import pytest

from test_gpu_attn_tree import Call
from tree_reference import HALF_STEP, Batch, attention, rounded, tree_mask

pytestmark = pytest.mark.gpu

D = 6e-6


@pytest.mark.parametrize("new,lens,qheads,dim,page", [
    ([25, 9, 14], [1000, 350, 700], 8, 128, 64),   # one tile a kv head, blocks in turn
    ([60, 50], [1000, 1024], 8, 128, 32),          # two tiles
    ([3] * 6, [900] * 6, 16, 64, 64),
])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_results_are_rounded_once(fbctx, torch_cuda, kind, new, lens, qheads, dim, page):
    torch = torch_cuda
    rng = np.random.default_rng(len(new) + dim)
    B = Batch(rng, new, lens, 2, dim, page)
    mask = tree_mask(rng, new, 2)
    qd, q = rounded(torch, 1.5 * rng.normal(0, 1, (B.total, qheads, dim)), kind)
    scale = 1 / math.sqrt(dim)
    got = Call(torch, fbctx, B, qd, mask, kind, qheads, words=2).result(scale)
    exact = attention(q, B, mask, scale)
    _, want = rounded(torch, exact, kind)
    if kind == "f16":
        limit = 1.5 * math.sqrt(2 * HALF_STEP[kind] * D)
        assert np.linalg.norm(got - want) <= limit * np.linalg.norm(want), np.linalg.norm(got - want) / np.linalg.norm(want)
    else:
        assert np.linalg.norm(got - exact) <= 1.015 * np.linalg.norm(want - exact)
    assert fbctx.error_word() == 0
