"""Scores so large that f32 has no fractions, or no small integers, at their size.

Queries and keys are 0 outside dimension 0, where the keys hold 1, 2 or 3: equal
keys have equal scores and unequal ones lie at least |s| / 3 apart, thousands and
more, so that a row is the mean of its largest keys' values.  The weights are equal
then, to the 2^-21 that the probabilities' parts hold: bound 2^-18 max|v| (eight
times that, for the sums), and half a step of the type."""
import numpy as np
import pytest

from test_gpu_attn_tree import Call
from tree_reference import HALF_STEP, Batch, attention, rounded, tree_mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,size", [
    ("f32", 1e4), ("f32", 1e7), ("f32", 2e8), ("f32", -3e8), ("f32", 1e10), ("f32", -1e12), ("f32", 1e25), ("f32", -2e33),
    ("f32", 1e37), ("f32", -1e37), ("f16", 1e4), ("f16", 2e8), ("f16", -3e9), ("bf16", 3e8), ("bf16", -1e12), ("bf16", 1e31),
    ("bf16", -2e33),
])
@pytest.mark.parametrize("new,page,prefix", [(9, 64, 100), (9, 32, 2500), (45, 64, 100), (45, 64, 1800), (7, 64, 0)])
def test_rows_are_means_of_their_largest_keys(fbctx, torch_cuda, kind, size, new, page, prefix):
    torch = torch_cuda
    rng = np.random.default_rng(new + prefix)
    B = Batch(rng, [new, new], [prefix + new, prefix // 2 + new], 2, 64, page)
    B.k[:] = 0
    B.k[:, :, 0] = rng.integers(1, 4, B.k[:, :, 0].shape)
    mask = tree_mask(rng, B.new, 2)
    scale = 1.0 if kind != "f16" else abs(size) / 1e4  # (f16 queries reach 6e4)
    qv = np.zeros((2 * new, 8, 64))
    qv[..., 0] = size / scale * rng.uniform(0.5, 1.0, (2 * new, 8))
    qd, q = rounded(torch, qv, kind)
    got = Call(torch, fbctx, B, qd, mask, kind, 8, words=2).result(scale)
    want = attention(q, B, mask, float(np.float32(scale)))
    vmax = float(np.abs(B.v).max())
    tol = 2.0 ** -18 * vmax + (0 if kind == "f32" else HALF_STEP[kind] * np.abs(want) * 1.01 + 2.0 ** -25)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    assert fbctx.error_word() == 0
