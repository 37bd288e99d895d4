"""More sequences than a warp has lanes, some without new rows, behind rows of
nobody: the shares of later sequences are found past the first 32."""
import numpy as np
import pytest

from test_gpu_attn_tree import Call, check
from tree_reference import Batch, attention, rounded, tree_mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch,reach", [(33, 900), (100, 600), (70, 200)])
def test_many_sequences(fbctx, torch_cuda, kind, batch, reach):
    torch = torch_cuda
    rng = np.random.default_rng(batch)
    new = [int(n) for n in rng.integers(0, 5, batch)]
    new[0], new[31], new[32], new[-1] = 0, 4, 0, 3
    lens = [n + int(x) for n, x in zip(new, rng.integers(0, reach, batch))]
    B = Batch(rng, new, lens, 2, 64, 64)
    skipped = 3
    mask = np.concatenate([np.zeros((skipped, 1), np.uint32), tree_mask(rng, new, 1)])
    qd, q = rounded(torch, rng.normal(0, 1, (B.total + skipped, 8, 64)), kind)
    c = Call(torch, fbctx, B, qd, mask, kind, 8, extra=skipped)
    c.off += skipped
    got = c.result(0.125)
    assert (got[:skipped] == 7.0).all() and fbctx.error_word() == 0
    check(got[skipped:], attention(q[skipped:], B, mask[skipped:], 0.125), q[skipped:], B, 0.125, kind)
