"""Inputs and outputs in column ranges of the same rows, which do not overlap:
queries rotated into another part of their buffer, attention from there into a
third part, and everything else left as it was."""
import numpy as np
import pytest

import ferrite_b200 as fb
from test_gpu_attn_tree import check as check_rows
from test_gpu_rotary import check as check_turned
from tree_reference import Batch, attention, frequencies, pair_size, rotate, rounded, tree_mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,gap", [(4, 64, 0), (8, 128, 24), (1, 64, 3)])
def test_columns_of_one_buffer(fbctx, torch_cuda, heads, dim, gap):
    torch = torch_cuda
    rng = np.random.default_rng(heads)
    B = Batch(rng, [5, 9, 1], [70, 200, 33], 1, dim, 64)
    row = heads * dim
    width = 3 * row + gap
    buf, held = rounded(torch, rng.normal(0, 1, (B.total, width)), "f32")
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    pos = rng.integers(0, 5000, B.total).astype(np.int32)
    pd = t(pos)
    at = [buf.data_ptr() + 4 * row * i for i in range(3)]
    r = fb.Rotary(dim, 1e4)
    fb.rotary_apply(fbctx, r, fb.F32, at[0], width, dim, at[1], width, dim, pd.data_ptr(), B.total, heads, dim)
    mask = tree_mask(rng, B.new, 1)
    k, v, bt, off, ln, md = (t(a) for a in (B.k, B.v, B.table, B.offsets, np.array(B.lens, np.int32), mask.view(np.int32)))
    ws = torch.empty(max(16, fb.attn_tree_workspace(fbctx, 3, 9, heads, 1, dim, 64, 200)), dtype=torch.uint8, device="cuda")
    fb.attn_tree(fbctx, fb.F32, at[1], width, k.data_ptr(), v.data_ptr(), bt.data_ptr(), off.data_ptr(), ln.data_ptr(),
                 md.data_ptr(), 1, at[2], width, 3, B.total, 9, heads, 1, dim, 64, B.max_pages, B.num_pages, 200, 0.1,
                 ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    got = buf.double().cpu().numpy()
    part = lambda i: got[:, i * row:(i + 1) * row].reshape(B.total, heads, dim)  # noqa: E731
    assert np.array_equal(got[:, :row], held[:, :row]) and np.array_equal(got[:, 3 * row:], held[:, 3 * row:])
    freq, amp = frequencies(dim, 1e4)
    check_turned(part(1), rotate(part(0), pos, freq, amp, 1), pair_size(part(0), dim, amp, 1), "f32")
    check_rows(part(2), attention(part(1), B, mask, 0.1), part(1), B, 0.1, "f32")
    # heads interleaved: every second head's place is the output's
    pairs, held = rounded(torch, rng.normal(0, 1, (B.total, heads, 2, dim)), "f32")
    fb.rotary_apply(fbctx, r, fb.F32, pairs.data_ptr(), 2 * row, 2 * dim, pairs.data_ptr() + 4 * dim, 2 * row, 2 * dim,
                    pd.data_ptr(), B.total, heads, dim)
    torch.cuda.synchronize()
    got = pairs.double().cpu().numpy()
    assert np.array_equal(got[:, :, 0], held[:, :, 0])
    check_turned(got[:, :, 1], rotate(held[:, :, 0], pos, freq, amp, 1), pair_size(held[:, :, 0], dim, amp, 1), "f32")
    assert fbctx.error_word() == 0
