"""The tree verification operators past 32 bits: pools of more than 2^32 bytes a
tensor, and rows whose strides put them more than 2^31 elements apart."""
import numpy as np
import pytest

import ferrite_b200 as fb
from test_gpu_attn_tree import check as check_rows
from test_gpu_rotary import check as check_turned
from tree_reference import Batch, attention, frequencies, pair_size, rotate, sample

pytestmark = pytest.mark.gpu

FAR = (1 << 31) // 3 + 5  # elements between rows: the fourth lies past 2^31 elements


def far_rows(torch, a, dtype):
    """Rows of a [n, ...] tensor, FAR elements apart, as (whole buffer, view of the rows)."""
    n, width = a.shape[0], a[0].numel()
    buf = torch.empty((n - 1) * FAR + width, dtype=dtype, device="cuda")
    view = buf.as_strided((n, width), (FAR, 1))
    view.copy_(a.reshape(n, width).to(dtype))
    return buf, view


def test_rows_far_apart(fbctx, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(1)
    n, heads, dim = 5, 2, 64
    x = torch.from_numpy(rng.normal(0, 1, (n, heads, dim))).cuda()
    xb, xv = far_rows(torch, x, torch.float16)
    held = xv.double().cpu().numpy().reshape(n, heads, dim)
    pos = torch.tensor([5, 2, 9, 100, 77], dtype=torch.int32, device="cuda")
    freq, amp = frequencies(dim, 1e4)
    fb.rotary_apply(fbctx, fb.Rotary(dim, 1e4), fb.F16, xb.data_ptr(), FAR, dim, xb.data_ptr(), FAR, dim, pos.data_ptr(), n,
                    heads, dim)
    torch.cuda.synchronize()
    check_turned(xv.double().cpu().numpy().reshape(n, heads, dim), rotate(held, pos.cpu().numpy(), freq, amp, 1),
                 pair_size(held, dim, amp, 1), "f16")
    # logits of the same rows
    u = rng.random(n).astype(np.float32)
    ud, tok = torch.from_numpy(u).cuda(), torch.full((n,), -9, dtype=torch.int32, device="cuda")
    fb.sample_rows(fbctx, fb.F16, xb.data_ptr(), FAR, n, heads * dim, 0, 0, 0, 0, ud.data_ptr(), tok.data_ptr())
    want = [sample(xv[r].double().cpu().numpy(), 1.0, 0, 1.0, 0.0, float(u[r]))[0] for r in range(n)]
    assert tok.tolist() == want and fbctx.error_word() == 0


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_pools_past_four_gigabytes(fbctx, torch_cuda, kind):
    torch = torch_cuda
    rng = np.random.default_rng(2)
    dtype = torch.float32 if kind == "f32" else torch.float16
    heads, dim, page, pages, qheads = 8, 128, 64, 40003, 16
    new, lens = [3, 2], [700, 65]
    need = [-(-n // page) for n in lens]
    ids = np.concatenate([[pages - 1, 32767, 32768, 16383, 16384], rng.permutation(pages - 40000)[:2] + 40000 - 3,
                          rng.integers(100, 16000, sum(need))])[:sum(need)].astype(np.int32)
    assert len(set(ids)) == len(ids)
    small = Batch(rng, new, lens, heads, dim, page, spare=0)  # the same pages numbered 0, 1, ..
    k, v = (torch.empty(pages, heads, *s, dtype=torch.float16, device="cuda") for s in ((dim, page), (page, dim)))
    real = torch.from_numpy(ids.astype(np.int64)).cuda()
    k[real], v[real] = torch.from_numpy(small.k).cuda(), torch.from_numpy(small.v).cuda()
    table = np.where(small.table >= 0, ids[np.maximum(small.table, 0)], -1).astype(np.int32)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    bt, off, ln = t(table), t(small.offsets), t(np.array(lens, np.int32))
    # new rows appended from far-apart rows, then attended to
    kb, kv_ = far_rows(torch, torch.from_numpy(rng.normal(0, 1, (5, heads, dim))).cuda(), torch.float16)
    fb.kv_append(fbctx, None, fb.F16, kb.data_ptr(), FAR, kb.data_ptr(), FAR, off.data_ptr(), ln.data_ptr(), 0, bt.data_ptr(),
                 k.data_ptr(), v.data_ptr(), 2, 5, 3, heads, dim, page, small.max_pages, pages)
    rows = kv_.cpu().numpy().reshape(5, heads, dim)
    for b in range(2):
        for i in range(new[b]):
            pg, s = small.place(b, lens[b] - new[b] + i)
            small.k[pg, :, :, s] = small.v[pg, :, s] = rows[small.offsets[b] + i]
    torch.cuda.synchronize()
    assert torch.equal(k[real].cpu(), torch.from_numpy(small.k)) and torch.equal(v[real].cpu(), torch.from_numpy(small.v))
    q = torch.from_numpy(rng.normal(0, 1, (5, qheads, dim))).cuda()
    qb, qv = far_rows(torch, q, dtype)
    out = torch.full((5, qheads, dim), 7.0, dtype=dtype, device="cuda")
    ws = torch.empty(max(16, fb.attn_tree_workspace(fbctx, 2, 3, qheads, heads, dim, page, 700)), dtype=torch.uint8, device="cuda")
    fb.attn_tree(fbctx, fb.F32 if kind == "f32" else fb.F16, qb.data_ptr(), FAR, k.data_ptr(), v.data_ptr(), bt.data_ptr(),
                 off.data_ptr(), ln.data_ptr(), 0, 1, out.data_ptr(), qheads * dim, 2, 5, 3, qheads, heads, dim, page,
                 small.max_pages, pages, 700, 0.09, ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    held = qv.double().cpu().numpy().reshape(5, qheads, dim)
    check_rows(out.double().cpu().numpy(), attention(held, small, None, 0.09), held, small, 0.09, kind)
    assert fbctx.error_word() == 0
    del k, v, kb, kv_, qb, qv
    torch.cuda.empty_cache()
