"""Host threads with a context each call the row sampler and the cache append
with sizes of their own at the same time: a kernel's launch limits belong to the
process, so a small call must not take away what a large one needs."""
import threading

import numpy as np
import pytest

import ferrite_b200 as fb
from tree_reference import sample

pytestmark = pytest.mark.gpu


def together(torch, large, smalls, n):
    """large(ctx) and each of smalls n times, each from a thread with a stream of its own."""
    calls = [large, *smalls]
    failed, start = [], threading.Barrier(len(calls))

    def body(call):
        try:
            torch.cuda.set_device(0)
            stream = torch.cuda.Stream()
            ctx = fb.Context(0, stream.cuda_stream)
            start.wait(60)
            for _ in range(n):
                call(ctx)
            stream.synchronize()
            ctx.close()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=body, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join(300)
    assert not failed, failed[0]


def test_row_sampling_of_two_sizes(torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(1)
    tokens, want = [], []

    def call(rows, vocab):
        x = torch.from_numpy(rng.normal(0, 1, (rows, vocab)).astype(np.float32)).cuda()
        u = torch.from_numpy(rng.random(rows).astype(np.float32)).cuda()
        tok = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
        tokens.append(tok)
        want.append(sample(x[-1].double().cpu().numpy(), 1.0, 0, 1.0, 0.0, float(u[-1]))[0])
        return lambda ctx: fb.sample_rows(ctx, fb.F32, x.data_ptr(), vocab, rows, vocab, 0, 0, 0, 0, u.data_ptr(),
                                          tok.data_ptr())

    together(torch, call(230, 151936), [call(230, 300) for _ in range(3)], 2000)
    assert [int(t[-1]) for t in tokens] == want


@pytest.mark.parametrize("rots", [(128, 64), (120, 6)])  # whole chunks, two heads a block or one; the general form
def test_cache_append_of_two_sizes(torch_cuda, rots):
    torch = torch_cuda
    pages, page, heads, dim = 80, 64, 8, 128
    checks = []

    def call(rot, batch, new):
        rows = batch * new
        x = torch.randn(rows, 2, heads, dim, device="cuda")
        off = torch.arange(0, rows + 1, new, dtype=torch.int32, device="cuda")
        lens = torch.full((batch,), new, dtype=torch.int32, device="cuda")
        bt = torch.arange(pages, dtype=torch.int32, device="cuda").reshape(batch, -1).contiguous()
        k, v = (torch.zeros(pages, heads, dim, page, dtype=torch.float16, device="cuda") for _ in range(2))
        r = fb.Rotary(rot, 1e5)
        checks.append((v, x, bt, new))
        at, row = x.data_ptr(), heads * dim
        return lambda ctx: fb.kv_append(ctx, r, fb.F32, at, 2 * row, at + 4 * row, 2 * row, off.data_ptr(), lens.data_ptr(), 0,
                                        bt.data_ptr(), k.data_ptr(), v.data_ptr(), batch, rows, new, heads, dim, page,
                                        bt.shape[1], pages)

    together(torch, call(rots[0], 40, 100), [call(rots[1], 1, 1) for _ in range(3)], 4000)
    for v, x, bt, new in checks:
        last = v.view(pages, heads, page, dim)[bt[-1, (new - 1) // page], :, (new - 1) % page]
        assert torch.equal(last, x[-1, 1].half())
