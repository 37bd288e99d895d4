"""Host threads with a context each call the row sampler with sizes of their own
at the same time: the kernel's launch limits belong to the process, so a small
call must not take away what a large one needs."""
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
