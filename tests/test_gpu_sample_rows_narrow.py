"""Nuclei so wide that the approximate masses leave thousands of logits open, and
rows of many equal ones: the same rules, in a few passes over the row."""
import numpy as np
import pytest

import ferrite_b200 as fb
from test_gpu_sample_rows import check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (30, 20011), (460, 2003)])
@pytest.mark.parametrize("p", [0.99, 0.999, 0.99999, 0.9999999])
def test_top_p_next_to_one(fbctx, torch_cuda, kind, rows, vocab, p):
    rng = np.random.default_rng(vocab)
    x = 2.5 * rng.normal(0, 1, (rows, vocab))
    x[rows // 2, ::3] = -np.inf
    for s in (dict(t=0.7), dict(t=2.0), dict(t=1.0, k=1500), dict(t=1.5, m=1e-6)):
        check(*run(torch_cuda, fbctx, x, kind, p=p, u=rng.random(rows), **s))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("values", [1, 3, 40])
def test_few_distinct_values(fbctx, torch_cuda, kind, values):
    """Thousands of equal logits on either side of the cut, which goes by their index."""
    rng = np.random.default_rng(values)
    x = rng.integers(0, values, (6, 30011)) * 0.25
    for s in (dict(p=0.9), dict(p=0.37), dict(k=5000), dict(k=12345, p=0.6), dict(p=0.71, m=0.5), dict(p=0.5, t=np.inf)):
        for u in (0.0, 0.613, 0.99999994):
            check(*run(torch_cuda, fbctx, x, kind, u=u, **s))


def test_passes_do_not_depend_on_top_p(fbctx, torch_cuda):
    """Nuclei next to one, infinite temperatures and equal logits took up to 64 passes over the row, thirty times the time of
    an ordinary nucleus; now less than four times (equal logits: twenty, their counts share a bin)."""
    torch = torch_cuda
    plain = 2.5 * torch.randn(16, 151936, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    flat = torch.zeros_like(plain)
    a = lambda v, dt: torch.full((16,), v, dtype=dt, device="cuda")  # noqa: E731
    u, tok = a(0.5, torch.float32), a(0, torch.int32)
    stream = torch.cuda.Stream()
    ctx = fb.Context(0, stream.cuda_stream)

    def best(x, t, p):
        tt, pp = a(t, torch.float32), a(p, torch.float32)
        call = lambda: fb.sample_rows(ctx, fb.F32, x.data_ptr(), 151936, 16, 151936, tt.data_ptr(), 0, pp.data_ptr(), 0,  # noqa: E731
                                      u.data_ptr(), tok.data_ptr())
        torch.cuda.synchronize()
        call()
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            for _ in range(10):
                call()
        times = []
        for _ in range(8):
            start, end = torch.cuda.Event(True), torch.cuda.Event(True)
            start.record()
            g.replay()
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    usual = best(plain, 1.0, 0.95)
    for x, t, p, most in ((plain, 0.7, 0.999, 4), (plain, 0.7, 0.99999, 4), (plain, float("inf"), 0.9, 4), (flat, 1.0, 0.9, 20)):
        assert best(x, t, p) < most * usual, (t, p, best(x, t, p), usual)
    ctx.close()
