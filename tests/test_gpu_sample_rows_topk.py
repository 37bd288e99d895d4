"""A top-k alone whose cut lies far below the maximum in temperatures: found in a
few passes over the row, as at temperatures where it lies near."""
import numpy as np
import pytest

import ferrite_b200 as fb
from test_gpu_sample_rows import check, run
from tree_reference import fb_type, rounded, torch_type

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (40, 30011), (48, 5003)])
@pytest.mark.parametrize("k", [257, 1000, 4000])
def test_cuts_far_below_the_maximum(fbctx, torch_cuda, kind, rows, vocab, k):
    """Plain rows, rows masked by -inf and by the type's lowest value, rows of a few distinct values."""
    torch = torch_cuda
    rng = np.random.default_rng(vocab + k)
    lowest = float(torch.finfo(torch_type(torch, kind)).min)
    plain = 2.5 * rng.normal(0, 1, (rows, vocab))
    shifted = 1e-3 * plain + 50.0  # all of one sign, close together
    hidden = np.where(rng.random((rows, vocab)) < 0.6, lowest, plain)
    gone = np.where(rng.random((rows, vocab)) < 0.9, -np.inf, plain)
    few = np.round(plain)
    for x in (plain, shifted, hidden, gone, few):
        for t in (0.2, 0.05, 0.004, 1e-5):
            # (at such temperatures a draw by weight rarely leaves the first tokens: u at its end asks for the last kept)
            for u in (0.3, 1.0):
                check(*run(torch, fbctx, x, kind, t=t, k=k, u=u))


def last_kept(torch, ctx, x, kind, t, k):
    """The last kept token in index order: u = 1 (every kept logit weighs something)."""
    rows, vocab = x.shape
    d, held = rounded(torch, x, kind)
    a = lambda v, dt: torch.full((rows,), v, dtype=dt, device="cuda")  # noqa: E731
    tt, kk, uu, tok = a(t, torch.float32), a(k, torch.int32), a(1.0, torch.float32), a(-9, torch.int32)
    fb.sample_rows(ctx, fb_type(fb, kind), d.data_ptr(), vocab, rows, vocab, tt.data_ptr(), kk.data_ptr(), 0, 0, uu.data_ptr(),
                   tok.data_ptr())
    order = np.argsort(-held, axis=1, kind="stable")[:, :k]
    return tok.cpu().numpy(), order.max(axis=1)


@pytest.mark.parametrize("k", [257, 1000, 4000])
def test_the_cut_itself(fbctx, torch_cuda, k):
    rng = np.random.default_rng(k)
    x = 2.5 * rng.normal(0, 1, (8, 60000))
    for t in (0.2, 0.05, 0.03):  # (the k-th logit within 745 T of the maximum: its weight is not 0)
        got, want = last_kept(torch_cuda, fbctx, x, "f32", t, k)
        assert got.tolist() == want.tolist()


def test_passes_do_not_depend_on_the_temperature(fbctx, torch_cuda):
    """Low temperatures took some seventy passes over the row; a few are less than four times the time of one temperature
    above.  (Best of several replays, each of ten calls.)"""
    torch = torch_cuda
    x = 2.5 * torch.randn(8, 151936, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    x[4:] = x[4:].masked_fill(x[4:] < 0, torch.finfo(torch.float32).min)
    a = lambda v, dt: torch.full((8,), v, dtype=dt, device="cuda")  # noqa: E731
    k, u, tok = a(1000, torch.int32), a(0.5, torch.float32), a(0, torch.int32)
    stream = torch.cuda.Stream()
    ctx = fb.Context(0, stream.cuda_stream)
    best = {}
    for t in (2.0, 0.1, 0.004):
        tt = a(t, torch.float32)
        call = lambda: fb.sample_rows(ctx, fb.F32, x.data_ptr(), 151936, 8, 151936, tt.data_ptr(), k.data_ptr(), 0, 0,  # noqa: E731,B023
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
        best[t] = min(times)
    assert best[0.1] < 4 * best[2.0] and best[0.004] < 4 * best[2.0], best
    ctx.close()
