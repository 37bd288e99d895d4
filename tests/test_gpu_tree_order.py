"""What stands behind a tree attention on its stream sees its results: short
sequences under a large max_seq_len, where the joining kernel is launched and no
row group needs it, followed at once by kernels that read the rows, write the
queries, or use the workspace again -- the same bits with and without
programmatic dependent launch."""
import numpy as np
import pytest

import ferrite_b200 as fb
from oracle import oracle as O
from tree_reference import Batch, attention, fb_type, rounded

pytestmark = pytest.mark.gpu

QH, KV, DIM, PAGE, CAPACITY = 32, 8, 128, 64, 4096


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[40 + i for i in range(16)], [64, 3000, 25, 40, 33, 64, 25, 50]])
def test_readers_and_writers_behind_the_attention(torch_cuda, kind, lens):
    torch = torch_cuda
    rng = np.random.default_rng(len(lens))
    new = [20] * len(lens)
    B = Batch(rng, new, lens, KV, DIM, PAGE)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    qd, q = rounded(torch, rng.normal(0, 1, (B.total, QH, DIM)), kind)
    k, v, off, ln = t(B.k), t(B.v), t(B.offsets), t(np.array(lens, np.int32))
    width, row = CAPACITY // PAGE, QH * DIM  # a table as wide as the capacity
    table = np.zeros((len(lens), width), np.int32)
    table[:, :B.max_pages] = np.maximum(B.table[:, :width], 0)
    bt = t(table)
    w = O.quantize(O.Q4_K, rng.normal(0, 0.02, (256, row)).astype(np.float32))
    scale = 0.09

    stream = torch.cuda.Stream()
    ctx = fb.Context(0, stream.cuda_stream)
    weight = fb.QTensor.upload(ctx, O.Q4_K, 256, row, w)
    n = fb.attn_tree_workspace(ctx, len(lens), 20, QH, KV, DIM, PAGE, CAPACITY)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    runs = []
    for pdl in (False, True, True, True):
        ctx.set_pdl(pdl)
        q1, first, second, third = (torch.full_like(qd, 7.0) for _ in range(4))
        y = torch.full((B.total, 256), 7.0, device="cuda")
        q1.copy_(qd)
        ws.fill_(255)
        torch.cuda.synchronize()

        def call(src, dst):
            fb.attn_tree(ctx, fb_type(fb, kind), src.data_ptr(), row, k.data_ptr(), v.data_ptr(), bt.data_ptr(),
                         off.data_ptr(), ln.data_ptr(), 0, 1, dst.data_ptr(), row, len(lens), B.total, 20, QH, KV, DIM, PAGE,
                         width, B.num_pages, CAPACITY, scale, ws.data_ptr(), n)

        call(q1, first)
        call(first, second)  # reads the rows, uses the workspace again
        call(second, q1)     # writes what the first call read
        call(q1, third)
        if kind == "f32":    # (quantises the rows for an integer product, its kernels programmatic dependents too)
            fb.QMatMul(weight).forward(third.data_ptr(), y.data_ptr(), B.total)
        stream.synchronize()
        assert ctx.error_word() == 0
        runs.append([x.clone() for x in (first, second, q1, third, y)])
    for r in runs[1:]:
        for a, b in zip(r, runs[0]):
            assert torch.equal(a, b)
    # (what the rows are has tests of its own; here that they are there at all, to two half steps of the coarser type)
    got, want = runs[0][0].double().cpu().numpy(), attention(q, B, None, scale)
    assert np.linalg.norm(got - want) <= 2.0 ** -7 * np.linalg.norm(want)
    if kind == "f32":
        assert (runs[0][4] != 7.0).any(dim=1).all()
    weight.close()
    ctx.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_appends_behind_the_attention(torch_cuda, kind):
    """Append, attend, overwrite the same cache places, attend again, captured and replayed: each attention sees the rows
    appended before it and none of the later ones."""
    torch = torch_cuda
    rng = np.random.default_rng(3)
    lens, n = [40 + i for i in range(16)], 20
    B = Batch(rng, [n] * 16, lens, KV, DIM, PAGE)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    row, kvrow = QH * DIM, KV * DIM
    qd, _ = rounded(torch, rng.normal(0, 1, (B.total, QH, DIM)), kind)
    rows = [rounded(torch, rng.normal(0, 1, (B.total, 2, KV, DIM)), kind)[0] for _ in range(4)]
    k, v, off, ln, bt = t(B.k), t(B.v), t(B.offsets), t(np.array(lens, np.int32)), t(np.maximum(B.table, 0))
    outs = [torch.empty_like(qd) for _ in rows]
    stream = torch.cuda.Stream()
    ctx = fb.Context(0, stream.cuda_stream)
    capacity = B.max_pages * PAGE
    longer = t(np.zeros((16, CAPACITY // PAGE), np.int32))
    longer[:, :B.max_pages] = bt
    ws = torch.empty(fb.attn_tree_workspace(ctx, 16, n, QH, KV, DIM, PAGE, CAPACITY), dtype=torch.uint8, device="cuda")

    def step(i):
        at = rows[i].data_ptr()
        fb.kv_append(ctx, None, fb_type(fb, kind), at, 2 * kvrow, at + kvrow * rows[i].element_size(), 2 * kvrow, off.data_ptr(),
                     ln.data_ptr(), 0, longer.data_ptr(), k.data_ptr(), v.data_ptr(), 16, B.total, n, KV, DIM, PAGE,
                     CAPACITY // PAGE, B.num_pages)
        fb.attn_tree(ctx, fb_type(fb, kind), qd.data_ptr(), row, k.data_ptr(), v.data_ptr(), longer.data_ptr(), off.data_ptr(),
                     ln.data_ptr(), 0, 1, outs[i].data_ptr(), row, 16, B.total, n, QH, KV, DIM, PAGE, CAPACITY // PAGE,
                     B.num_pages, CAPACITY, 0.09, ws.data_ptr(), ws.numel())

    assert capacity < CAPACITY
    want = []
    torch.cuda.synchronize()
    for i in range(4):
        step(i)
        stream.synchronize()
        want.append(outs[i].clone())
    assert not any(torch.equal(a, b) for a, b in zip(want, want[1:]))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        for i in range(4):
            step(i)
    for _ in range(3):
        for o in outs:
            o.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    for o in outs:
        o.fill_(7.0)
    torch.cuda.synchronize()
    for i in range(4):
        step(i)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and ctx.error_word() == 0
    ctx.close()
