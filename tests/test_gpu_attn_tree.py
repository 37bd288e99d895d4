"""Tree attention against its definition in binary64.

Tolerances count roundings.  A score is a sum of dim products of f32 q (its
fp16 high and low parts hold it to 2^-21) with fp16 k, in units of log 2, where
it has a magnitude of S = scale log2(e) sum |q||k|: its error is below
(2^-21 + 2^-22) S, as independent roundings far below.  A relative error d of
the weights moves a row by at most 2 d max|v|.  Each element is held to 2 (2^-20
S + 2^-18) max|v| (2^-18: 2^-21 of the probabilities' own parts and
exponentials, eight times for the sums), each row set to 4e-6 in the 2-norm (twice
2^-20 S rounding as independent errors, with S of 8), and half a step of
the output type on top of either.  For 16-bit types the probabilities are one
fp16 value each, off by 2^-11 of it at most: the weights, normalised, by 2^-10,
which moves an element by 2^-10 max|v| at most, and a row set's 2-norm by no
more than the half step that is allowed for the output already (both are
uniform in their steps, so each is 0.42 of its largest, 0.6 together)."""
import math

import numpy as np
import pytest

import ferrite_b200 as fb
from tree_reference import HALF_STEP, Batch, attention, fb_type, rounded, torch_type, tree_mask

pytestmark = pytest.mark.gpu


class Call:
    """Device side of a Batch, with a workspace of its own."""

    def __init__(self, torch, ctx, B, q, mask, kind, qheads, out=None, extra=0, words=None, max_seq=None, max_new=None):
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.torch, self.ctx, self.B, self.kind, self.qheads = torch, ctx, B, kind, qheads
        self.k, self.v, self.bt, self.off = t(B.k), t(B.v), t(B.table), t(B.offsets)
        self.lens = t(np.array(B.lens, np.int32))
        self.q = q
        self.words = words or max(1, -(-max(B.new) // 32))
        self.mask = None if mask is None else t(mask.view(np.int32))
        self.row = qheads * B.dim
        self.n_rows = B.total + extra
        self.out = out if out is not None else torch.full((self.n_rows, qheads, B.dim), 7.0, dtype=q.dtype, device="cuda")
        self.max_seq = max_seq or max(max(B.lens), 1)
        self.max_new = max_new or max(max(B.new), 1)
        n = fb.attn_tree_workspace(ctx, B.batch, self.max_new, qheads, B.heads, B.dim, B.page, self.max_seq)
        self.ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")  # NaN patterns: contents are ignored

    def go(self, scale, ctx=None, q_stride=None):
        B = self.B
        fb.attn_tree(ctx or self.ctx, fb_type(fb, self.kind), self.q.data_ptr(), q_stride or self.row, self.k.data_ptr(),
                     self.v.data_ptr(), self.bt.data_ptr(), self.off.data_ptr(), self.lens.data_ptr(),
                     self.mask.data_ptr() if self.mask is not None else 0, self.words, self.out.data_ptr(), self.row,
                     B.batch, self.n_rows, self.max_new, self.qheads, B.heads, B.dim, B.page, B.max_pages, B.num_pages,
                     self.max_seq, scale, self.ws.data_ptr(), self.ws.numel())
        return self.out

    def result(self, scale):
        self.go(scale)
        self.torch.cuda.synchronize()
        return self.out.double().cpu().numpy()


def check(got, want, q, B, scale, kind, rows=None):
    vmax = max(float(np.abs(B.v[np.isfinite(B.v)]).max()), 1e-3)
    kmax = float(np.abs(B.k[np.isfinite(B.k)]).max())
    s = scale * 1.4427 * np.abs(q).sum(-1, keepdims=True) * kmax
    tol = 2 * (2.0 ** -20 * s + 2.0 ** -18) * vmax + (
        0 if kind == "f32" else HALF_STEP[kind] * np.abs(want) * 1.01 + 2.0 ** -25 + 2.0 ** -10 * vmax)
    err = np.abs(got - want)
    assert np.isfinite(got).all() and (err <= tol).all(), f"over by {(err - tol).max()}"
    norm = np.linalg.norm(want)
    if norm > 0:
        limit = 4e-6 + (0 if kind == "f32" else HALF_STEP[kind])
        assert np.linalg.norm(got - want) <= limit * norm, f"2-norm {np.linalg.norm(got - want) / norm}"


# new rows, lens, query heads, kv heads, dim, page, type
CASES = [
    ([1], [1], 4, 4, 128, 64, "f32"), ([1], [64], 8, 1, 128, 64, "f32"), ([1], [65], 32, 8, 128, 32, "f16"),
    ([3], [3], 5, 1, 64, 64, "f32"), ([7], [190], 32, 8, 128, 64, "f32"), ([60], [700], 8, 2, 128, 64, "f32"),
    ([33], [1500], 8, 2, 64, 32, "bf16"), ([5, 0, 12, 1], [300, 77, 12, 129], 8, 2, 128, 32, "f32"),
    ([64, 1, 31], [64, 640, 95], 10, 2, 128, 64, "f16"), ([40], [500], 16, 1, 128, 64, "f32"),
    ([100], [163], 8, 1, 64, 64, "f16"), ([2] * 20, [2 + 13 * i for i in range(20)], 4, 2, 64, 32, "f32"),
    ([1, 1], [4000, 10], 8, 8, 128, 64, "bf16"), ([20], [2100], 7, 7, 64, 64, "f32"), ([0, 0], [5, 0], 2, 1, 64, 64, "f32"),
    ([3], [600], 160, 1, 64, 64, "f32"), ([13], [4097], 8, 2, 128, 32, "f32"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{max(c[1])}-{c[2]}.{c[3]}-{c[4]}-{c[5]}-{c[6]}")
@pytest.mark.parametrize("chain", [False, True])
def test_attn_tree(fbctx, torch_cuda, case, chain):
    torch = torch_cuda
    new, lens, qh, heads, dim, page, kind = case
    rng = np.random.default_rng(sum(lens) + sum(new))
    B = Batch(rng, new, lens, heads, dim, page)
    words = max(1, -(-max(new) // 32)) + 1
    mask = None if chain else tree_mask(rng, new, words)
    qd, q = rounded(torch, 1.5 * rng.normal(0, 1, (B.total + 2, qh, dim)), kind)
    c = Call(torch, fbctx, B, qd, mask, kind, qh, extra=2, words=words)
    scale = 1 / math.sqrt(dim)
    got = c.result(scale)
    assert fbctx.error_word() == 0
    assert (got[B.total:] == 7.0).all()  # rows behind the last sequence
    if B.total:
        check(got[:B.total], attention(q[:B.total], B, mask, scale), q[:B.total], B, scale, kind)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_rows_that_see_nothing(fbctx, torch_cuda, kind):
    """No prefix and no mask bit: zeros; garbage bits past the sequence's rows count for nothing."""
    torch = torch_cuda
    rng = np.random.default_rng(2)
    B = Batch(rng, [6, 35], [6, 35], 2, 64, 64)
    mask = tree_mask(rng, B.new, 2)
    mask[0] = 0
    mask[3] = [0xFFFFFFC0, 0xFFFFFFFF]
    mask[20] = 0
    qd, q = rounded(torch, rng.normal(0, 1, (41, 4, 64)), kind)
    got = Call(torch, fbctx, B, qd, mask, kind, 4).result(0.125)
    assert (got[[0, 3, 20]] == 0).all()
    check(got, attention(q, B, mask, 0.125), q, B, 0.125, kind)


@pytest.mark.parametrize("page", [32, 64])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_never_reaches_it(fbctx, torch_cuda, page, value):
    """Non-finite k and v behind the end of the last page and at drafted rows
    that others do not descend from; rows that see such a v get its value."""
    torch = torch_cuda
    rng = np.random.default_rng(6)
    B = Batch(rng, [9], [70 + 9], 1, 128, page)
    clean = attention
    mask = np.array([[1 << i | (1 << 0)] for i in range(9)], np.uint32)  # siblings under row 0
    for slot in range(79, -(-79 // page) * page):
        pg, s = B.place(0, slot)
        B.k[pg, :, :, s] = value
        B.v[pg, :, s] = value
    qd, q = rounded(torch, rng.normal(0, 1, (9, 4, 128)), "f32")
    want = clean(q, B, mask, 0.1)
    pg, s = B.place(0, 70 + 4)
    B.k[pg, :, :, s] = value
    pg, s = B.place(0, 70 + 6)
    B.v[pg, 0, s, 17] = value
    B.v[pg, 0, s, 100] = value
    got = Call(torch, fbctx, B, qd, mask, "f32", 4).result(0.1)
    others = [i for i in range(9) if i not in (4, 6)]
    check(got[others], want[others], q[others], B, 0.1, "f32")
    assert not np.isfinite(got[6][:, [17, 100]]).any()
    rest = [d for d in range(128) if d not in (17, 100)]
    check(got[[6]][..., rest], want[[6]][..., rest], q[[6]], B, 0.1, "f32")


def test_nan_in_one_query_stays_in_its_row(fbctx, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(7)
    B = Batch(rng, [5], [333], 2, 64, 64)
    qd, q = rounded(torch, rng.normal(0, 1, (5, 4, 64)), "f32")
    want = attention(q, B, None, 0.125)
    qd[2, 1, 9] = float("nan")
    got = Call(torch, fbctx, B, qd, None, "f32", 4).result(0.125)
    assert np.isnan(got[2, 1]).all()
    got[2, 1] = want[2, 1]
    check(got, want, q, B, 0.125, "f32")


@pytest.mark.parametrize("qsize,kind", [(1e-6, "f32"), (3e5, "f32"), (1e30, "bf16")])
def test_large_and_small_queries(fbctx, torch_cuda, qsize, kind):
    """Queries beyond fp16's range, with the scale that brings the scores back."""
    torch = torch_cuda
    rng = np.random.default_rng(9)
    B = Batch(rng, [4], [200], 1, 64, 64)
    qd, q = rounded(torch, qsize * rng.normal(0, 1, (4, 8, 64)), kind)
    scale = float(np.float32(0.125 / qsize))
    got = Call(torch, fbctx, B, qd, None, kind, 8).result(scale)
    check(got, attention(q, B, None, scale), q, B, scale, kind)


def test_sharp_softmax(fbctx, torch_cuda):
    """Scores that span hundreds: one key holds the row, late maxima replace early ones."""
    torch = torch_cuda
    rng = np.random.default_rng(10)
    B = Batch(rng, [16], [1024], 2, 128, 64)
    qd, q = rounded(torch, 12 * rng.normal(0, 1, (16, 8, 128)), "f32")
    mask = tree_mask(rng, B.new, 1)
    got = Call(torch, fbctx, B, qd, mask, "f32", 8).result(0.25)
    check(got, attention(q, B, mask, 0.25), q, B, 0.25, "f32")


def test_strided_misaligned_queries(fbctx, torch_cuda):
    """q inside fused rows, and q, out off 16-byte boundaries."""
    torch = torch_cuda
    rng = np.random.default_rng(11)
    B = Batch(rng, [5, 3], [130, 66], 2, 64, 32)
    for start, width in ((0, 6 * 64 + 256), (1, 6 * 64 + 1)):
        flat, held = rounded(torch, rng.normal(0, 1, start + 8 * width), "f32")
        q = held[start:].reshape(8, width)[:, :384].reshape(8, 6, 64)
        buf = torch.full((8 * 384 + 2,), 7.0, device="cuda")
        c = Call(torch, fbctx, B, flat[start:], None, "f32", 6, out=buf[start:])
        c.go(0.125, q_stride=width)
        torch.cuda.synchronize()
        got = buf.double().cpu().numpy()
        assert (got[start + 8 * 384:] == 7.0).all() and (got[:start] == 7.0).all()
        check(got[start:start + 8 * 384].reshape(8, 6, 64), attention(q, B, None, 0.125), q, B, 0.125, "f32")


def test_shared_and_bad_pages(fbctx, torch_cuda):
    """Two sequences over the same prefix pages; then page ids outside the pool: their tokens are skipped."""
    torch = torch_cuda
    for page in (64, 32):
        rng = np.random.default_rng(12)
        B = Batch(rng, [4, 4], [400, 400], 1, 128, page)
        B.table[1, :3] = B.table[0, :3]
        mask = tree_mask(rng, B.new, 1)
        qd, q = rounded(torch, rng.normal(0, 1, (8, 2, 128)), "f32")
        got = Call(torch, fbctx, B, qd, mask, "f32", 2).result(0.1)
        check(got, attention(q, B, mask, 0.1), q, B, 0.1, "f32")
        assert fbctx.error_word() == 0
        bad = (0, 2, 5)
        want = attention(q, B, mask, 0.1, bad_pages=bad)
        for j, p in zip(bad, (-1, B.num_pages, 2 ** 30)):
            B.table[:, j] = p
        got = Call(torch, fbctx, B, qd, mask, "f32", 2).result(0.1)
        assert fbctx.error_word() == 8
        check(got, want, q, B, 0.1, "f32")


def test_bad_sequences_are_left_out(fbctx, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(13)
    B = Batch(rng, [3, 3, 3], [90, 90, 90], 2, 64, 64)
    qd, q = rounded(torch, rng.normal(0, 1, (9, 4, 64)), "f32")
    want = attention(q, B, None, 0.125)
    for lens in ([90, 2, 90], [90, 91, 90], [90, -1, 90]):
        c = Call(torch, fbctx, B, qd, None, "f32", 4)
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        got = c.result(0.125)
        assert fbctx.error_word() == 4
        assert (got[3:6] == 7.0).all()
        check(got[[0, 1, 2, 6, 7, 8]], want[[0, 1, 2, 6, 7, 8]], q[[0, 1, 2, 6, 7, 8]], B, 0.125, "f32")


def test_single_rows_match_decode_attention(fbctx, torch_cuda):
    """One new token a sequence is fb_attn_decode's call."""
    torch = torch_cuda
    rng = np.random.default_rng(14)
    B = Batch(rng, [1] * 5, [1, 64, 700, 130, 2000], 8, 128, 64)
    qd, q = rounded(torch, rng.normal(0, 1, (5, 32, 128)), "f32")
    scale = 1 / math.sqrt(128)
    c = Call(torch, fbctx, B, qd, None, "f32", 32)
    got = c.result(scale)
    other = torch.empty_like(c.out)
    table = c.bt.clamp(min=0)
    fb.attn_decode(fbctx, qd.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), table.data_ptr(), c.lens.data_ptr(),
                   other.data_ptr(), 5, 32, 8, 128, 64, B.max_pages, B.num_pages, 2000, scale)
    torch.cuda.synchronize()
    ref = attention(q, B, None, scale)
    check(got, ref, q, B, scale, "f32")
    check(other.double().cpu().numpy(), ref, q, B, scale, "f32")


def test_same_bits_every_time_on_streams_and_in_graphs(fbctx, torch_cuda):
    """Two captured calls with workspaces of their own, replayed together on two streams, give the bits of the plain call."""
    torch = torch_cuda
    rng = np.random.default_rng(15)
    calls, plain = [], []
    for n, length, heads in ((30, 3000, 2), (8, 900, 4)):
        B = Batch(rng, [n, 3], [length, 257], heads, 128, 64)
        qd, _ = rounded(torch, rng.normal(0, 1, (n + 3, 8, 128)), "f32")
        c = Call(torch, fbctx, B, qd, tree_mask(rng, B.new, 1), "f32", 8)
        plain.append(c.result(0.1).copy())
        calls.append(c)
    streams = [torch.cuda.Stream() for _ in calls]
    graphs, ctxs = [], []
    for c, s in zip(calls, streams):
        ctx = fb.Context(0, s.cuda_stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.go(0.1, ctx=ctx)
        graphs.append(g)
        ctxs.append(ctx)
    for _ in range(5):
        for c in calls:
            c.out.fill_(7.0)
            c.ws.fill_(255)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, p in zip(calls, plain):
            assert np.array_equal(c.out.double().cpu().numpy(), p)
    for ctx in ctxs:
        assert ctx.error_word() == 0


@pytest.mark.parametrize("kind,page,qheads", [("f16", 32, 32), ("f32", 64, 32), ("bf16", 64, 64)])
def test_same_bits_over_many_runs(fbctx, torch_cuda, kind, page, qheads):
    """Unequal lengths whose one-tile groups start on every ring stage: keys that arrive out of order change nothing."""
    torch = torch_cuda
    rng = np.random.default_rng(16)
    new = [int(n) for n in rng.integers(1, 34, 12)]
    B = Batch(rng, new, [n + int(x) for n, x in zip(new, rng.integers(60, 5000, 12))], 8, 128, page)
    qd, q = rounded(torch, rng.normal(0, 1, (B.total, qheads, 128)), kind)
    mask = tree_mask(rng, new, 2)
    c = Call(torch, fbctx, B, qd, mask, kind, qheads, words=2)
    first = c.result(0.09)
    assert np.isfinite(first).all()
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    want = c.out.clone()
    for i in range(150):
        c.out.fill_(7.0)
        if i % 3 == 0:
            flush.fill_(i)  # keys from memory one time, from L2 another
        c.go(0.09)
        assert torch.equal(c.out, want), f"run {i}"
    assert fbctx.error_word() == 0


def test_in_place_is_refused(fbctx, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(18)
    B = Batch(rng, [2], [70], 2, 64, 64)
    qd, _ = rounded(torch, rng.normal(0, 1, (2, 4, 64)), "f32")
    c = Call(torch, fbctx, B, qd, None, "f32", 4, out=qd)
    with pytest.raises(fb.FerriteError, match="overlap"):
        c.go(0.1)


def test_sums_of_long_contexts(fbctx, torch_cuda):
    """Some seventy blocks of keys to an SM: what a matrix instruction drops of a running sum must not add up over them."""
    torch = torch_cuda
    rng = np.random.default_rng(17)
    B = Batch(rng, [2, 1], [40000, 40001], 8, 128, 64)
    qd, q = rounded(torch, rng.normal(0, 1, (3, 16, 128)), "f32")
    got = Call(torch, fbctx, B, qd, None, "f32", 16).result(0.09)
    check(got, attention(q, B, None, 0.09), q, B, 0.09, "f32")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_scales_of_either_sign_and_none(fbctx, torch_cuda, kind):
    torch = torch_cuda
    rng = np.random.default_rng(19)
    B = Batch(rng, [9, 2], [500, 64], 2, 128, 64)
    qd, q = rounded(torch, rng.normal(0, 1, (11, 8, 128)), kind)
    mask = tree_mask(rng, B.new, 1)
    for scale in (-0.09, 0.0):
        got = Call(torch, fbctx, B, qd, mask, kind, 8).result(scale)
        check(got, attention(q, B, mask, scale), q, B, abs(scale), kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_equal_values_come_out_as_they_are(fbctx, torch_cuda, kind):
    """Every key has the same value row, of numbers that each type holds: their mean, however the weights are rounded."""
    torch = torch_cuda
    rng = np.random.default_rng(20)
    B = Batch(rng, [12, 3], [3000, 130], 2, 128, 64)
    row = rng.integers(-255, 256, 128) / 64.0
    B.v[:] = row
    qd, q = rounded(torch, 1.5 * rng.normal(0, 1, (15, 8, 128)), kind)
    got = Call(torch, fbctx, B, qd, None, kind, 8).result(0.09)
    np.testing.assert_allclose(got, np.broadcast_to(row, got.shape), rtol=2.0 ** -18 if kind == "f32" else 0, atol=0)
