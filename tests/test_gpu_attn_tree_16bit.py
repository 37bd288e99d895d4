"""The hard cases of tree attention in 16-bit types, whose kernel has a softmax of
its own: lazily rescaled accumulators, one tile whose blocks two groups take in
turn and merge, or two tiles.  Each case runs in both forms (`new` rows of 4 heads
a kv head: up to 128 rows, above) and both page sizes.  Bounds as in the f32 cases."""
import numpy as np
import pytest

import ferrite_b200 as fb
from test_gpu_attn_tree import Call, check
from tree_reference import Batch, attention, rounded, tree_mask

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("kind", ["f16", "bf16"])
FORMS = pytest.mark.parametrize("new,page", [(9, 64), (9, 32), (45, 64), (45, 32)])


@TYPES
@FORMS
@pytest.mark.parametrize("step", [9.0, 40.0])
@pytest.mark.parametrize("order", ["rising", "falling", "by turns"])
@pytest.mark.parametrize("batch,heads,length", [(2, 1, 250), (3, 8, 1500)])
def test_maxima_that_move_from_block_to_block(fbctx, torch_cuda, kind, new, page, step, order, batch, heads, length):
    """Scores whose 64-key blocks lie `step` powers of two apart: rising ones rescale the accumulator at every block
    (above 8), falling ones never, and some rows of a warp do it while others do not.  The short sequences are four blocks
    of one CTA; the longer ones are four or five blocks a CTA, joined."""
    torch = torch_cuda
    rng = np.random.default_rng(new + page)
    B = Batch(rng, [new] * batch, [length - 40 * b for b in range(batch)], heads, 64, page)
    at = np.arange(-(-length // 64))
    level = {"rising": at, "falling": -at, "by turns": at * (at % 3)}[order]
    # dimension 0 of every key carries its block's level, the queries' dimension 0 what it counts: 0, 1 or 2 a row
    for b in range(batch):
        for p in range(B.lens[b]):
            pg, s = B.place(b, p)
            B.k[pg, :, 0, s] = level[p // 64]
    mask = tree_mask(rng, B.new, 2)
    qv = rng.normal(0, 1, (B.total, 4 * heads, 64))
    qv[..., 0] = step / (0.125 * 1.4426950408889634) * rng.integers(0, 3, qv.shape[:2])
    qd, q = rounded(torch, qv, kind)
    got = Call(torch, fbctx, B, qd, mask, kind, 4 * heads, words=2).result(0.125)
    check(got, attention(q, B, mask, 0.125), q, B, 0.125, kind)
    assert fbctx.error_word() == 0


@TYPES
@FORMS
def test_sharp_softmax(fbctx, torch_cuda, kind, new, page):
    """Scores that span hundreds: one key holds the row, late maxima replace early ones."""
    torch = torch_cuda
    rng = np.random.default_rng(10)
    B = Batch(rng, [new, 3], [1024, 260], 2, 128, page)
    qd, q = rounded(torch, 12 * rng.normal(0, 1, (new + 3, 8, 128)), kind)
    mask = tree_mask(rng, B.new, 2)
    got = Call(torch, fbctx, B, qd, mask, kind, 8, words=2).result(0.25)
    check(got, attention(q, B, mask, 0.25), q, B, 0.25, kind)


@TYPES
@FORMS
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("prefix", [0, 70, 700])
def test_what_a_row_does_not_see_never_reaches_it(fbctx, torch_cuda, kind, new, page, value, prefix):
    """Non-finite k and v behind the end of the last page and at drafted rows that others do not descend from; rows that
    see such a v get its value.  In whole groups, and in ones that several CTAs share."""
    torch = torch_cuda
    rng = np.random.default_rng(6)
    end = prefix + new
    B = Batch(rng, [new], [end], 1, 128, page)
    mask = np.zeros((new, 2), np.uint32)
    for i in range(new):  # siblings under row 0
        mask[i, 0] |= 1
        mask[i, i // 32] |= np.uint32(1 << (i % 32))
    for slot in range(end, -(-end // page) * page):
        pg, s = B.place(0, slot)
        B.k[pg, :, :, s] = value
        B.v[pg, :, s] = value
    qd, q = rounded(torch, rng.normal(0, 1, (new, 4, 128)), kind)
    want = attention(q, B, mask, 0.1)
    odd_k, odd_v = 4, new - 3
    pg, s = B.place(0, prefix + odd_k)
    B.k[pg, :, :, s] = value
    pg, s = B.place(0, prefix + odd_v)
    B.v[pg, 0, s, 17] = value
    B.v[pg, 0, s, 100] = value
    got = Call(torch, fbctx, B, qd, mask, kind, 4, words=2).result(0.1)
    others = [i for i in range(new) if i not in (odd_k, odd_v)]
    check(got[others], want[others], q[others], B, 0.1, kind)
    assert not np.isfinite(got[odd_v][:, [17, 100]]).any()
    rest = [d for d in range(128) if d not in (17, 100)]
    check(got[[odd_v]][..., rest], want[[odd_v]][..., rest], q[[odd_v]], B, 0.1, kind)


@TYPES
@FORMS
def test_nan_in_one_query_stays_in_its_row(fbctx, torch_cuda, kind, new, page):
    torch = torch_cuda
    rng = np.random.default_rng(7)
    B = Batch(rng, [new], [333], 2, 64, page)
    qd, q = rounded(torch, rng.normal(0, 1, (new, 8, 64)), kind)
    want = attention(q, B, None, 0.125)
    qd[2, 1, 9] = float("nan")
    qd[new - 1, 7, 63] = float("nan")
    got = Call(torch, fbctx, B, qd, None, kind, 8).result(0.125)
    for row, head in ((2, 1), (new - 1, 7)):
        assert np.isnan(got[row, head]).all()
        got[row, head] = want[row, head]
    check(got, want, q, B, 0.125, kind)


@TYPES
@FORMS
@pytest.mark.parametrize("prefix", [400, 3000])
def test_shared_and_bad_pages(fbctx, torch_cuda, kind, new, page, prefix):
    """Two sequences over the same prefix pages; then page ids outside the pool, first and last ones among them, and every
    page of a sequence."""
    torch = torch_cuda
    rng = np.random.default_rng(12)
    n = prefix + new
    B = Batch(rng, [new, new], [n, n], 1, 128, page)
    B.table[1, :3] = B.table[0, :3]
    mask = tree_mask(rng, B.new, 2)
    qd, q = rounded(torch, rng.normal(0, 1, (2 * new, 4, 128)), kind)
    got = Call(torch, fbctx, B, qd, mask, kind, 4, words=2).result(0.1)
    check(got, attention(q, B, mask, 0.1), q, B, 0.1, kind)
    assert fbctx.error_word() == 0
    last = -(-n // page) - 1
    bad = (0, 2, 5, last)
    want = attention(q, B, mask, 0.1, bad_pages=bad)
    for j, p in zip(bad, (-1, B.num_pages, 2 ** 30, -2 ** 31)):
        B.table[:, j] = p
    got = Call(torch, fbctx, B, qd, mask, kind, 4, words=2).result(0.1)
    assert fbctx.error_word() == 8
    check(got, want, q, B, 0.1, kind)
    B.table[1] = -1
    got = Call(torch, fbctx, B, qd, mask, kind, 4, words=2).result(0.1)
    assert fbctx.error_word() == 8
    check(got[:new], want[:new], q[:new], B, 0.1, kind)
    assert (got[new:] == 0).all()


@TYPES
@FORMS
def test_bad_sequences_are_left_out(fbctx, torch_cuda, kind, new, page):
    torch = torch_cuda
    rng = np.random.default_rng(13)
    B = Batch(rng, [new] * 3, [90] * 3, 2, 64, page)
    qd, q = rounded(torch, rng.normal(0, 1, (3 * new, 8, 64)), kind)
    want = attention(q, B, None, 0.125)
    keep = list(range(new)) + list(range(2 * new, 3 * new))
    for lens in ([90, new - 1, 90], [90, 91, 90], [90, -1, 90]):
        c = Call(torch, fbctx, B, qd, None, kind, 8)
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        got = c.result(0.125)
        assert fbctx.error_word() == 4
        assert (got[new:2 * new] == 7.0).all()
        check(got[keep], want[keep], q[keep], B, 0.125, kind)


@TYPES
@FORMS
@pytest.mark.parametrize("scale", [0.125, -0.125])
def test_strided_misaligned_queries(fbctx, torch_cuda, kind, new, page, scale):
    """q inside fused rows, and q, out off 16-byte boundaries."""
    torch = torch_cuda
    rng = np.random.default_rng(11)
    B = Batch(rng, [new, 3], [130, 66], 2, 64, page)
    rows, row = new + 3, 8 * 64
    for start, width in ((0, row + 256), (1, row + 1), (3, row + 8)):
        flat, held = rounded(torch, rng.normal(0, 1, start + rows * width), kind)
        q = held[start:].reshape(rows, width)[:, :row].reshape(rows, 8, 64)
        buf = torch.full((rows * row + 8,), 7.0, device="cuda", dtype=flat.dtype)
        c = Call(torch, fbctx, B, flat[start:], None, kind, 8, out=buf[start:])
        c.go(scale, q_stride=width)
        torch.cuda.synchronize()
        got = buf.double().cpu().numpy()
        assert (got[start + rows * row:] == 7.0).all() and (got[:start] == 7.0).all()
        check(got[start:start + rows * row].reshape(rows, 8, 64), attention(q, B, None, scale), q, B, abs(scale), kind)
