"""Rotary positions and the cache append against their definitions in binary64.

Tolerances count roundings.  A rotated value is x0 c - x1 s: the angle's
remainder (2^-28 turns = 2.4e-8 rad), sincospi (one unit, 2^-24 relative to
1), the amplitude and the products (2^-24 each) and the sum: at most 6 * 2^-24
of A (|x0| + |x1|).  Then half a step of the output type, and for fp16 half of
the smallest subnormal."""
import numpy as np
import pytest

import ferrite_b200 as fb
from tree_reference import HALF_STEP, Batch, fb_type, frequencies, pair_size, rotate, rounded, torch_type

pytestmark = pytest.mark.gpu

SCALE = {"plain": (fb.ROTARY_PLAIN, {}), "linear": (fb.ROTARY_LINEAR, dict(factor=4.0)),
         "bands": (fb.ROTARY_BANDS, dict(factor=8.0, orig_ctx=8192, low=1.0, high=4.0)),
         "yarn": (fb.ROTARY_YARN, dict(factor=4.0, orig_ctx=4096, low=1.0, high=32.0))}


def bound(want, size, kind):
    out = 0.0 if kind == "f32" else HALF_STEP[kind] * np.abs(want) * (1 + 2.0 ** -7)
    return 6 * 2.0 ** -24 * size + out + (2.0 ** -25 if kind == "f16" else 1e-37)


def check(got, want, size, kind, what=""):
    err = np.abs(got - want) - bound(want, size, kind)
    assert (err <= 0).all(), f"{what}: over the bound by {err.max()} at {np.unravel_index(err.argmax(), err.shape)}"


# tokens, heads, dim, rot, mode, scaling, type, (gap in the token stride, offset of the first value)
CASES = [
    (1, 32, 128, 128, 1, "plain", "f32", 0, 0), (1, 1, 64, 64, 0, "plain", "f16", 0, 0),
    (3, 8, 128, 128, 0, "bands", "f32", 2048, 0), (17, 5, 128, 64, 1, "yarn", "bf16", 0, 0),
    (33, 40, 80, 40, 1, "linear", "f16", 8, 0), (9, 3, 96, 48, 0, "linear", "bf16", 0, 0),
    (5, 2, 20, 10, 1, "plain", "f32", 0, 0), (5, 2, 21, 6, 0, "plain", "bf16", 3, 1), (4, 3, 6, 2, 1, "plain", "f16", 0, 0),
    (7, 1, 1024, 256, 1, "plain", "f16", 0, 0), (300, 4, 256, 256, 0, "yarn", "f32", 0, 0),
    (700, 1, 64, 32, 1, "bands", "f32", 0, 0), (64, 300, 64, 64, 1, "plain", "bf16", 0, 0), (2, 8, 128, 128, 1, "plain", "f32", 0, 1),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("inplace", [False, True])
def test_rotary_apply(fbctx, torch_cuda, case, inplace):
    torch = torch_cuda
    tok, heads, dim, rot, mode, scaling, kind, gap, start = case
    rng = np.random.default_rng(sum(case[:4]))
    width = heads * dim + gap
    flat, held = rounded(torch, rng.normal(0, 2, start + tok * width), kind)
    pos = rng.integers(-50, 1 << 20, tok).astype(np.int32)
    pos[0] = 2 ** 31 - 1 if tok > 2 else pos[0]
    kindid, kw = SCALE[scaling]
    r = fb.Rotary(rot, 5e5, mode, kindid, **kw)
    freq, amp = frequencies(rot, 5e5, scaling, **kw)
    x = held[start:].reshape(tok, width)[:, :heads * dim].reshape(tok, heads, dim)
    pd = torch.from_numpy(pos).cuda()
    esz = flat.element_size()
    if inplace:
        y, yt = flat, width
        yp = flat.data_ptr() + start * esz
    else:
        y = torch.full((tok * heads * dim + 16,), 7.0, dtype=torch_type(torch, kind), device="cuda")
        yt, yp = heads * dim, y.data_ptr()
    fb.rotary_apply(fbctx, r, fb_type(fb, kind), flat.data_ptr() + start * esz, width, dim, yp, yt, dim, pd.data_ptr(), tok,
                    heads, dim)
    torch.cuda.synchronize()
    got = y.double().cpu().numpy()
    if inplace:
        full = got[start:].reshape(tok, width)
        assert np.array_equal(full[:, heads * dim:], held[start:].reshape(tok, width)[:, heads * dim:])
        out = full[:, :heads * dim].reshape(tok, heads, dim)
    else:
        assert (got[tok * heads * dim:] == 7.0).all()
        out = got[:tok * heads * dim].reshape(tok, heads, dim)
    want = rotate(x, pos, freq, amp, mode)
    assert np.array_equal(out[..., rot:], x[..., rot:])
    check(out, want, pair_size(x, rot, amp, mode), kind)


def test_rotary_head_major_strides(fbctx, torch_cuda):
    """Heads outermost: head stride above the token stride."""
    torch = torch_cuda
    rng = np.random.default_rng(3)
    xd, held = rounded(torch, rng.normal(0, 1, (4, 9, 128)), "f32")
    pos = np.arange(9, dtype=np.int32)[::-1].copy()
    y = torch.empty_like(xd)
    fb.rotary_apply(fbctx, fb.Rotary(128, 1e4, 0), fb.F32, xd.data_ptr(), 128, 9 * 128, y.data_ptr(), 128, 9 * 128,
                    torch.from_numpy(pos).cuda().data_ptr(), 9, 4, 128)
    torch.cuda.synchronize()
    x = held.transpose(1, 0, 2)
    freq, amp = frequencies(128, 1e4)
    check(y.double().cpu().numpy().transpose(1, 0, 2), rotate(x, pos, freq, amp, 0), pair_size(x, 128, amp, 0), "f32")


def test_rotary_turns_back(fbctx, torch_cuda):
    """Positions p, then -p: the values come back within two rotations' bound."""
    torch = torch_cuda
    xd, x = rounded(torch, np.random.default_rng(4).normal(0, 1, (50, 8, 128)), "f32")
    pos = torch.arange(0, 50 * 40961, 40961, dtype=torch.int32, device="cuda")
    r = fb.Rotary(128, 1e6)
    for p in (pos, -pos):
        fb.rotary_apply(fbctx, r, fb.F32, xd.data_ptr(), 1024, 128, xd.data_ptr(), 1024, 128, p.data_ptr(), 50, 8, 128)
    torch.cuda.synchronize()
    assert (np.abs(xd.double().cpu().numpy() - x) <= 2 * 1.5 * 6 * 2.0 ** -24 * pair_size(x, 128, 1.0, 1)).all()


def test_rotary_leaves_nan_in_its_pair(fbctx, torch_cuda):
    torch = torch_cuda
    x = torch.ones(2, 2, 64, device="cuda")
    x[0, 1, 3], x[1, 0, 63] = float("nan"), float("inf")
    pos = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    y = torch.empty_like(x)
    fb.rotary_apply(fbctx, fb.Rotary(32, 1e4), fb.F32, x.data_ptr(), 128, 64, y.data_ptr(), 128, 64, pos.data_ptr(), 2, 2, 64)
    torch.cuda.synchronize()
    bad = ~torch.isfinite(y)
    assert bad.nonzero().tolist() == [[0, 1, 3], [0, 1, 19], [1, 0, 63]]


# new rows, lens, heads, dim, page, rot, mode, type
APPENDS = [
    ([1], [1], 8, 128, 64, 128, 1, "f32"), ([1, 1, 1], [64, 65, 4000], 8, 128, 64, 128, 0, "f16"),
    ([7, 0, 25, 1], [7, 300, 90, 32], 2, 64, 32, 64, 1, "bf16"), ([130], [130], 1, 128, 64, 64, 0, "f32"),
    ([200, 63], [263, 64], 3, 64, 64, 0, 1, "f16"), ([33], [96], 8, 128, 32, 20, 1, "bf16"), ([0, 0], [10, 0], 1, 64, 32, 64, 1, "f32"),
    ([64, 128, 1], [64, 192, 129], 5, 128, 64, 128, 1, "bf16"), ([40] * 40, [100] * 40, 8, 64, 32, 64, 0, "f32"),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{c[7]}")
@pytest.mark.parametrize("own_positions,start", [(True, 0), (False, 1)])
def test_kv_append(fbctx, torch_cuda, case, own_positions, start):
    torch = torch_cuda
    new, lens, heads, dim, page, rot, mode, kind = case
    rng = np.random.default_rng(sum(new) + page)
    B = Batch(rng, new, lens, heads, dim, page)
    width = heads * dim
    n = B.total + 2  # rows behind the last sequence belong to nobody
    flat, held = rounded(torch, rng.normal(0, 2, start + n * 2 * width), kind)
    rows = held[start:].reshape(n, 2, heads, dim)
    place = np.concatenate([np.arange(l - m, l) for m, l in zip(new, lens)] + [np.zeros(0, int)]).astype(np.int32)
    pos = rng.integers(0, 1 << 17, n).astype(np.int32) if own_positions else None
    t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    kd, vd, bt, off, ln = t(B.k.copy()), t(B.v.copy()), t(B.table), t(B.offsets), t(np.array(lens, np.int32))
    pd = t(pos) if own_positions else None
    r = fb.Rotary(rot, 1e5, mode) if rot else None
    at = flat.data_ptr() + start * flat.element_size()
    fb.kv_append(fbctx, r, fb_type(fb, kind), at, 2 * width, at + width * flat.element_size(), 2 * width, off.data_ptr(),
                 ln.data_ptr(), pd.data_ptr() if own_positions else 0, bt.data_ptr(), kd.data_ptr(), vd.data_ptr(),
                 B.batch, n, max(new) if max(new) else 1, heads, dim, page, B.max_pages, B.num_pages)
    torch.cuda.synchronize()
    assert fbctx.error_word() == 0
    gk, gv = kd.double().cpu().numpy(), vd.double().cpu().numpy()
    freq, amp = frequencies(rot, 1e5) if rot else (np.zeros(0), 1.0)
    p = pos[:B.total] if own_positions else place
    wk = rotate(rows[:B.total, 0], p, freq, amp, mode)
    size = pair_size(rows[:B.total, 0], rot, amp, mode)
    touched = np.zeros((B.num_pages, page), bool)
    for b in range(B.batch):
        for i in range(new[b]):
            row = B.offsets[b] + i
            pg, s = B.place(b, lens[b] - new[b] + i)
            touched[pg, s] = True
            check(gk[pg, :, :, s], wk[row], size[row], "f16", f"k row {row}")
            assert np.array_equal(gv[pg, :, s], rows[row, 1].astype(np.float16).astype(np.float64))
    keep = ~touched
    assert np.array_equal(gk.transpose(0, 3, 1, 2)[keep], B.k.astype(np.float64).transpose(0, 3, 1, 2)[keep])
    assert np.array_equal(gv.transpose(0, 2, 1, 3)[keep], B.v.astype(np.float64).transpose(0, 2, 1, 3)[keep])


def test_kv_append_leaves_bad_sequences_out(fbctx, torch_cuda):
    """Offsets out of order, lengths below the new rows or past the block table,
    page ids outside the pool: nothing is written for them, the others are."""
    torch = torch_cuda
    rng = np.random.default_rng(8)
    good = Batch(rng, [3, 3, 3, 3], [70, 70, 70, 70], 2, 64, 64)
    x = torch.randn(12, 2, 64, device="cuda")
    t = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731

    def go(offsets, lens, table, n_rows=12, max_new=3):
        kd, vd = torch.from_numpy(good.k.copy()).cuda(), torch.from_numpy(good.v.copy()).cuda()
        off, ln, bt = t(offsets), t(lens), t(table)
        fb.kv_append(fbctx, None, fb.F32, x.data_ptr(), 128, x.data_ptr(), 128, off.data_ptr(), ln.data_ptr(), 0,
                     bt.data_ptr(), kd.data_ptr(), vd.data_ptr(), 4, n_rows, max_new, 2, 64, 64, good.max_pages,
                     good.num_pages)
        torch.cuda.synchronize()
        changed = (kd.cpu().numpy() != good.k).any(axis=(1, 2)) | (vd.cpu().numpy() != good.v).any(axis=(1, 3))
        return fbctx.error_word(), changed  # [page, slot]

    ok = np.zeros((good.num_pages, 64), bool)
    for b in range(4):
        ok[good.table[b, 1], 3:6] = True
    word, changed = go([0, 3, 6, 9, 12], [70] * 4, good.table)
    assert word == 0 and np.array_equal(changed, ok)
    some = ok.copy()
    some[good.table[1, 1]] = False
    for offsets, lens, kw in [([0, 3, 6, 9, 12], [70, 2, 70, 70], {}), ([0, 3, 6, 9, 12], [70, good.max_pages * 64 + 1, 70, 70], {}),
                              ([0, 3, 6, 9, 12], [70, -70, 70, 70], {})]:
        word, changed = go(offsets, lens, good.table, **kw)
        assert word == 4 and np.array_equal(changed, some), (offsets, lens)
    word, changed = go([0, 3, -6, 9, 12], [70] * 4, good.table)  # two sequences lose their rows
    assert word == 4 and changed[good.table[0, 1], 3:6].all() and not changed[good.table[1, 1]].any() and not changed[good.table[2, 1]].any()
    word, changed = go([0, 3, 6, 9, 12], [70] * 4, good.table, n_rows=11)
    last = ok.copy()
    last[good.table[3, 1]] = False
    assert word == 4 and np.array_equal(changed, last)
    for page in (-1, good.num_pages, 2 ** 31 - 1):
        table = good.table.copy()
        table[1, 1] = page
        word, changed = go([0, 3, 6, 9, 12], [70] * 4, table)
        assert word == 8 and np.array_equal(changed, some)
