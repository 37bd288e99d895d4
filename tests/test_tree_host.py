"""Host side of the tree verification operators, without a GPU: rotary
frequencies against their definition, and the refusals (raised before any
device work)."""
import numpy as np
import pytest

import ferrite_b200 as fb
from tree_reference import frequencies

SCALINGS = {"plain": fb.ROTARY_PLAIN, "linear": fb.ROTARY_LINEAR, "bands": fb.ROTARY_BANDS, "yarn": fb.ROTARY_YARN}


@pytest.mark.parametrize("kw", [
    dict(rot=128, theta=1e6),
    dict(rot=2, theta=1e4),
    dict(rot=40, theta=1e4, scaling="linear", factor=4.0),
    dict(rot=128, theta=5e5, scaling="bands", factor=8.0, orig_ctx=8192, low=1.0, high=4.0),
    dict(rot=64, theta=1e4, scaling="yarn", factor=16.0, orig_ctx=2048, low=1.0, high=32.0),
    dict(rot=128, theta=1e6, scaling="yarn", factor=4.0, orig_ctx=32768, low=1.0, high=32.0, amplitude=1.25),
    dict(rot=64, theta=1e4, scaling="yarn", factor=2.0, orig_ctx=4, low=1.0, high=2.0),  # both ramp ends at pair 0
])
def test_frequencies(kw):
    want, amp = frequencies(**kw)
    d = dict(kw)
    r = fb.Rotary(d.pop("rot"), d.pop("theta"), scaling=SCALINGS[d.pop("scaling", "plain")], **d)
    got, gamp = r.frequencies()
    # a power, a logarithm and a few products in binary64 on both sides
    np.testing.assert_allclose(got, want, rtol=1e-13)
    assert abs(gamp - amp) < 1e-14


@pytest.mark.parametrize("kw,msg", [
    (dict(rot_dim=3, theta=1e4), "rot_dim"), (dict(rot_dim=0, theta=1e4), "rot_dim"),
    (dict(rot_dim=258, theta=1e4), "rot_dim"), (dict(rot_dim=64, theta=1.0), "theta"),
    (dict(rot_dim=64, theta=float("nan")), "theta"), (dict(rot_dim=64, theta=1e4, mode=2), "mode"),
    (dict(rot_dim=64, theta=1e4, scaling=4), "scaling"), (dict(rot_dim=64, theta=1e4, scaling=1, factor=0.0), "factor"),
    (dict(rot_dim=64, theta=1e4, scaling=2, factor=8.0, low=1.0, high=4.0), "orig_ctx"),
    (dict(rot_dim=64, theta=1e4, scaling=3, factor=8.0, orig_ctx=8192, low=4.0, high=4.0), "low"),
    (dict(rot_dim=64, theta=1e4, amplitude=-1.0), "amplitude"),
])
def test_rotary_create_refuses(kw, msg):
    with pytest.raises(fb.FerriteError, match=msg):
        fb.Rotary(**kw)


class NoContext:
    h = None


A = 1 << 20  # an address no refused call reads


def rotary_args(**over):
    d = dict(dtype=fb.F32, x_ptr=A, x_token_stride=512, x_head_stride=128, y_ptr=2 * A, y_token_stride=512,
             y_head_stride=128, positions_ptr=A, n_tok=2, n_heads=4, head_dim=128)
    d.update(over)
    return d


@pytest.mark.parametrize("over,msg", [
    (dict(dtype=fb.Q4_K), "dtype"), (dict(n_tok=-1), "bad shape"), (dict(n_heads=0), "bad shape"),
    (dict(head_dim=1025), "bad shape"), (dict(head_dim=32), "rot_dim exceeds"), (dict(y_head_stride=64), "overlap"),
    (dict(y_token_stride=100), "overlap"), (dict(x_token_stride=-1), "negative"),
    (dict(y_ptr=A, y_token_stride=1024), "equal strides"), (dict(), "null argument"),
])
def test_rotary_apply_refuses(over, msg):
    with pytest.raises(fb.FerriteError, match=msg):
        fb.rotary_apply(NoContext, fb.Rotary(64, 1e4), **rotary_args(**over))


def append_args(**over):
    d = dict(dtype=fb.F32, k_ptr=A, k_token_stride=1024, v_ptr=A, v_token_stride=1024, row_offsets_ptr=A,
             seq_lens_ptr=A, positions_ptr=0, bt_ptr=A, k_pages_ptr=A, v_pages_ptr=A, batch=2, n_rows=4, max_new=3,
             n_kv=8, head_dim=128, page_size=64, max_pages=4, num_pages=9)
    d.update(over)
    return d


@pytest.mark.parametrize("over,msg", [
    (dict(dtype=fb.Q8_K), "dtype"), (dict(head_dim=96), "head_dim"), (dict(page_size=16), "page_size"),
    (dict(batch=-1), "bad shape"), (dict(batch=70000), "bad shape"), (dict(n_kv=0), "bad shape"),
    (dict(max_new=257), "max_new exceeds"), (dict(max_pages=1 << 25), "too long"),
    (dict(k_token_stride=-8), "negative"), (dict(), "null argument"),
])
def test_kv_append_refuses(over, msg):
    with pytest.raises(fb.FerriteError, match=msg):
        fb.kv_append(NoContext, None, **append_args(**over))


def test_kv_append_refuses_wide_rotation():
    with pytest.raises(fb.FerriteError, match="rot_dim exceeds"):
        fb.kv_append(NoContext, fb.Rotary(128, 1e4), **append_args(head_dim=64))


def tree_args(**over):
    d = dict(dtype=fb.F32, q_ptr=A, q_token_stride=4096, k_ptr=A, v_ptr=A, bt_ptr=A, row_offsets_ptr=A, seq_lens_ptr=A,
             mask_ptr=A, mask_words=2, out_ptr=A, out_token_stride=4096, batch=2, n_rows=60, max_new=40, n_heads=32,
             n_kv=8, head_dim=128, page_size=64, max_pages=4, num_pages=9, max_seq_len=256, scale=0.1)
    d.update(over)
    return d


@pytest.mark.parametrize("over,msg", [
    (dict(dtype=fb.Q4_K), "dtype"), (dict(head_dim=80), "head_dim"), (dict(page_size=128), "page_size"),
    (dict(n_heads=33), "multiple"), (dict(batch=-1), "bad shape"), (dict(max_seq_len=257), "max_seq_len exceeds"),
    (dict(mask_words=1), "mask_words"), (dict(out_token_stride=100), "token stride"),
    (dict(scale=float("inf")), "scale"), (dict(), "null argument"),
])
def test_attn_tree_refuses(over, msg):
    with pytest.raises(fb.FerriteError, match=msg):
        fb.attn_tree(NoContext, **tree_args(**over))


def sample_args(**over):
    d = dict(dtype=fb.F32, logits_ptr=A, row_stride=1000, rows=2, vocab=1000, temperature_ptr=0, top_k_ptr=0,
             top_p_ptr=0, min_p_ptr=0, uniform_ptr=A, tokens_ptr=A)
    d.update(over)
    return d


@pytest.mark.parametrize("over,msg", [
    (dict(dtype=fb.Q4_K), "dtype"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 19) + 1), "vocab"),
    (dict(rows=-1), "rows"), (dict(row_stride=999), "row_stride"), (dict(), "null argument"),
])
def test_sample_rows_refuses(over, msg):
    with pytest.raises(fb.FerriteError, match=msg):
        fb.sample_rows(NoContext, **sample_args(**over))


@pytest.mark.parametrize("tok,head,fits", [(512, 128, True), (128, 256, True), (511, 128, False), (128, 255, False),
                                           (256, 128, False), (1 << 40, 128, True), (200, 150, False)])
def test_rotary_rows_that_overlap(tok, head, fits):
    """Two tokens of four heads, 128 wide: nested strides reach the next check, others are refused."""
    with pytest.raises(fb.FerriteError, match="null argument" if fits else "overlap"):
        fb.rotary_apply(NoContext, fb.Rotary(64, 1e4), **rotary_args(y_token_stride=tok, y_head_stride=head))


def test_rotary_refuses_a_vanishing_factor():
    with pytest.raises(fb.FerriteError, match="factor"):
        fb.Rotary(64, 1e4, scaling=1, factor=1e-300)


def test_nothing_to_do_needs_no_device():
    fb.rotary_apply(NoContext, fb.Rotary(64, 1e4), **rotary_args(n_tok=0))
    fb.kv_append(NoContext, None, **append_args(n_rows=0))
    fb.attn_tree(NoContext, **tree_args(batch=0))
    fb.sample_rows(NoContext, **sample_args(rows=0))


@pytest.mark.parametrize("factor", [0.25, 0.5, 0.999, 1.0])
def test_yarn_amplitude_of_factors_up_to_one(factor):
    """0.1 ln(factor) + 1 below a factor of one too."""
    kw = dict(factor=factor, orig_ctx=4096, low=1.0, high=32.0)
    want, amp = frequencies(64, 1e4, "yarn", **kw)
    got, gamp = fb.Rotary(64, 1e4, scaling=fb.ROTARY_YARN, **kw).frequencies()
    np.testing.assert_allclose(got, want, rtol=1e-13)
    assert abs(gamp - amp) < 1e-14 and (amp < 1.0 or factor == 1.0)


def test_yarn_refuses_an_amplitude_of_nothing():
    """0.1 ln(factor) + 1 reaches 0 at e^-10; an amplitude given replaces it."""
    kw = dict(scaling=fb.ROTARY_YARN, factor=4e-5, orig_ctx=4096, low=1.0, high=32.0)
    with pytest.raises(fb.FerriteError, match="amplitude"):
        fb.Rotary(64, 1e4, **kw)
    assert fb.Rotary(64, 1e4, amplitude=1.5, **kw).frequencies()[1] == 1.5


def test_a_closed_rotary_handle_is_refused():
    r = fb.Rotary(64, 1e4)
    r.close()
    with pytest.raises(fb.FerriteError, match="closed"):
        fb.kv_append(NoContext, r, **append_args(n_rows=0))
    with pytest.raises(fb.FerriteError, match="rotary"):
        fb.rotary_apply(NoContext, r, **rotary_args())


class AnyContext:
    h = A  # never read by a refused call


@pytest.mark.parametrize("over", [
    dict(y_ptr=A + 4), dict(y_ptr=A - 4 * 127), dict(y_ptr=A + 4 * 512),  # shifted by a value, almost a head, a token
    dict(y_ptr=A + 4 * 128 * 3, n_tok=1),
    dict(y_ptr=A + 4 * 1000, x_token_stride=1024, y_token_stride=1024),  # 24 values into the next token
    dict(y_ptr=A + 4 * 100, x_token_stride=256, x_head_stride=1024, y_token_stride=256, y_head_stride=1024),
    dict(y_ptr=A + 4 * 512, x_token_stride=1024, y_token_stride=512),    # unequal strides over the same memory
    dict(dtype=fb.F16, y_ptr=A + 2 * 127, n_tok=1, n_heads=1),
])
def test_rotary_apply_refuses_overlap(over):
    with pytest.raises(fb.FerriteError, match="x and y overlap"):
        fb.rotary_apply(AnyContext, fb.Rotary(64, 1e4), **rotary_args(**over))


@pytest.mark.parametrize("over", [
    dict(out_ptr=A), dict(out_ptr=A + 4 * 4095), dict(out_ptr=A - 4 * 4095), dict(out_ptr=A + 4 * 4096 * 59),
    dict(q_token_stride=8192, out_token_stride=8192, out_ptr=A + 4 * 8192 * 30 + 4 * 4095),
    dict(q_token_stride=8192, out_token_stride=4096, out_ptr=A + 4 * 4096),
    dict(q_token_stride=0, out_ptr=A + 16), dict(n_rows=1, q_token_stride=1, out_token_stride=0, out_ptr=A + 4 * 100),
])
def test_attn_tree_refuses_overlap(over):
    with pytest.raises(fb.FerriteError, match="q and out must not overlap"):
        fb.attn_tree(AnyContext, **tree_args(**{"q_ptr": A, **over}))
