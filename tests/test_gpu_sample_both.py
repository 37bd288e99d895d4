"""fb_sample and fb_sample_rows on the same rows: without a repetition penalty,
which the row sampler does not have, the same random number draws the same token.

fb_sample's weights are f32 (relative errors of 10^-6 at these logits), the row
sampler's exact: a draw differs where u comes within that of a border, one in some
ten thousand of these; the seeded ones do not."""
import numpy as np
import pytest

import ferrite_b200 as fb
from oracle import sampling as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cfg", [
    dict(), dict(temperature=0.0), dict(temperature=1.0, top_p=1.0, min_p=0.0, top_k=40),
    dict(temperature=1.0, top_p=0.95, min_p=0.0), dict(temperature=1.3, top_p=1.0, min_p=0.1),
    dict(temperature=1.5, top_p=0.8, top_k=100, min_p=0.02), dict(temperature=0.5, top_p=0.5, top_k=3, min_p=0.0),
])
@pytest.mark.parametrize("vocab", [4096, 151936])
def test_the_same_token(fbctx, torch_cuda, vocab, cfg):
    torch = torch_cuda
    cfg = {**dict(temperature=0.7, top_p=0.9, top_k=0, min_p=0.05), **cfg}
    rows = 16
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 2.0, (rows, vocab)).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, vocab, 5)] += 7.0
    xd = torch.from_numpy(x).cuda()
    one = fb.Sampler(fbctx, repetition_penalty=1.0, seed=99, **cfg)
    want, u, state = [], [], 99
    for r in range(rows):
        want.append(one.sample(xd[r].data_ptr(), vocab, [1, 2, 3]))
        if cfg["temperature"] > 0:
            state, draw = S.xorshift64(state)
            u.append(draw)
        else:
            u.append(0.0)
    assert one.state.value == state
    a = lambda v, dt: torch.full((rows,), v, dtype=dt, device="cuda")  # noqa: E731
    t, k, p, m = (a(cfg["temperature"], torch.float32), a(cfg["top_k"], torch.int32), a(cfg["top_p"], torch.float32),
                  a(cfg["min_p"], torch.float32))
    ud, tok = torch.tensor(u, dtype=torch.float32, device="cuda"), a(-9, torch.int32)
    fb.sample_rows(fbctx, fb.F32, xd.data_ptr(), vocab, rows, vocab, t.data_ptr(), k.data_ptr(), p.data_ptr(), m.data_ptr(),
                   ud.data_ptr(), tok.data_ptr())
    assert tok.tolist() == want
