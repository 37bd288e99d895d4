"""One verification step as a program uses it: a prompt appended and extended
by drafted trees, rotated queries, tree attention, logits, sampled tokens, the
accepted path appended again -- against the same steps in binary64."""
import math

import numpy as np
import pytest

import ferrite_b200 as fb
from tree_reference import Batch, attention, frequencies, rotate, rounded, sample, tree_mask

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE, VOCAB = 8, 2, 128, 64, 1000


def test_verification_step(fbctx, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(21)
    prompts, drafts = [70, 5, 130], [6, 9, 1]
    lens = [a + b for a, b in zip(prompts, drafts)]
    B = Batch(rng, drafts, lens, KV, DIM, PAGE)
    mask = tree_mask(rng, drafts, 1)
    r = fb.Rotary(64, 1e6, 1)
    freq, amp = frequencies(64, 1e6)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    kp, vp, bt = t(B.k), t(B.v), t(B.table)
    width = (HEADS + 2 * KV) * DIM

    def rows_of(counts):
        d, held = rounded(torch, rng.normal(0, 1, (sum(counts), width)), "f32")
        q = held[:, :HEADS * DIM].reshape(-1, HEADS, DIM)
        kv = held[:, HEADS * DIM:].reshape(-1, 2, KV, DIM)
        return d, q, kv[:, 0], kv[:, 1]

    def append(d, counts, upto, pos):
        off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        od, ld, pd = t(off), t(np.array(upto, np.int32)), t(pos.astype(np.int32))
        base = d.data_ptr() + HEADS * DIM * 4
        fb.kv_append(fbctx, r, fb.F32, base, width, base + KV * DIM * 4, width, od.data_ptr(), ld.data_ptr(), pd.data_ptr(),
                     bt.data_ptr(), kp.data_ptr(), vp.data_ptr(), 3, int(off[-1]), max(counts), KV, DIM, PAGE, B.max_pages,
                     B.num_pages)
        return od, ld, pd

    def store(k, v, counts, upto, pos):  # the same into the reference's pages
        turned = rotate(k, pos, freq, amp, 1)
        row = 0
        for b, c in enumerate(counts):
            for i in range(c):
                pg, s = B.place(b, upto[b] - c + i)
                B.k[pg, :, :, s] = turned[row]
                B.v[pg, :, s] = v[row]
                row += 1

    # prompts
    pd_rows, _, pk, pv = rows_of(prompts)
    ppos = np.concatenate([np.arange(n) for n in prompts])
    append(pd_rows, prompts, prompts, ppos)
    store(pk, pv, prompts, prompts, ppos)
    # drafted trees: a token's position is its depth behind the prompt
    dd, q, k, v = rows_of(drafts)
    depth = np.array([bin(int(m[0])).count("1") - 1 for m in mask])
    pos = np.concatenate([[p] * n for p, n in zip(prompts, drafts)]) + depth
    od, ld, posd = append(dd, drafts, lens, pos)
    store(k, v, drafts, lens, pos)
    total = sum(drafts)
    turned = torch.empty(total, HEADS, DIM, device="cuda")
    fb.rotary_apply(fbctx, r, fb.F32, dd.data_ptr(), width, DIM, turned.data_ptr(), HEADS * DIM, DIM, posd.data_ptr(), total,
                    HEADS, DIM)
    out = torch.empty_like(turned)
    ws = torch.empty(max(16, fb.attn_tree_workspace(fbctx, 3, 9, HEADS, KV, DIM, PAGE, max(lens))), dtype=torch.uint8,
                     device="cuda")
    scale = 1 / math.sqrt(DIM)
    md = t(mask.view(np.int32))
    fb.attn_tree(fbctx, fb.F32, turned.data_ptr(), HEADS * DIM, kp.data_ptr(), vp.data_ptr(), bt.data_ptr(), od.data_ptr(),
                 ld.data_ptr(), md.data_ptr(), 1, out.data_ptr(), HEADS * DIM, 3, total, 9, HEADS, KV, DIM, PAGE,
                 B.max_pages, B.num_pages, max(lens), scale, ws.data_ptr(), ws.numel())
    # a head of the model's: logits, one token a row
    w = torch.randn(HEADS * DIM, VOCAB, device="cuda", dtype=torch.float64)
    logits = (out.double().reshape(total, -1) @ w).float()
    u = t(rng.random(total).astype(np.float32))
    top_p = torch.full((total,), 0.9, device="cuda")
    tokens = torch.empty(total, dtype=torch.int32, device="cuda")
    fb.sample_rows(fbctx, fb.F32, logits.data_ptr(), VOCAB, total, VOCAB, 0, 0, top_p.data_ptr(), 0, u.data_ptr(),
                   tokens.data_ptr())
    # every step above in binary64; fp16 keys and values rounded the same way
    want = attention(rotate(q, pos, freq, amp, 1), B, mask, scale)
    got = out.double().cpu().numpy()
    # the pages' fp16 keys may round either way: half a step of 2^-11 in a key moves a score by 2^-11 of its products at
    # most in the few entries on a border; the rows' 2-norm keeps to that against the score size of 3
    assert np.linalg.norm(got - want) <= 3 * 2.0 ** -11 * np.linalg.norm(want)
    lg = logits.double().cpu().numpy()
    tp = float(np.float32(0.9))
    assert tokens.tolist() == [sample(lg[i], 1.0, 0, tp, 0.0, float(u[i]))[0] for i in range(total)]
    # the longest path of each tree accepted: its rows again, now in a line behind the prompt
    paths = []
    for b in range(3):
        rows = range(B.offsets[b], B.offsets[b + 1])
        best = max(rows, key=lambda i: depth[i])
        paths.append([int(B.offsets[b]) + j for j in range(drafts[b]) if (int(mask[best, 0]) >> j) & 1])
    counts = [len(p) for p in paths]
    pick = np.concatenate(paths)
    upto = [p + c for p, c in zip(prompts, counts)]
    again = dd[torch.from_numpy(pick).cuda()].contiguous()
    append(again, counts, upto, pos[pick])
    store(k[pick], v[pick], counts, upto, pos[pick])
    line = Batch.__new__(Batch)
    line.__dict__.update(B.__dict__, new=counts, lens=upto, total=sum(counts),
                         offsets=np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
    chain_q = rounded(torch, rotate(q[pick], pos[pick], freq, amp, 1), "f32")
    out2 = torch.empty(line.total, HEADS, DIM, device="cuda")
    od, ld = t(line.offsets), t(np.array(upto, np.int32))
    fb.attn_tree(fbctx, fb.F32, chain_q[0].data_ptr(), HEADS * DIM, kp.data_ptr(), vp.data_ptr(), bt.data_ptr(),
                 od.data_ptr(), ld.data_ptr(), 0, 1, out2.data_ptr(), HEADS * DIM, 3, line.total, 9, HEADS, KV, DIM, PAGE,
                 B.max_pages, B.num_pages, max(lens), scale, ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    assert fbctx.error_word() == 0
    # an accepted path sees the same keys in a line as it saw in the tree
    np.testing.assert_allclose(out2.double().cpu().numpy(), got[pick], atol=2e-5)
    want = attention(chain_q[1], line, None, scale)
    assert np.linalg.norm(out2.double().cpu().numpy() - want) <= 3 * 2.0 ** -11 * np.linalg.norm(want)
