"""Definitions in binary64 of the tree verification operators (rotary
positions, cache append, tree attention, row sampling), and seeded inputs."""
from __future__ import annotations

import math

import numpy as np

# half a step of each type, relative to the value
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def torch_type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def fb_type(fb, name):
    return {"f32": fb.F32, "f16": fb.F16, "bf16": fb.BF16}[name]


def rounded(torch, x, kind):
    """x (numpy f64) as a device tensor of a type, and the values it holds."""
    t = torch.from_numpy(np.ascontiguousarray(x)).to(torch_type(torch, kind))
    return t.cuda(), t.double().numpy()


def frequencies(rot, theta, scaling="plain", factor=1.0, orig_ctx=0, low=0.0, high=0.0, amplitude=0.0):
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    amp = amplitude or 1.0
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "bands":
        out = []
        for x in f:
            wave = 2 * math.pi / x
            if wave < orig_ctx / high:
                out.append(x)
            elif wave > orig_ctx / low:
                out.append(x / factor)
            else:
                s = (orig_ctx / wave - low) / (high - low)
                out.append((1 - s) * x / factor + s * x)
        f = out
    elif scaling == "yarn":
        def at(turns):
            return rot * math.log(orig_ctx / (turns * 2 * math.pi)) / (2 * math.log(theta))
        a, b = max(math.floor(at(high)), 0), min(math.ceil(at(low)), rot - 1)
        g = [min(max((i - a) / max(b - a, 0.001), 0.0), 1.0) for i in range(rot // 2)]
        f = [x / factor * r + x * (1 - r) for x, r in zip(f, g)]
        amp = amplitude or 0.1 * math.log(factor) + 1.0
    return np.array(f), amp


def rotate(x, positions, freq, amp, mode):
    """x [tokens, heads, dim] (f64) turned at positions."""
    rot = 2 * len(freq)
    y = x.copy()
    a = positions.astype(np.float64)[:, None] * freq[None]
    c, s = (amp * np.cos(a))[:, None], (amp * np.sin(a))[:, None]
    i0, i1 = (slice(0, rot, 2), slice(1, rot, 2)) if mode == 0 else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def pair_size(x, rot, amp, mode):
    """|x0| + |x1| of every dimension's pair, times the amplitude (0 behind the rotated part)."""
    m = np.zeros_like(x)
    i0, i1 = (slice(0, rot, 2), slice(1, rot, 2)) if mode == 0 else (slice(0, rot // 2), slice(rot // 2, rot))
    m[..., i0] = m[..., i1] = amp * (np.abs(x[..., i0]) + np.abs(x[..., i1]))
    return m


class Batch:
    """A ragged batch over shuffled pages."""

    def __init__(self, rng, new, lens, heads, dim, page, spare=2, kv=None):
        self.new, self.lens, self.heads, self.dim, self.page = list(new), list(lens), heads, dim, page
        self.batch, self.total = len(new), sum(new)
        self.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        need = [-(-n // page) for n in lens]
        self.max_pages = max(need + [1]) + 1
        self.num_pages = sum(need) + spare
        order = rng.permutation(self.num_pages).astype(np.int32)
        self.table = np.full((self.batch, self.max_pages), -1, np.int32)  # entries past the end are never read
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k = rng.normal(0, 1, (self.num_pages, heads, dim, page)).astype(np.float16)
        self.v = rng.normal(0, 1, (self.num_pages, heads, page, dim)).astype(np.float16)

    def place(self, b, pos):
        return self.table[b, pos // self.page], pos % self.page


def tree_mask(rng, new, words):
    """Ancestor bits of random trees, uint32 [rows, words]."""
    rows = []
    for n in new:
        bits = []
        for i in range(n):
            parent = int(rng.integers(-1, i)) if i else -1
            bits.append((bits[parent] if parent >= 0 else 0) | (1 << i))
        rows += bits
    return np.array([[(r >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for r in rows], np.uint32).reshape(-1, words)


def attention(q, B, mask, scale, bad_pages=()):
    """out [rows, heads, dim] f64 (q f64 [rows, heads, dim]); mask None: a chain."""
    qh = q.shape[1]
    out = np.zeros(q.shape)
    for b in range(B.batch):
        n, length = B.new[b], B.lens[b]
        if n == 0:
            continue
        pages = B.table[b, : -(-length // B.page)]
        k = np.concatenate([B.k[p] for p in pages], 2)[:, :, :length].astype(np.float64)
        v = np.concatenate([B.v[p] for p in pages], 1)[:, :length].astype(np.float64)
        good = np.repeat([p not in bad_pages for p in range(len(pages))], B.page)[:length]
        for i in range(n):
            row, pre = B.offsets[b] + i, length - n
            see = np.ones(length, bool)
            for j in range(n):
                see[pre + j] = j <= i if mask is None else (int(mask[row, j // 32]) >> (j % 32)) & 1
            see &= good
            if not see.any():
                continue
            for h in range(qh):
                kv = h // (qh // B.heads)
                s = scale * (q[row, h] @ k[kv][:, see])
                p = np.exp(s - s.max())
                out[row, h] = p @ v[kv][see] / p.sum()
    return out


def sample(x, t, top_k, top_p, min_p, u):
    """(token, probability) of one row (f64 logits; settings as f32 values)."""
    ok = ~np.isnan(x)
    if not ok.any():
        return -1, 0.0
    mx = x[ok].max()
    if t <= 0:
        return int(np.flatnonzero(ok & (x == mx))[0]), 1.0
    if mx == -np.inf:
        return -1, 0.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == mx, 1.0, np.exp((x - mx) / t))
    w = np.where(ok & (x > -np.inf), w, 0.0)
    if np.isinf(mx):
        w = (x == mx).astype(np.float64)
    order = np.argsort(-np.where(ok, x, -np.inf), kind="stable")
    down = w[order]
    n = x.size
    if min_p > 0:
        n = int((down >= min(float(min_p), 1.0)).sum())
    if top_p < 1:
        mass = np.cumsum(down[:n])
        n = min(n, int((mass < max(float(top_p), 0.0) * mass[-1]).sum()) + 1)
    if top_k > 0:
        n = min(n, int(top_k))
    kept = np.sort(order[:n])
    mass = np.cumsum(w[kept])
    u = min(max(float(u), 0.0), 1.0)
    hit = np.flatnonzero(mass > u * mass[-1])
    i = hit[0] if hit.size else np.flatnonzero(w[kept] > 0)[-1]
    return int(kept[i]), float(w[kept[i]] / mass[-1])
