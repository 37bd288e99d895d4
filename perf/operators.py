"""Cases of the operators that verify a batch of drafted token trees over the
paged cache: rotary positions, the cache append, tree attention and row
sampling.  Each has a plain form in elementary torch operations, a definition
in 64 bits, and the calls of the ferrite_b200 package."""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode token of the 32-head model, q of a fused projection row
        dict(name="rotary one token", op="rotary", tokens=1, heads=32, dim=128, rot=128, mode="half", scaling="plain",
             type="f32", far=4096, fused=True),
        # an odd count of tokens of a long-context model that rotates half of each head, far positions
        dict(name="rotary half head far", op="rotary", tokens=777, heads=64, dim=128, rot=64, mode="interleaved",
             scaling="bands", type="bf16", far=1000000, fused=False),
        # a 2048-token prompt of the 32-head model, scaled context
        dict(name="rotary prompt", op="rotary", tokens=2048, heads=32, dim=128, rot=128, mode="half", scaling="yarn",
             type="f16", far=65536, fused=True),
        # the drafted trees of a decode batch: a few new tokens a sequence
        dict(name="append drafts", op="append", batch=16, new=25, context=4096, heads=8, dim=128, page=64, rot=128,
             mode="half", type="f32"),
        # three prompts of unequal length written at once
        dict(name="append prompts", op="append", batch=3, new=2731, context=4096, heads=8, dim=128, page=64, rot=128,
             mode="interleaved", type="bf16"),
        # the smallest verification: one short sequence, a few drafts
        dict(name="tree short", op="tree", batch=1, new=7, context=190, qheads=32, heads=8, dim=128, page=64,
             type="f32"),
        # one sequence at the 4096-token context, a tree of 60
        dict(name="tree 4096", op="tree", batch=1, new=60, context=4096, qheads=32, heads=8, dim=128, page=64,
             type="f32"),
        # a decode batch of unequal contexts
        dict(name="tree batch ragged", op="tree", batch=16, new=25, context=4096, qheads=32, heads=8, dim=128, page=32,
             type="f16"),
        # long contexts of the 64-head model
        dict(name="tree long", op="tree", batch=4, new=40, context=32000, qheads=64, heads=8, dim=128, page=64,
             type="bf16"),
        # one row with the sampler's default settings
        dict(name="sample one row", op="sample", rows=1, vocab=151936, type="f32", top_k=0, top_p=0.9, min_p=0.05,
             hidden=0.0, spread=2.5),
        # the rows of a drafted tree under a grammar mask, nucleus only: a wide kept set
        dict(name="sample masked tree", op="sample", rows=65, vocab=128256, type="f32", top_k=0, top_p=0.95, min_p=0.0,
             hidden=0.3, spread=2.0),
        # every row of a large batch of trees, top-k and top-p together
        dict(name="sample batch", op="sample", rows=400, vocab=151936, type="bf16", top_k=50, top_p=0.9, min_p=0.0,
             hidden=0.0, spread=2.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "tree", "tree", "sample"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        return dict(op=op, tokens=_log_int(rng, 1, 2500), heads=rng.choice([1, 5, 8, 32, 40]), dim=dim,
                    rot=rng.choice([dim, dim // 2]), mode=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["plain", "linear", "bands", "yarn"]), type=kind, far=_log_int(rng, 512, 2000000),
                    fused=rng.choice([True, False]))
    if op == "append":
        dim = rng.choice([64, 128])
        return dict(op=op, batch=_log_int(rng, 1, 24), new=_log_int(rng, 1, 300), context=_log_int(rng, 400, 9000),
                    heads=rng.choice([1, 2, 8]), dim=dim, page=rng.choice([32, 64]), rot=rng.choice([0, dim // 2, dim]),
                    mode=rng.choice(["half", "interleaved"]), type=kind)
    if op == "tree":
        heads = rng.choice([1, 2, 4, 8])
        return dict(op=op, batch=_log_int(rng, 1, 16), new=_log_int(rng, 1, 64), context=_log_int(rng, 70, 7900),
                    qheads=heads * rng.choice([1, 2, 4, 5, 8]), heads=heads, dim=rng.choice([64, 128]),
                    page=rng.choice([32, 64]), type=kind)
    return dict(op=op, rows=_log_int(rng, 1, 200), vocab=_log_int(rng, 1000, 200000), type=kind,
                top_k=rng.choice([0, 1, 20, 200]), top_p=rng.choice([1.0, 0.95, 0.5]), min_p=rng.choice([0.0, 0.02, 0.1]),
                hidden=rng.choice([0.0, 0.5]), spread=rng.choice([1.0, 2.5, 4.0]))


# ----------------------------------------------------------------- inputs
def _scaling(case):
    """The settings of each scaled form, as a checkpoint's configuration gives them."""
    return {"plain": dict(scaling="plain", theta=1e6),
            "linear": dict(scaling="linear", theta=1e4, factor=4.0),
            "bands": dict(scaling="bands", theta=5e5, factor=8.0, context=8192, low=1.0, high=4.0),
            "yarn": dict(scaling="yarn", theta=1e6, factor=4.0, context=32768, low=1.0, high=32.0)}[case["scaling"]]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(case):
    """Ragged sequences: new rows and cache lengths (new rows included), host lists.  Part of the case: outputs keep their shapes."""
    b, most, ctx = case["batch"], case["new"], case["context"]
    c = torch.Generator()
    c.manual_seed(b * most + ctx)
    if b == 1:
        return [most], [ctx]
    new = torch.randint((most + 1) // 2, most + 1, (b,), generator=c).tolist()
    new[-1] = most
    lens = torch.randint((ctx + 3) // 4, ctx + 1, (b,), generator=c).tolist()
    lens[0] = ctx
    return new, [max(n, l) for n, l in zip(new, lens)]


def _cache(case, lens, g):
    """Pools of shuffled pages with some spare ones, and the block table."""
    page, heads, dim = case["page"], case["heads"], case["dim"]
    need = [-(-n // page) for n in lens]
    total, most = sum(need) + 3, max(need) + 1
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), most, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    k = torch.randn(total, heads, dim, page, generator=g, device="cuda", dtype=torch.float16)
    v = torch.randn(total, heads, page, dim, generator=g, device="cuda", dtype=torch.float16)
    return k, v, table


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(new):
    off = [0]
    for n in new:
        off.append(off[-1] + n)
    return _int32(off)


def _trees(new, words, seed):
    """Drafted trees: each token's parent is an earlier one or the last verified token; a bit for every ancestor and itself."""
    c = torch.Generator()
    c.manual_seed(seed)
    rows = []
    for n in new:
        parent = (torch.rand(n, generator=c) * (torch.arange(n) + 1)).long().tolist()
        bits = []
        for i in range(n):
            bits.append((bits[parent[i] - 1] if parent[i] else 0) | (1 << i))
        rows += bits
    flat = [[(r >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for r in rows]
    return torch.tensor([[x - (1 << 32) if x >> 31 else x for x in r] for r in flat], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op = case["op"]
    if op == "rotary":
        kind, t, h, d = _TYPES[case["type"]], case["tokens"], case["heads"], case["dim"]
        wide = (h + 16) * d if case["fused"] else h * d  # a fused row holds k and v behind q
        s["x"] = torch.randn(t, wide, generator=g, device="cuda").to(kind)
        s["positions"] = torch.randint(0, case["far"], (t,), generator=g, device="cuda", dtype=torch.int32)
        s["y"] = torch.empty(t, h, d, device="cuda", dtype=kind)
    elif op == "append":
        kind = _TYPES[case["type"]]
        new, lens = _rows(case)
        s["lens"], s["offsets"], s["total"] = _int32(lens), _offsets(new), sum(new)
        s["kpool"], s["vpool"], s["table"] = _cache(case, lens, g)
        s["kv"] = torch.randn(sum(new), 2, case["heads"], case["dim"], generator=g, device="cuda").to(kind)
        # drafted siblings share a position: the rotary position is not the place in the cache
        place = torch.cat([torch.arange(l - n, l) for n, l in zip(new, lens)])
        s["positions"] = (place // 2).to(torch.int32).cuda()
    elif op == "tree":
        kind = _TYPES[case["type"]]
        new, lens = _rows(case)
        s["lens"], s["offsets"], s["total"] = _int32(lens), _offsets(new), sum(new)
        s["kpool"], s["vpool"], s["table"] = _cache(case, lens, g)
        s["words"] = (case["new"] + 31) // 32
        s["mask"] = _trees(new, s["words"], seed)
        s["q"] = (1.5 * torch.randn(sum(new), case["qheads"], case["dim"], generator=g, device="cuda")).to(kind)
        s["out"] = torch.empty_like(s["q"])
    else:
        kind, r, v = _TYPES[case["type"]], case["rows"], case["vocab"]
        x = case["spread"] * torch.randn(r, v, generator=g, device="cuda")
        if case["hidden"]:
            x = x.masked_fill(torch.rand(r, v, generator=g, device="cuda") < case["hidden"], -math.inf)
        s["logits"] = x.to(kind)
        s["uniform"] = torch.rand(r, generator=g, device="cuda")
        s["temperature"] = 0.5 + torch.rand(r, generator=g, device="cuda")
        s["temperature"][r // 2 + 1::7] = 0.0  # some greedy requests in a batch
        s["top_k"] = torch.full((r,), case["top_k"], dtype=torch.int32, device="cuda")
        s["top_p"] = torch.full((r,), case["top_p"], device="cuda")
        s["min_p"] = torch.full((r,), case["min_p"], device="cuda")
        s["tokens"] = torch.empty(r, dtype=torch.int32, device="cuda")
        s["probs"] = torch.empty(r, device="cuda")
    return s


# ----------------------------------------------------------- plain forms
def _frequencies(rot, scaling, theta, factor=1.0, context=0, low=0.0, high=0.0):
    """Radians a position for each rotated pair, and what cos and sin are scaled by (64 bits)."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(-2.0 * i / rot * math.log(theta))
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "bands":
        turns = context * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return f * keep + f / factor * (1 - keep), 1.0
    if scaling == "yarn":
        first, last = (rot * math.log(context / (2 * math.pi * b)) / (2 * math.log(theta)) for b in (high, low))
        first, last = max(math.floor(first), 0), min(math.ceil(last), rot - 1)
        ramp = ((i - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rotate(x, positions, rot, mode, setting):
    """x [tokens, heads, dim] in 32 bits; angles in 64."""
    if rot == 0:
        return x
    f, amp = _frequencies(rot, **setting)
    angle = positions.double()[:, None] * f
    cos, sin = ((t(angle) * amp).float()[:, None, :] for t in (torch.cos, torch.sin))
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if mode == "interleaved" else (x[..., :rot // 2], x[..., rot // 2:rot])
    p, q = a * cos - b * sin, a * sin + b * cos
    if mode == "interleaved":
        y[..., 0:rot:2], y[..., 1:rot:2] = p, q
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = p, q
    return y


def _places(s):
    """For every new row: its sequence and its place in the cache."""
    off, row = s["offsets"].long(), torch.arange(s["total"], device="cuda")
    b = torch.searchsorted(off, row, right=True) - 1
    return b, s["lens"].long()[b] - (off[b + 1] - row)


def _plain_rotary(s):
    x = s["x"][:, :s["heads"] * s["dim"]].reshape(s["tokens"], s["heads"], s["dim"]).float()
    return _rotate(x, s["positions"], s["rot"], s["mode"], _scaling(s)).to(s["x"].dtype)


def _plain_append(s):
    b, place = _places(s)
    page, inside = s["table"].long()[b, place // s["page"]], place % s["page"]
    k = _rotate(s["kv"][:, 0].float(), s["positions"], s["rot"], s["mode"], _scaling({"scaling": "plain"}))
    s["kpool"][page, :, :, inside] = k.half()
    s["vpool"][page, :, inside, :] = s["kv"][:, 1].half()
    return s["kpool"], s["vpool"]


def _plain_tree(s):
    batch, page, heads, dim, most = s["batch"], s["page"], s["heads"], s["dim"], s["new"]
    group, total = s["qheads"] // heads, s["total"]
    pages = s["table"].long()[:, :-(-s["context"] // page)]
    k = s["kpool"][pages].permute(0, 2, 3, 1, 4).reshape(batch, heads, dim, -1).float()
    v = s["vpool"][pages].permute(0, 2, 1, 3, 4).reshape(batch, heads, -1, dim).float()
    off, lens = s["offsets"].long(), s["lens"].long()
    b, _ = _places(s)
    i = torch.arange(total, device="cuda") - off[b]
    q = torch.zeros(batch, heads, most, group, dim, device="cuda")
    q[b, :, i] = s["q"].float().reshape(total, heads, group, dim)
    x = torch.matmul(q.reshape(batch, heads, most * group, dim), k).mul_(1.0 / math.sqrt(dim))
    # visible: the prefix, and the drafted tokens whose bit is set
    place = torch.arange(k.shape[-1], device="cuda")[None]
    first = (lens - (off[1:] - off[:-1]))[:, None]
    j = (place - first).clamp(0, most - 1)
    bits = torch.zeros(batch, most, s["words"], dtype=torch.int32, device="cuda")
    bits[b, i] = s["mask"]
    drafted = (torch.gather(bits, 2, (j // 32)[:, None].expand(-1, most, -1)) >> (j % 32)[:, None].int()) & 1
    see = (place < first)[:, None] | ((place < lens[:, None])[:, None] & (drafted != 0))
    x = x.view(batch, heads, most, group, -1).masked_fill_(~see[:, None, :, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    v = torch.where((place < lens[:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(x.view(batch, heads, most * group, -1), v).view(batch, heads, most, group, dim)
    total_p = x.sum(-1, keepdim=True)
    o = torch.where(total_p > 0, o / total_p, torch.zeros_like(o))
    return o[b, :, i].reshape(total, s["qheads"], dim).to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    down, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((down - down[:, :1]) / t)
    floor = s["min_p"].double()[:, None]
    w1 = torch.where(w >= floor, w, torch.zeros_like(w))
    before = torch.cumsum(w1, 1) - w1
    top_p = s["top_p"].double()[:, None]
    keep = (w >= floor) & ((before < top_p * w1.sum(1, keepdim=True)) | (top_p >= 1))
    rank = torch.arange(vocab, device="cuda")[None]
    k = s["top_k"].long()[:, None]
    keep &= (k <= 0) | (rank < k)
    keep &= ~greedy[:, None] | (rank < 1)
    keep[:, 0] = True
    p = torch.zeros_like(x).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))
    mass = torch.cumsum(p, 1)
    token = (mass > s["uniform"].double()[:, None] * mass[:, -1:]).int().argmax(1, keepdim=True)
    prob = torch.gather(p, 1, token) / mass[:, -1:]
    return token[:, 0].int(), prob[:, 0].float()


# --------------------------------------------------- the framework's calls
def _package():
    at = os.path.join(_ROOT, "ferrite-llm_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ferrite_b200
    return ferrite_b200


def _context(fb, s):
    if "context_handle" not in s:
        s["context_handle"] = fb.Context(0, torch.cuda.current_stream().cuda_stream)
    return s["context_handle"]


def _rotary_handle(fb, s, setting):
    if "rotary" not in s:
        kinds = {"plain": fb.ROTARY_PLAIN, "linear": fb.ROTARY_LINEAR, "bands": fb.ROTARY_BANDS, "yarn": fb.ROTARY_YARN}
        mode = 0 if s["mode"] == "interleaved" else 1
        s["rotary"] = fb.Rotary(s["rot"], setting["theta"], mode, kinds[setting["scaling"]], setting.get("factor", 1.0),
                                setting.get("context", 0), setting.get("low", 0.0), setting.get("high", 0.0)) if s["rot"] else None
    return s["rotary"]


def _dtype(fb, s):
    return {"f32": fb.F32, "f16": fb.F16, "bf16": fb.BF16}[s["type"]]


def _own_rotary(s):
    fb = _package()
    ctx, d = _context(fb, s), s["dim"]
    fb.rotary_apply(ctx, _rotary_handle(fb, s, _scaling(s)), _dtype(fb, s), s["x"].data_ptr(), s["x"].shape[1], d,
                    s["y"].data_ptr(), s["heads"] * d, d, s["positions"].data_ptr(), s["tokens"], s["heads"], d)
    return s["y"]


def _own_append(s):
    fb = _package()
    ctx = _context(fb, s)
    rotary = _rotary_handle(fb, s, _scaling({"scaling": "plain"}))
    row = s["heads"] * s["dim"]
    kv = s["kv"].data_ptr()
    fb.kv_append(ctx, rotary, _dtype(fb, s), kv, 2 * row, kv + row * s["kv"].element_size(), 2 * row,
                 s["offsets"].data_ptr(), s["lens"].data_ptr(), s["positions"].data_ptr(), s["table"].data_ptr(),
                 s["kpool"].data_ptr(), s["vpool"].data_ptr(), s["batch"], s["total"], s["new"], s["heads"], s["dim"],
                 s["page"], s["table"].shape[1], s["kpool"].shape[0])
    return s["kpool"], s["vpool"]


def _own_tree(s):
    fb = _package()
    ctx = _context(fb, s)
    row = s["qheads"] * s["dim"]
    if "workspace" not in s:
        n = fb.attn_tree_workspace(ctx, s["batch"], s["new"], s["qheads"], s["heads"], s["dim"], s["page"], s["context"])
        s["workspace"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    fb.attn_tree(ctx, _dtype(fb, s), s["q"].data_ptr(), row, s["kpool"].data_ptr(), s["vpool"].data_ptr(),
                 s["table"].data_ptr(), s["offsets"].data_ptr(), s["lens"].data_ptr(), s["mask"].data_ptr(), s["words"],
                 s["out"].data_ptr(), row, s["batch"], s["total"], s["new"], s["qheads"], s["heads"], s["dim"], s["page"],
                 s["table"].shape[1], s["kpool"].shape[0], s["context"], 1.0 / math.sqrt(s["dim"]),
                 s["workspace"].data_ptr(), s["workspace"].numel())
    return s["out"]


def _own_sample(s):
    fb = _package()
    ctx = _context(fb, s)
    fb.sample_rows(ctx, _dtype(fb, s), s["logits"].data_ptr(), s["vocab"], s["rows"], s["vocab"], s["temperature"].data_ptr(),
                   s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["uniform"].data_ptr(),
                   s["tokens"].data_ptr(), s["probs"].data_ptr())
    return s["tokens"], s["probs"]


def run(state):
    op = state["op"]
    if own:
        call = {"rotary": _own_rotary, "append": _own_append, "tree": _own_tree, "sample": _own_sample}[op]
    else:
        call = {"rotary": _plain_rotary, "append": _plain_append, "tree": _plain_tree, "sample": _plain_sample}[op]
    return call(state)


# ------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    op = case["op"]
    if op == "rotary":
        values = case["tokens"] * case["heads"] * case["dim"]
        return dict(bytes=2 * values * size + 4 * case["tokens"],
                    flops=3 * case["tokens"] * case["heads"] * case["rot"])
    if op == "sample":
        return dict(bytes=case["rows"] * (case["vocab"] * size + 28), flops=4 * case["rows"] * case["vocab"])
    # the ragged lengths of a batch, at their mean
    b = case["batch"]
    new = case["new"] if b == 1 else (0.75 * case["new"] * (b - 1) + case["new"])
    if op == "append":
        values = new * case["heads"] * case["dim"]
        return dict(bytes=values * 2 * (size + 2), flops=3 * new * case["heads"] * case["rot"])
    keys = case["context"] if b == 1 else (0.625 * case["context"] * (b - 1) + case["context"])
    q = new * case["qheads"] * case["dim"]
    return dict(bytes=keys * case["heads"] * case["dim"] * 4 + 2 * q * size + new * 4 * ((case["new"] + 31) // 32),
                flops=4 * q * keys / b)


# ------------------------------------------------------------- definition
def exact(case, seed):
    """The operator's definition in 64 bits, one sequence (or row) after another."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        x = s["x"].double()[:, :case["heads"] * case["dim"]].reshape(case["tokens"], case["heads"], case["dim"])
        return _turned(x, s["positions"], case["rot"], case["mode"], _scaling(case))
    if op == "append":
        k = _turned(s["kv"][:, 0].double(), s["positions"], case["rot"], case["mode"], _scaling({"scaling": "plain"}))
        kpool, vpool, off, lens = s["kpool"].double(), s["vpool"].double(), s["offsets"].tolist(), s["lens"].tolist()
        for b in range(case["batch"]):
            n = off[b + 1] - off[b]
            at = torch.arange(lens[b] - n, lens[b], device="cuda")
            page = s["table"][b].long()[at // case["page"]]
            kpool[page, :, :, at % case["page"]] = k[off[b]:off[b + 1]]
            vpool[page, :, at % case["page"], :] = s["kv"][off[b]:off[b + 1], 1].double()
        return kpool, vpool
    if op == "tree":
        off, lens, out = s["offsets"].tolist(), s["lens"].tolist(), []
        for b in range(case["batch"]):
            n, length = off[b + 1] - off[b], lens[b]
            page = s["table"][b, :-(-length // case["page"])].long()
            k = s["kpool"][page].permute(1, 0, 3, 2).reshape(case["heads"], -1, case["dim"])[:, :length].double()
            v = s["vpool"][page].permute(1, 0, 2, 3).reshape(case["heads"], -1, case["dim"])[:, :length].double()
            see = torch.ones(n, length, dtype=torch.bool, device="cuda")
            for j in range(n):
                see[:, length - n + j] = (s["mask"][off[b]:off[b + 1], j // 32] >> (j % 32)) & 1 != 0
            for h in range(case["qheads"]):
                kv = h // (case["qheads"] // case["heads"])
                x = s["q"][off[b]:off[b + 1], h].double() @ k[kv].T / math.sqrt(case["dim"])
                out.append(torch.softmax(x.masked_fill(~see, -math.inf), 1) @ v[kv])
        pieces, at = [], 0
        for b in range(case["batch"]):
            pieces.append(torch.stack(out[at:at + case["qheads"]], 1))
            at += case["qheads"]
        return torch.cat(pieces)
    tokens, probs = [], []
    for r in range(case["rows"]):
        x, t = s["logits"][r].double(), float(s["temperature"][r])
        if t <= 0:
            best = x.max()
            tokens.append(int((x == best).nonzero()[0]))
            probs.append(1.0)
            continue
        w = ((x - x.max()) / t).exp()
        order = torch.argsort(-x, stable=True)
        n = int((w >= float(s["min_p"][r])).sum())
        if float(s["top_p"][r]) < 1:
            mass = torch.cumsum(w[order[:n]], 0)
            n = int((mass < float(s["top_p"][r]) * mass[-1]).sum()) + 1
        n = min(n, case["top_k"]) if case["top_k"] > 0 else n
        kept = order[:n].sort().values
        mass = torch.cumsum(w[kept], 0)
        i = int((mass > float(s["uniform"][r]) * float(mass[-1])).nonzero()[0])
        tokens.append(int(kept[i]))
        probs.append(float(w[kept[i]] / mass[-1]))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)


def _turned(x, positions, rot, mode, setting):
    """Each rotated pair as a complex number times amp * e^(i pos f)."""
    if rot == 0:
        return x
    freq = []
    theta, s = setting["theta"], setting.get("factor", 1.0)
    amp = 0.1 * math.log(s) + 1.0 if setting["scaling"] == "yarn" else 1.0
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        if setting["scaling"] == "linear":
            f /= s
        elif setting["scaling"] == "bands":
            wave = 2 * math.pi / f
            if wave > setting["context"] / setting["low"]:
                f /= s
            elif wave >= setting["context"] / setting["high"]:
                m = (setting["context"] / wave - setting["low"]) / (setting["high"] - setting["low"])
                f = (1 - m) * f / s + m * f
        elif setting["scaling"] == "yarn":
            at = [rot * math.log(setting["context"] / (2 * math.pi * setting[b])) / (2 * math.log(theta)) for b in ("high", "low")]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
            m = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f / s * m + f * (1 - m)
        freq.append(f)
    angle = positions.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, amp), angle)[:, None]
    y = x.clone()
    if mode == "interleaved":
        z = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:2], rot // 2, 2).contiguous()) * turn
        y[..., :rot] = torch.view_as_real(z).reshape(*x.shape[:2], rot)
    else:
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * turn
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    return y
