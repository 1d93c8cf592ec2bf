"""The operators of the paged KV cache: rotary positions stored into pages, attention of new rows over pages, and the
pages' own upkeep (reserve, fork, release, compact), as a serving loop calls them.

``own`` false computes them with elementary torch operations, in 32 bits (positions' angles in 64), rounded once at the end;
``own`` true makes the calls of ``allpaka_b200.gpu``.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

_GPU = None


def _gpu():
    """The process's one context of the framework."""
    global _GPU
    from allpaka_b200 import gpu

    if _GPU is None:
        _GPU = gpu.Gpu(0)
    return gpu, _GPU


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one token of one session in the framework's own activation type, far into its context: pure latency
        dict(name="rope_one_token", op="rope", dtype="f32", cache="f16", heads=64, kv=8, dim=128, page=16, n=1, rows_lo=1, rows_hi=1,
             len_lo=32000, len_hi=32768, rot=128, layout="half", scaling="none", factor=1.0, norms=False, mix=1),
        # a ragged batch of chunks, neighbouring pairs, half of the head, stretched context
        dict(name="rope_chunks_yarn", op="rope", dtype="bf16", cache="bf16", heads=32, kv=4, dim=128, page=16, n=7, rows_lo=1, rows_hi=1003,
             len_lo=1003, len_hi=40000, rot=64, layout="pairs", scaling="yarn", factor=4.0, norms=False, mix=2),
        # a whole prompt's layer, with the per-head norms in front
        dict(name="rope_prompt", op="rope", dtype="f16", cache="f16", heads=64, kv=8, dim=128, page=64, n=1, rows_lo=8192, rows_hi=8192,
             len_lo=8192, len_hi=8192, rot=128, layout="half", scaling="linear", factor=2.0, norms=True, mix=3),
        # the next token of one short session, 32-bit rows: latency
        dict(name="attend_one_short", op="attend", dtype="f32", cache="f16", heads=64, kv=8, dim=128, page=16, n=1, rows_lo=1, rows_hi=1,
             len_lo=512, len_hi=512, causal=True, window=0, mix=4),
        # drafts being verified, 32-bit rows: five rows a session
        dict(name="attend_verify", op="attend", dtype="f32", cache="f16", heads=40, kv=8, dim=128, page=32, n=6, rows_lo=5, rows_hi=5,
             len_lo=900, len_hi=6001, causal=True, window=0, mix=5),
        # the next token of a batch of sessions whose lengths differ by a factor of forty
        dict(name="attend_batch", op="attend", dtype="f16", cache="f16", heads=32, kv=8, dim=128, page=64, n=64, rows_lo=1, rows_hi=1,
             len_lo=200, len_hi=8192, causal=True, window=0, mix=6),
        # the next token of one very long session
        dict(name="attend_one_long", op="attend", dtype="bf16", cache="bf16", heads=64, kv=8, dim=128, page=64, n=1, rows_lo=1, rows_hi=1,
             len_lo=131077, len_hi=131077, causal=True, window=0, mix=7),
        # prompts in pieces beside sessions that decode, a sliding window, small heads in groups of seven
        dict(name="attend_mixed_window", op="attend", dtype="bf16", cache="bf16", heads=28, kv=4, dim=64, page=16, n=9, rows_lo=1, rows_hi=509,
             len_lo=300, len_hi=4099, causal=True, window=1000, mix=8),
        # the second half of a long prompt
        dict(name="attend_prompt", op="attend", dtype="f16", cache="f16", heads=32, kv=8, dim=128, page=128, n=1, rows_lo=4096, rows_hi=4096,
             len_lo=8192, len_hi=8192, causal=True, window=0, mix=9),
        # one session branches once and goes on
        dict(name="fork_one", op="fork", cache="f16", layers=64, kv=8, dim=128, page=16, pages=96, parents=1, children=1, len_lo=900, len_hi=901,
             grow=1, mix=10),
        # beams or samples: eight sessions branch into forty-eight, each goes on by a few tokens
        dict(name="fork_many", op="fork", cache="bf16", layers=32, kv=8, dim=128, page=64, pages=240, parents=8, children=48, len_lo=300, len_hi=1500,
             grow=5, mix=11),
        # half of the sessions have ended: their pages go back and the rest moves together
        dict(name="release_compact", op="compact", cache="f16", layers=32, kv=8, dim=128, page=64, pages=240, parents=24, ended=12, len_lo=200,
             len_hi=900, mix=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "attend", "attend", "attend", "fork", "compact"])
    mix = rng.randrange(1 << 30)
    kv = rng.choice([1, 2, 4, 8])
    if op == "rope":
        cache = rng.choice(["f16", "bf16"])
        dim = rng.choice([64, 128])
        n = _log_int(rng, 1, 32)
        rows = _log_int(rng, 1, max(1, 8192 // n))
        return dict(op=op, dtype=rng.choice(["f32", cache]), cache=cache, heads=kv * rng.choice([1, 4, 5, 8]), kv=kv, dim=dim,
                    page=rng.choice([16, 32, 64, 128]), n=n, rows_lo=max(1, rows // 3), rows_hi=rows, len_lo=rows, len_hi=rows + _log_int(rng, 1, 60000),
                    rot=rng.choice([dim, dim // 2, 40]), layout=rng.choice(["half", "pairs"]), scaling=rng.choice(["none", "linear", "yarn"]),
                    factor=rng.choice([2.0, 4.0, 8.0]), norms=rng.random() < 0.5, mix=mix)
    if op == "attend":
        dim, group = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 5, 7, 8])
        page, cache = rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16"])
        kind = rng.choice(["next", "verify", "chunk", "prompt"])
        if kind in ("next", "verify"):
            n = _log_int(rng, 1, 64)
            rows = 1 if kind == "next" else rng.randint(2, 8)
            hi = max(rows, _log_int(rng, 64, 131072 // n))
            f32 = rng.random() < 0.3
            return dict(op=op, dtype="f32" if f32 else cache, cache="f16" if f32 else cache, heads=kv * group, kv=kv, dim=dim, page=page, n=n,
                        rows_lo=rows, rows_hi=rows, len_lo=max(rows, hi // rng.choice([1, 3, 20])), len_hi=hi, causal=True,
                        window=rng.choice([0, 0, 0, 777]), mix=mix)
        n = _log_int(rng, 2, 8) if kind == "chunk" else 1
        rows = _log_int(rng, 9, 512 if kind == "chunk" else 3500)
        hi = _log_int(rng, rows, max(rows, 8192 // n))
        return dict(op=op, dtype=cache, cache=cache, heads=kv * min(group, 4 if kind == "prompt" else 8), kv=kv, dim=dim, page=page, n=n,
                    rows_lo=1 if kind == "chunk" else rows, rows_hi=rows, len_lo=max(rows, hi // 3), len_hi=hi,
                    causal=rng.random() < 0.85, window=rng.choice([0, 0, 0, 640]), mix=mix)
    layers, page = rng.choice([2, 24, 32]), rng.choice([16, 32, 64])
    base = dict(op=op, cache=rng.choice(["f16", "bf16"]), layers=layers, kv=kv, dim=rng.choice([64, 128]), page=page, pages=240, mix=mix)
    if op == "fork":
        parents = _log_int(rng, 1, 8)
        return dict(base, parents=parents, children=_log_int(rng, 1, 40), len_lo=1, len_hi=max(2, 150 * page // parents), grow=rng.randint(1, page))
    parents = rng.randint(2, 24)
    return dict(base, parents=parents, ended=rng.randint(1, parents - 1), len_lo=1, len_hi=max(2, 200 * page // parents))


# ---------------------------------------------------------------------------------------- sizes of a case

def _lengths(case):
    """Rows and length of every sequence: part of the case, not of the seed."""
    rng = random.Random(case["mix"])
    rows = [_log_int(rng, case["rows_lo"], case["rows_hi"]) for _ in range(case["n"])]
    return rows, [max(r, _log_int(rng, case["len_lo"], case["len_hi"])) for r in rows]


def _pool_lengths(case):
    rng = random.Random(case["mix"])
    return [_log_int(rng, case["len_lo"], case["len_hi"]) for _ in range(case["parents"])]


def _pages_of(length, page):
    return -(-length // page)


def _visible(rows, length, case):
    """Positions that at least one row sees, and (row, position) pairs."""
    pos = torch.arange(length - rows, length, dtype=torch.int64)
    hi = pos + 1 if case["causal"] else torch.full_like(pos, length)
    lo = (pos - case["window"] + 1).clamp(min=0) if case["window"] else torch.zeros_like(pos)
    return int(hi[-1] - lo[0]), int((hi - lo).clamp(min=0).sum())


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "rope":
        rows, lens = _lengths(case)
        t, d, c = sum(rows), case["dim"], size[case["cache"]]
        q = 2 * t * case["heads"] * d * size[case["dtype"]]
        kv = 2 * t * case["kv"] * d * (size[case["dtype"]] + c)
        return {"bytes": q + kv, "flops": 3.0 * t * (case["heads"] + case["kv"]) * case["rot"]}
    if case["op"] == "attend":
        rows, lens = _lengths(case)
        seen = [_visible(r, l, case) for r, l in zip(rows, lens)]
        q = 2 * sum(rows) * case["heads"] * case["dim"] * size[case["dtype"]]
        kv = 2 * sum(s[0] for s in seen) * case["kv"] * case["dim"] * size[case["cache"]]
        return {"bytes": q + kv, "flops": 4.0 * case["dim"] * case["heads"] * sum(s[1] for s in seen)}
    lens, page = _pool_lengths(case), case["page"]
    token = 2 * case["layers"] * case["kv"] * case["dim"] * 2  # K and V of one token in every layer
    if case["op"] == "fork":
        kids = [lens[i % len(lens)] for i in range(case["children"])]
        # every child takes over a part-filled last page; its parent keeps the original
        return {"bytes": 2 * token * sum(l % page for l in kids) + 4 * case["pages"] + 4 * sum(_pages_of(l, page) for l in kids), "flops": 0}
    moved = _moves(case)
    return {"bytes": 2 * token * page * moved + 4 * case["pages"] + 4 * sum(_pages_of(l, page) for l in lens), "flops": 0}


def _assign(case):
    """Which pages the sequences of a pool case hold: a random part of the pool, in random order."""
    ids = list(range(case["pages"]))
    random.Random(case["mix"] + 1).shuffle(ids)
    return ids[:sum(_pages_of(l, case["page"]) for l in _pool_lengths(case))]


def _moves(case):
    lens = _pool_lengths(case)
    gone = sum(_pages_of(l, case["page"]) for l in lens[:case["ended"]])
    kept = _assign(case)[gone:]
    return sum(p >= len(kept) for p in kept)


# ------------------------------------------------------------------------------------------------ inputs

def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if case["op"] in ("rope", "attend"):
        rows, lens = _lengths(case)
        n, page, dt, ct = case["n"], case["page"], TYPES[case["dtype"]], TYPES[case["cache"]]
        total, width, slots = sum(_pages_of(l, page) for l in lens), max(_pages_of(l, page) for l in lens) + 2, n + 3
        pages = total + 5
        # a pool in use: every slot of every page holds something, the rest of the last pages included
        shape = (1, pages, page, case["kv"], case["dim"])
        s["k"], s["v"] = _normal(gen, shape, ct), _normal(gen, shape, ct)
        order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
        table = torch.zeros((slots, width), dtype=torch.int32, device=DEV)
        slot = torch.randperm(slots, generator=gen, device=DEV)[:n].to(torch.int32)
        all_lens = torch.zeros(slots, dtype=torch.int32, device=DEV)
        at = 0
        for i, sl in enumerate(slot.tolist()):
            need = _pages_of(lens[i], page)
            table[sl, :need] = order[at:at + need]
            all_lens[sl] = lens[i]
            at += need
        refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        refs[order[:at].long()] = 1
        cu = [0]
        for r in rows:
            cu.append(cu[-1] + r)
        s |= dict(table=table, lens=all_lens, refs=refs, seqs=slot, cu=_int(cu), max_rows=max(rows), max_pages=width - 2)
        h, d, t = case["heads"], case["dim"], cu[-1]
        if case["op"] == "attend":
            s["q"] = _normal(gen, (t, h, d), dt, 1.5)
            s["out"] = torch.empty_like(s["q"])
            s["scale"] = 1.0 / math.sqrt(d)
        else:
            # the fused projection's rows: Q | K | V beside one another
            qkv = _normal(gen, (t, (h + 2 * case["kv"]) * d), dt, 1.5).view(t, h + 2 * case["kv"], d)
            s["q"], s["kn"], s["vn"] = qkv[:, :h], qkv[:, h:h + case["kv"]], qkv[:, h + case["kv"]:]
            s["out"] = torch.empty((t, h, d), dtype=dt, device=DEV)
            s["q_norm"] = 1 + 0.1 * _normal(gen, (d,), torch.float32) if case["norms"] else None
            s["k_norm"] = 1 + 0.1 * _normal(gen, (d,), torch.float32) if case["norms"] else None
    else:
        lens, page, ct = _pool_lengths(case), case["page"], TYPES[case["cache"]]
        shape = (case["layers"], case["pages"], page, case["kv"], case["dim"])
        s["k"], s["v"] = _normal(gen, shape, ct), _normal(gen, shape, ct)
        kids = case.get("children", 0)
        slots, width = len(lens) + kids + 2, max(_pages_of(l, page) for l in lens) + 2
        held = _assign(case)
        table = torch.zeros((slots, width), dtype=torch.int32)
        at = 0
        for i, l in enumerate(lens):
            need = _pages_of(l, page)
            table[i, :need] = torch.tensor(held[at:at + need], dtype=torch.int32)
            at += need
        refs = torch.zeros(case["pages"], dtype=torch.int32)
        refs[torch.tensor(held)] = 1
        s |= dict(table=table.to(DEV), lens=_int(lens + [0] * (slots - len(lens))), refs=refs.to(DEV))
        if case["op"] == "fork":
            s |= dict(src=[i % len(lens) for i in range(kids)], dst=[len(lens) + i for i in range(kids)], grow=[case["grow"]] * kids)
        else:
            # what the scheduler's step began with; each pass starts from it
            s |= dict(table0=s["table"].clone(), lens0=s["lens"].clone(), refs0=s["refs"].clone(), ended=list(range(case["ended"])))
            s["map"] = torch.empty(case["pages"], dtype=torch.int32, device=DEV)
    if own:  # the handle that a user of the framework keeps for a pool
        gpu, g = _gpu()
        s["pages"] = gpu.KvPages(g, s["k"], s["v"], s["table"], s["lens"], s["refs"])
        if case["op"] == "rope":
            s["rope"] = gpu.Rope(case["rot"], layout=case["layout"], base=BASE, scaling=case["scaling"], factor=case["factor"], orig_ctx=ORIG)
    return s


BASE, ORIG, EPS = 1e6, 8192, 1e-6
BETA_FAST, BETA_SLOW = 32.0, 1.0


# ---------------------------------------------------------------------------------------- the plain forms

def _frequencies(case):
    """Radians a position, in 64 bits, and the factor on sine and cosine."""
    rot = case["rot"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    f = BASE ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        return f / case["factor"], 1.0
    if case["scaling"] == "yarn":
        edge = [rot * math.log(ORIG / (b * 2 * math.pi)) / (2 * math.log(BASE)) for b in (BETA_FAST, BETA_SLOW)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f / case["factor"] * ramp + f * (1 - ramp), 0.1 * math.log(case["factor"]) + 1.0
    return f, 1.0


def _token_rows(s):
    """Slot and position of every row of the batch."""
    t = torch.arange(s["q"].shape[0], device=DEV)
    i = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    slot = s["seqs"].long()[i]
    rows = (s["cu"][1:] - s["cu"][:-1]).long()[i]
    return slot, s["lens"].long()[slot] - rows + t - s["cu"].long()[i]


def _rotate(x, cos, sin, case):
    rot, half = case["rot"], case["rot"] // 2
    if case["layout"] == "half":
        a, b = x[..., :half], x[..., half:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., rot:]], -1)


def _head_norm(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_rope(s):
    case = s["case"]
    slot, pos = _token_rows(s)
    f, m = _frequencies(case)
    angle = (pos.double()[:, None] * f)[:, None]
    cos, sin = (angle.cos() * m).float(), (angle.sin() * m).float()
    s["out"].copy_(_rotate(_head_norm(s["q"].float(), s["q_norm"]), cos, sin, case))
    kr = _rotate(_head_norm(s["kn"].float(), s["k_norm"]), cos, sin, case)
    page = s["table"][slot, pos // case["page"]].long()
    s["k"][0, page, pos % case["page"]] = kr.to(s["k"].dtype)
    s["v"][0, page, pos % case["page"]] = s["vn"].to(s["v"].dtype)


def _plain_attend(s):
    case = s["case"]
    n, g, d = case["n"], case["heads"] // case["kv"], case["dim"]
    lens = s["lens"].long()[s["seqs"].long()]
    pages = s["table"][s["seqs"].long(), :s["max_pages"]].long()
    k = s["k"][0][pages].flatten(1, 2).float().permute(0, 2, 1, 3)  # [n, kv, positions, dim]
    v = s["v"][0][pages].flatten(1, 2).float().permute(0, 2, 1, 3)
    row = s["cu"][:-1].long()[:, None] + torch.arange(s["max_rows"], device=DEV)  # [n, rows]
    real = row < s["cu"][1:].long()[:, None]
    q = s["q"][row.clamp(max=s["q"].shape[0] - 1)].float().view(n, -1, case["kv"], g, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    pos = lens[:, None] - (s["cu"][1:] - s["cu"][:-1]).long()[:, None] + torch.arange(s["max_rows"], device=DEV)
    j = torch.arange(k.shape[2], device=DEV)
    see = (j < lens[:, None])[:, None, :].expand(-1, pos.shape[1], -1)
    if case["causal"]:
        see = see & (j <= pos[:, :, None])
    if case["window"]:
        see = see & (j > pos[:, :, None] - case["window"])
    score = score.view(n, case["kv"], g, -1, j.numel()).masked_fill(~see[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    del score
    total = p.sum(-1, keepdim=True)
    v = torch.where((j < lens[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(p.flatten(2, 3), v).view(n, case["kv"], g, -1, d) / total.clamp(min=1e-38)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).flatten(2, 3)[real])


def _release(s, seqs, keep):
    """Cuts the sequences down to `keep` tokens and gives the pages behind them back."""
    at = torch.tensor(seqs, device=DEV)
    page, col = s["case"]["page"], torch.arange(s["table"].shape[1], device=DEV)
    old = s["lens"][at]
    new = torch.minimum(old, _int(keep))
    gone = (col >= (new[:, None] + page - 1) // page) & (col < (old[:, None] + page - 1) // page)
    s["refs"].index_add_(0, s["table"][at][gone].long(), -torch.ones_like(s["table"][at][gone]))
    s["lens"][at] = new


def _plain_fork(s):
    case, page = s["case"], s["case"]["page"]
    src, dst, grow = torch.tensor(s["src"], device=DEV), torch.tensor(s["dst"], device=DEV), _int(s["grow"])
    col = torch.arange(s["table"].shape[1], device=DEV)
    # the children take their parents' pages, in place of what they held
    _release(s, s["dst"], [0] * len(s["dst"]))
    held = col < (s["lens"][src][:, None] + page - 1) // page
    s["table"][dst] = torch.where(held, s["table"][src], s["table"][dst])
    s["lens"][dst] = s["lens"][src]
    s["refs"].index_add_(0, s["table"][src][held].long(), torch.ones_like(s["table"][src][held]))
    # room for the new tokens, lowest free page first; who writes into a shared page gets a copy of it, the last holder keeps it
    old = s["lens"][dst]
    have, want = (old + page - 1) // page, (old + grow + page - 1) // page
    last = s["table"][dst, (have - 1).clamp(min=0).long()].long()
    writes = (old % page > 0) & (grow > 0)
    before = ((last[:, None] == last) & writes[:, None] & writes).tril(-1).sum(1)
    copy = writes & (s["refs"][last] - before > 1)
    need = copy.int() + want - have
    free = (s["refs"] == 0).nonzero().flatten()
    first = need.cumsum(0) - need
    short = (need.sum() - free.numel()).clamp(min=0)
    fresh = free[first[copy]]
    kept = (torch.arange(page, device=DEV) < (old % page)[copy][:, None])[None, :, :, None, None]
    for c in (s["k"], s["v"]):
        c[:, fresh] = torch.where(kept, c[:, last[copy]], c[:, fresh])
    s["refs"].index_add_(0, last[copy], -torch.ones_like(last[copy], dtype=torch.int32))
    s["table"][dst[copy], (have - 1)[copy].long()] = fresh.int()
    new = (col >= have[:, None]) & (col < want[:, None])
    pick = ((first + copy)[:, None] + col - have[:, None])[new]
    rows = s["table"][dst]
    rows[new] = free[pick].int()
    s["table"][dst] = rows
    s["refs"][fresh] = 1
    s["refs"][free[pick]] = 1
    s["lens"][dst] = old + grow
    return short.int()


def _plain_compact(s):
    page = s["case"]["page"]
    for name in ("table", "lens", "refs"):
        s[name].copy_(s[name + "0"])
    _release(s, s["ended"], [0] * len(s["ended"]))
    live = s["refs"] > 0
    at, count = torch.arange(live.numel(), device=DEV), live.sum()
    movers, holes = (live & (at >= count)).nonzero().flatten(), (~live & (at < count)).nonzero().flatten()
    s["map"].copy_(torch.where(live, at, -1))
    s["map"][movers] = holes.int()
    for c in (s["k"], s["v"]):
        c[:, holes] = c[:, movers]
    s["refs"][holes] = s["refs"][movers]
    s["refs"][movers] = 0
    held = torch.arange(s["table"].shape[1], device=DEV) < (s["lens"][:, None] + page - 1) // page
    s["table"].copy_(torch.where(held, s["map"][s["table"].long()], s["table"]))


# --------------------------------------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if own:
        gpu, g = _gpu()
        stream = torch.cuda.current_stream().cuda_stream
        if op == "rope":
            g.rope_append(s["pages"], 0, s["q"], s["kn"], s["vn"], s["cu"], s["rope"], out=s["out"], seqs=s["seqs"], q_norm=s["q_norm"],
                          k_norm=s["k_norm"], eps=EPS, stream=stream)
        elif op == "attend":
            g.attend_pages(s["pages"], 0, s["q"], s["cu"], s["scale"], out=s["out"], seqs=s["seqs"], causal=s["case"]["causal"],
                           window=s["case"]["window"], stream=stream)
        elif op == "fork":
            g.pages_fork(s["pages"], s["src"], s["dst"], stream=stream)
            g.pages_reserve(s["pages"], s["dst"], s["grow"], stream=stream, wait=False)
        else:
            for name in ("table", "lens", "refs"):
                s[name].copy_(s[name + "0"])
            g.pages_release(s["pages"], s["ended"], [0] * len(s["ended"]), stream=stream)
            g.pages_compact(s["pages"], page_map=s["map"], stream=stream)
    elif op == "rope":
        _plain_rope(s)
    elif op == "attend":
        _plain_attend(s)
    elif op == "fork":
        short = _plain_fork(s)
    else:
        _plain_compact(s)
    if op == "attend":
        return s["out"]
    if op == "rope":
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    got = {name: s[name] for name in ("k", "v", "table", "lens", "refs")}
    if op == "fork":
        return dict(got, short=s["pages"].short_by if own else short)
    return dict(got, map=s["map"])


# ---------------------------------------------------------------------------------- definition in 64 bits

def exact(case, seed):
    if case["op"] not in ("rope", "attend"):
        return None  # copies and whole numbers
    s = prepare(case, seed)
    cu, slots = s["cu"].tolist(), s["seqs"].tolist()
    lens, table, page = s["lens"].tolist(), s["table"].tolist(), case["page"]
    if case["op"] == "rope":
        k, v, q = s["k"].double(), s["v"].double(), torch.empty_like(s["out"], dtype=torch.float64)
        for b, sl in enumerate(slots):
            rows = range(cu[b], cu[b + 1])
            pos = torch.arange(lens[sl] - len(rows), lens[sl], device=DEV)
            where = torch.tensor(table[sl], device=DEV)[pos // page] * page + pos % page
            part = slice(cu[b], cu[b + 1])
            q[part] = _turn64(s["q"][part].double(), s["q_norm"], pos, case)
            k[0].flatten(0, 1)[where] = _turn64(s["kn"][part].double(), s["k_norm"], pos, case)
            v[0].flatten(0, 1)[where] = s["vn"][part].double()
        return {"q": q, "k": k, "v": v}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    group = case["heads"] // case["kv"]
    for b, sl in enumerate(slots):
        length, rows = lens[sl], cu[b + 1] - cu[b]
        ids = torch.tensor(table[sl][:_pages_of(length, page)], device=DEV)
        k = s["k"][0].index_select(0, ids).flatten(0, 1)[:length].double()
        v = s["v"][0].index_select(0, ids).flatten(0, 1)[:length].double()
        far = torch.arange(length - rows, length, device=DEV)[:, None] - torch.arange(length, device=DEV)  # how far back a position lies
        hidden = torch.zeros_like(far, dtype=torch.bool)
        if case["causal"]:
            hidden |= far < 0
        if case["window"]:
            hidden |= far >= case["window"]
        for head in range(case["heads"]):
            z = s["q"][cu[b]:cu[b + 1], head].double() @ k[:, head // group].T
            z.mul_(s["scale"])[hidden] = -math.inf
            out[cu[b]:cu[b + 1], head] = torch.softmax(z, 1) @ v[:, head // group]
    return out


def _turn64(x, w, pos, case):
    """Every pair of a head as a complex number, turned by its own angle."""
    if w is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    rot = case["rot"]
    turn = []
    for i in range(rot // 2):
        f, m = BASE ** (-2.0 * i / rot), 1.0
        if case["scaling"] == "linear":
            f /= case["factor"]
        elif case["scaling"] == "yarn":
            # the pair that makes `b` turns over the original context lies at this index
            at = lambda b: rot / 2 * math.log(ORIG / (2 * math.pi * b), BASE)  # noqa: E731
            lo, hi = max(0, math.floor(at(BETA_FAST))), min(rot - 1, math.ceil(at(BETA_SLOW)))
            share = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            f = f * (1 - share + share / case["factor"])
            m = 1 + math.log(case["factor"]) / 10
        turn.append(torch.polar(torch.full_like(pos, 1, dtype=torch.float64) * m, pos.double() * f))
    turn = torch.stack(turn, -1)[:, None]
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if case["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y
