"""A paged KV pool for tests, and its operators in 64 bits."""
import math

import numpy as np
import torch

TY = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#: half a step of each type, relative
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Pool:
    """Tensors of a pool whose slots all hold NaN until something is put there; ``order`` = memory order of the axes
    (layer, page, position, head) and a pad between the pages."""

    def __init__(self, layers, pages, page, kv, dim, cache, slots, width, order=(0, 1, 2, 3), pad=0, seed=0, device="cuda"):
        self.page, self.kv, self.dim, self.cache = page, kv, dim, cache
        rng = np.random.default_rng(seed)

        def storage():
            size = [layers, pages, page, kv]
            shape = [size[a] for a in order]
            shape[-1] += pad
            t = torch.full((*shape, dim), math.nan, dtype=TY[cache], device=device)
            t = t[..., : size[order[-1]], :]
            return t.permute(*[order.index(a) for a in range(4)], 4)

        self.k, self.v = storage(), storage()
        self.table = torch.full((slots, width + 3), -7, dtype=torch.int32, device=device)[:, :width]
        self.lens = torch.zeros(slots, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.free = list(rng.permutation(pages))

    def args(self):
        return self.k, self.v, self.table, self.lens, self.refs

    def fill(self, slot, length, gen, layer=0):
        """A sequence of ``length`` random positions in random pages; returns its K and V."""
        n = -(-length // self.page)
        pages = [int(self.free.pop()) for _ in range(n)]
        self.table[slot, :n] = torch.tensor(pages, dtype=torch.int32)
        self.lens[slot] = length
        k = torch.randn((length, self.kv, self.dim), generator=gen, device=self.k.device).to(TY[self.cache])
        v = torch.randn((length, self.kv, self.dim), generator=gen, device=self.k.device).to(TY[self.cache])
        for i, p in enumerate(pages):
            part = slice(i * self.page, min(length, (i + 1) * self.page))
            self.k[layer, p, : part.stop - part.start] = k[part]
            self.v[layer, p, : part.stop - part.start] = v[part]
            self.refs[p] = 1
        return k, v

    def read(self, slot, layer=0):
        """K and V of a sequence, position by position, through the table."""
        length = int(self.lens[slot])
        pages = self.table[slot, : -(-length // self.page)].long()
        return tuple(t[layer].index_select(0, pages).reshape(-1, self.kv, self.dim)[:length] for t in (self.k, self.v))


def attend64(q, k, v, scale, causal=True, window=0):
    """(o, a, s): attention of the last rows of one sequence in 64 bits, the same sum over |v|, and the largest sum of
    |q_d k_d| scale log2(e) of a visible position.  Hidden positions are left out of the sums, whatever they hold.  A row that
    sees nothing is 0."""
    rows, heads, dim = q.shape
    length = k.shape[0]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    a, most = torch.zeros_like(o), torch.zeros((rows, heads, 1), dtype=torch.float64, device=q.device)
    if length == 0 or rows == 0:
        return o, a, most
    group = heads // k.shape[1]
    pos = torch.arange(length - rows, length, device=q.device)
    j = torch.arange(length, device=q.device)
    see = torch.ones((rows, length), dtype=torch.bool, device=q.device)
    if causal:
        see &= j <= pos[:, None]
    if window:
        see &= j > pos[:, None] - window
    for h in range(heads):
        kk, vv = k[:, h // group].double(), v[:, h // group].double()
        s = (q[:, h].double() @ kk.T) * scale
        s[~see] = -math.inf
        size = q[:, h].double().abs() @ kk.abs().T * abs(scale) * math.log2(math.e)
        most[:, h, 0] = torch.where(see & torch.isfinite(size), size, 0.0).amax(1)
        m = s.amax(1, keepdim=True)
        p = torch.where(see, torch.exp(s - torch.where(torch.isfinite(m), m, 0.0)), 0.0)
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
        clean = torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)
        o[:, h], a[:, h] = p @ clean, p @ clean.abs()
        for bad in (~torch.isfinite(vv)).any(1).nonzero().flatten().tolist():
            o[:, h] += torch.where(see[:, bad, None] & ~torch.isfinite(vv[bad]), p[:, bad, None] * vv[bad], 0.0)
    return o, a, most


def attend_bound(o, a, scores, ty):
    """How far a row of the kernels may be from ``o``: the result's own rounding and the softmax weights', half a step each
    (weights of 32-bit rows are not rounded), and what 32-bit scores can be off: every term of a score s = sum q_d k_d passes
    through at most 24 roundings of 2^-24 and 2^s turns that into a relative error of the weight; ``scores`` is the largest sum
    of |q_d k_d| scale log2(e); twice, for the weight and for the sum of weights.  2^-20 for the rest (the exponential itself, the sums of weights)."""
    w = 0.0 if ty == "f32" else HALF[ty]
    return HALF[ty] * o.abs() + (w + 2 * scores * 24 * 2.0 ** -24 + 2.0 ** -20) * a + 1e-7


def freqs64(dim, base, scaling="none", factor=1.0, orig=0, fast=32.0, slow=1.0, attn=1.0, ff=None):
    i = np.arange(dim // 2, dtype=np.float64)
    f = base ** (-2 * i / dim)
    if ff is not None:
        f = f / np.asarray(ff, np.float64)
    mag = attn
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        c = [dim * math.log(orig / (2 * math.pi * b)) / (2 * math.log(base)) for b in (fast, slow)]
        lo, hi = max(0, math.floor(c[0])), min(dim - 1, math.ceil(c[1]))
        r = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        f = f / factor * r + f * (1 - r)
        if factor > 1:
            mag *= 0.1 * math.log(factor) + 1
    return f, mag


def rotate64(x, pos, f, mag, layout, w=None, eps=1e-6):
    """x [rows, heads, dim] turned by pos [rows]."""
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = len(f)
    ang = pos.double()[:, None] * torch.from_numpy(f).to(x.device)
    c, s = (ang.cos() * mag)[:, None], (ang.sin() * mag)[:, None]
    y = x.clone()
    ia, ib = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


class Book:
    """The pool's bookkeeping on the host, step by step as the header words it."""

    def __init__(self, pages, page, slots, width):
        self.page, self.width, self.refs = page, width, [0] * pages
        self.seqs = [([], 0) for _ in range(slots)]  # (pages, length)

    def _need(self, n):
        return -(-n // self.page)

    def reserve(self, seqs, n_new):
        """(short, copies): copies = (from, to, positions)."""
        refs, out, copies = list(self.refs), {}, []
        free = [p for p, r in enumerate(refs) if r == 0]
        want = 0
        for s, n in zip(seqs, n_new):
            pages, length = list(self.seqs[s][0]), self.seqs[s][1]
            if self._need(length + n) > self.width:
                return -1, []
            if n and length % self.page and refs[pages[-1]] > 1:
                want += 1
                if free:
                    new = free.pop(0)
                    refs[pages[-1]] -= 1
                    refs[new] = 1
                    copies.append((pages[-1], new, length % self.page))
                    pages[-1] = new
                else:
                    refs[pages[-1]] -= 1
            for _ in range(self._need(length + n) - self._need(length)):
                want += 1
                if free:
                    new = free.pop(0)
                    refs[new] = 1
                    pages.append(new)
            out[s] = (pages, length + n)
        short = want - sum(r == 0 for r in self.refs)
        if short > 0:
            return short, []
        self.refs = refs
        for s, x in out.items():
            self.seqs[s] = x
        return 0, copies

    def release(self, seqs, keep):
        for s, n in zip(seqs, keep):
            pages, length = self.seqs[s]
            n = min(n, length)
            for p in pages[self._need(n):]:
                self.refs[p] -= 1
            self.seqs[s] = (pages[: self._need(n)], n)

    def fork(self, src, dst):
        self.release(dst, [0] * len(dst))
        for a, b in zip(src, dst):
            self.seqs[b] = (list(self.seqs[a][0]), self.seqs[a][1])
            for p in self.seqs[b][0]:
                self.refs[p] += 1

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        to = {p: p for p in live}
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        movers = [p for p in live if p >= len(live)]
        to.update(zip(movers, holes))
        refs = [0] * len(self.refs)
        for p in live:
            refs[to[p]] = self.refs[p]
        self.refs = refs
        self.seqs = [([to[p] for p in pages], n) for pages, n in self.seqs]
        return [to.get(p, -1) for p in range(len(self.refs))], list(zip(movers, holes))
