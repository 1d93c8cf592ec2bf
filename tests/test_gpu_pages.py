"""The paged KV cache on a GPU: each operator against 64 bits or against the bookkeeping step by step, then a run of them together."""
import math
import random

import numpy as np
import pytest
import torch

from tests.pages_util import HALF, TY, Book, Pool, attend64, attend_bound, freqs64, rotate64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def G():
    from allpaka_b200 import gpu

    return gpu


@pytest.fixture(scope="module")
def g(G):
    ctx = G.Gpu(0)
    yield ctx
    ctx.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ attention

def attend_case(G, g, rows, lens, *, cache="f16", rows_ty=None, kv=2, group=4, dim=128, page=16, order=(0, 1, 2, 3), pad=0, causal=True,
                window=0, seed=1, spoil=None, seqs=None, scale=None, strided=False):
    """Runs one batch and holds every row against 64 bits; returns the output."""
    ty = rows_ty or cache
    n, total = len(rows), sum(rows)
    need = sum(-(-l // page) for l in lens)
    pool = Pool(2, need + 3, page, kv, dim, cache, n + 2, max(-(-l // page) for l in lens) + 1, order, pad, seed)
    r = gen(seed)
    slots = list(range(n, 0, -1)) if seqs is None else seqs
    held = [pool.fill(s, l, r, layer=1) for s, l in zip(slots, lens)]
    if spoil is not None:
        spoil(pool, slots)
        held = [pool.read(s, 1) for s in slots]
    heads = kv * group
    cu = [3]  # three rows in front and two behind belong to nobody
    for x in rows:
        cu.append(cu[-1] + x)
    wide = (heads + 1) * dim if strided else heads * dim
    q = (torch.randn((total + 5, wide), generator=r, device="cuda") * 1.5).to(TY[ty])[:, : heads * dim].view(total + 5, heads, dim)
    out = torch.full((total + 5, wide), 7.0, device="cuda", dtype=TY[ty])[:, : heads * dim].view(total + 5, heads, dim)
    scale = 1 / math.sqrt(dim) if scale is None else scale
    pages = G.KvPages(g, *pool.args())
    assert g.attend_pages(pages, 1, q, ints(cu), scale, out, seqs=ints(slots), causal=causal, window=window, wait=True), g.last_decline
    assert bool((out[:3] == 7).all()) and bool((out[total + 3:] == 7).all())
    if strided:
        assert bool((out.as_strided((total + 5, wide), (wide, 1))[:, heads * dim:] == 7).all())
    for i in range(n):
        part = slice(cu[i], cu[i + 1])
        k, v = held[i]
        o, a, most = attend64(q[part], k, v, scale, causal, window)
        got = out[part].double()
        fine = torch.isfinite(o)
        assert torch.equal(torch.isnan(got), torch.isnan(o))
        assert torch.equal(got[~fine & ~torch.isnan(o)], o[~fine & ~torch.isnan(o)])
        off = ((got - o).abs() - attend_bound(o, a, most, ty))[fine]
        assert off.numel() == 0 or float(off.max()) <= 0, (i, rows[i], lens[i], float(off.max()))
    return out


KINDS = [("f16", None), ("bf16", None), ("f16", "f32")]


@pytest.mark.parametrize("cache,rows_ty", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_lengths_from_nothing_to_many_tiles(G, g, cache, rows_ty, dim):
    rows = [1, 1, 0, 3, 2, 1, 17, 1, 64, 5]
    lens = [1, 0, 40, 3, 2, 127, 128, 129, 300, 1025]
    attend_case(G, g, rows, lens, cache=cache, rows_ty=rows_ty, dim=dim)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_attention_page_sizes(G, g, cache, page):
    attend_case(G, g, [1, 40, 260], [513, 300, 700], cache=cache, page=page, kv=2, group=2)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 12, 16, 48, 64])
@pytest.mark.parametrize("rows_ty", [None, "f32"])
def test_attention_groups(G, g, group, rows_ty):
    attend_case(G, g, [1, 9, 150 if rows_ty is None else 8], [333, 140, 260], kv=1 if group > 12 else 3, group=group, rows_ty=rows_ty)


@pytest.mark.parametrize("order,pad", [((0, 1, 3, 2), 0), ((1, 0, 2, 3), 1), ((3, 2, 1, 0), 2), ((2, 3, 0, 1), 0)])
@pytest.mark.parametrize("cache,rows_ty", KINDS)
def test_attention_layouts_of_the_pool(G, g, cache, rows_ty, order, pad):
    attend_case(G, g, [1, 130, 4], [200, 131, 70], cache=cache, rows_ty=rows_ty, order=order, pad=pad, strided=True)


@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 50), (True, 128), (True, 1000), (False, 50)])
@pytest.mark.parametrize("cache,rows_ty", KINDS)
def test_attention_masks(G, g, cache, rows_ty, causal, window):
    attend_case(G, g, [1, 7, 200, 1], [900, 300, 450, 20], cache=cache, rows_ty=rows_ty, causal=causal, window=window)


@pytest.mark.parametrize("cache,rows_ty", KINDS)
def test_attention_rows_that_see_nothing_are_zero(G, g, cache, rows_ty):
    """More rows than positions: the first rows stand before position 0."""
    out = attend_case(G, g, [9, 140, 3], [4, 100, 0], cache=cache, rows_ty=rows_ty)
    assert bool((out[3:8] == 0).all()) and bool((out[12:52] == 0).all()) and bool((out[152:155] == 0).all())
    attend_case(G, g, [9, 140, 3], [4, 100, 0], cache=cache, rows_ty=rows_ty, causal=False, window=60)


@pytest.mark.parametrize("cache,rows_ty", KINDS)
def test_attention_hidden_values_do_not_matter(G, g, cache, rows_ty):
    """A later position's infinities and NaN reach its own rows and those behind it only."""
    def spoil(pool, slots):
        for s, j, x in ((slots[0], 150, math.nan), (slots[1], 299, math.inf), (slots[2], 0, -math.inf)):
            p = int(pool.table[s, j // pool.page])
            pool.v[1, p, j % pool.page, :, 5] = x
            if j:
                pool.k[1, p, j % pool.page, 0, 3] = math.nan if x != x else 1.0

    out = attend_case(G, g, [120, 9, 5], [200, 300, 400], cache=cache, rows_ty=rows_ty, spoil=spoil, window=300)
    assert bool(torch.isfinite(out[3:73]).all()) and not bool(torch.isfinite(out[73:123, :, 5]).any())
    assert bool(torch.isfinite(out[132:137]).all())  # outside the window


def test_attention_bad_pages_and_sequences(G, g):
    """Page numbers outside the pool are pages that are not there; sequence numbers outside the table have no positions."""
    for ty in (None, "f32"):
        pool = Pool(1, 40, 16, 2, 128, "f16", 4, 12, seed=3)
        r = gen(3)
        k, v = pool.fill(1, 150, r)
        pool.fill(2, 60, r)
        pool.table[1, 2], pool.table[1, 5], pool.table[2, 0] = -1, 40, 2 ** 31 - 1
        pool.lens[0] = -5
        q = torch.randn((160, 8, 128), generator=r, device="cuda").to(TY[ty or "f16"])
        out = torch.full_like(q, 7.0)
        cu, seqs = ints([0, 1, 141, 144, 145, 146]), ints([1, 1, 2, 9, -3])
        assert g.attend_pages(G.KvPages(g, *pool.args()), 0, q, cu, 0.1, out, seqs=seqs, wait=True)
        there = torch.ones(150, dtype=torch.bool)
        there[32:48] = there[80:96] = False
        for part, rows in ((slice(0, 1), 1), (slice(1, 141), 140)):
            for t in range(rows):
                pos = 150 - rows + t
                sel = (there & (torch.arange(150) <= pos)).nonzero().flatten().cuda()
                ref = attend64(q[part][t:t + 1], k[sel], v[sel], 0.1, causal=False)
                assert float(((out[part][t:t + 1].double() - ref[0]).abs() - attend_bound(*ref, ty or "f16")).max()) <= 0
        assert bool((out[144:146] == 0).all()) and bool((out[146:] == 7).all())
        # offsets that fall, and that run past the rows: cut, nothing written outside
        out.fill_(7.0)
        assert g.attend_pages(G.KvPages(g, *pool.args()), 0, q, ints([0, 30, 10, 500, -4]), 0.1, out, seqs=ints([1, 1, 1, 1]), wait=True)


def test_attention_scores_far_from_zero(G, g):
    """Large scores of both signs and a scale of either sign: the running maximum moves by thousands."""
    def spoil(pool, slots):
        for s in slots:
            for j in range(0, int(pool.lens[s]), 7):
                p = int(pool.table[s, j // pool.page])
                pool.k[1, p, j % pool.page] *= 30.0

    for scale in (0.3, -0.3, 0.0):
        for ty in (None, "f32"):
            attend_case(G, g, [1, 60], [700, 400], rows_ty=ty, spoil=spoil, scale=scale)


@pytest.mark.parametrize("cache,rows_ty", KINDS)
def test_attention_many_sequences(G, g, cache, rows_ty):
    """More sequences than a block keeps a copy of, single tokens and small chunks, empty ones among them."""
    rnd = random.Random(12)
    rows = [rnd.choice([0, 1, 1, 1, 2, 5]) for _ in range(700)]
    lens = [max(r, rnd.choice([0, 1, 17, 130, 400])) for r in rows]
    attend_case(G, g, rows, lens, cache=cache, rows_ty=rows_ty, kv=1, group=4, dim=64, page=32)


@pytest.mark.parametrize("dim,group,cache", [(128, 4, "f16"), (64, 8, "bf16"), (128, 5, "bf16")])
def test_attention_long_chunks_and_long_sequences(G, g, dim, group, cache):
    """Tiles that are cut over many blocks of the grid: a chunk of a thousand rows, and one row over twenty thousand positions."""
    attend_case(G, g, [1000, 1, 33], [1500, 20000, 5000], cache=cache, kv=1, group=group, dim=dim, page=128)


def test_attention_long_sequence_of_32_bit_rows(G, g):
    attend_case(G, g, [8, 1], [9000, 12345], rows_ty="f32", kv=2, group=5, page=16)


def test_attention_of_rows_past_32_bit_offsets(G, g):
    """The pages of the sequence lie behind more than 2^31 elements of the pool."""
    n_pages, page, kv, dim = 140000, 16, 8, 128
    pool = Pool(1, 1, page, kv, dim, "f16", 2, 8)
    pool.k = torch.empty((1, n_pages, page, kv, dim), dtype=torch.float16, device="cuda")
    pool.v = torch.empty((1, n_pages, page, kv, dim), dtype=torch.float16, device="cuda")
    assert pool.k.numel() > 2 ** 31
    pool.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    pool.free = list(range(n_pages - 20, n_pages))
    r = gen(40)
    k, v = pool.fill(1, 100, r)
    pages = G.KvPages(g, *pool.args())
    q = torch.randn((3, 16, dim), generator=r, device="cuda").half()
    out = torch.empty_like(q)
    new = [torch.randn((3, h, dim), generator=r, device="cuda").half() for h in (16, kv, kv)]
    assert g.rope_append(pages, 0, *new, ints([0, 3]), None, out=out, seqs=ints([1]), wait=True)
    assert torch.equal(pool.read(1)[0][97:], new[1]) and torch.equal(pool.read(1)[1][97:], new[2])
    k, v = pool.read(1)
    assert g.attend_pages(pages, 0, q, ints([0, 3]), 0.1, out, seqs=ints([1]), wait=True)
    ref = attend64(q, k, v, 0.1)
    assert float(((out.double() - ref[0]).abs() - attend_bound(*ref, "f16")).max()) <= 0
    # a fork far up there, copied to the pool's front
    assert g.pages_fork(pages, [1], [0]) and g.pages_reserve(pages, [0], [1])
    assert int(pool.table[0, 6]) == 0 and torch.equal(pool.k[0, 0, :4], k[96:])


def test_attention_workspaces(G, g):
    """A workspace of the caller's own; too small a one is refused; two calls at once on two streams each have theirs."""
    pool = Pool(1, 700, 16, 2, 128, "f16", 2, 600, seed=50)
    r = gen(50)
    held = [pool.fill(0, 5000, r), pool.fill(1, 3000, r)]
    pages = G.KvPages(g, *pool.args())
    qs = [torch.randn((1, 8, 128), generator=r, device="cuda").half() for _ in range(2)]
    outs, cu = [torch.empty_like(q) for q in qs], ints([0, 1])
    seqs = [ints([0]), ints([1])]
    with pytest.raises(G.GpuError) as e:
        g.attend_pages(pages, 0, qs[0], cu, 0.1, outs[0], workspace=torch.empty(100, dtype=torch.uint8, device="cuda"))
    assert e.value.code == -1
    own = torch.empty(40 << 20, dtype=torch.uint8, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):   # handed a stream that is not the current one
            assert g.attend_pages(pages, 0, qs[i], cu, 0.1, outs[i], seqs=seqs[i], stream=streams[i].cuda_stream, workspace=own if i else None)
    torch.cuda.synchronize()
    for i in range(2):
        ref = attend64(qs[i], *held[i], 0.1)
        assert float(((outs[i].double() - ref[0]).abs() - attend_bound(*ref, "f16")).max()) <= 0


def test_attention_is_repeatable(G, g):
    """The same call gives the same bits: nothing depends on the order in which blocks come."""
    pool = Pool(1, 900, 16, 4, 128, "bf16", 3, 500, seed=51)
    r = gen(51)
    for s, l in enumerate((6000, 17, 2500)):
        pool.fill(s, l, r)
    pages = G.KvPages(g, *pool.args())
    q = torch.randn((302, 16, 128), generator=r, device="cuda").bfloat16()
    got = []
    for _ in range(5):
        out = torch.empty_like(q)
        assert g.attend_pages(pages, 0, q, ints([0, 1, 2, 302]), 0.09, out, wait=True)
        got.append(out)
    assert all(torch.equal(got[0], x) for x in got[1:])


def test_attention_agrees_with_the_contiguous_cache(G, g):
    """The same keys and values in an apk_kv and in pages: 32-bit rows, one and eight of them."""
    kv, dim, length = 4, 128, 777
    pool = Pool(1, 60, 16, kv, dim, "f16", 2, 60, seed=5)
    r = gen(5)
    k, v = pool.fill(1, length, r)
    cache = G.KvCache(g, 1, kv * dim, 800)
    cache.write(0, 0, k.cpu().numpy().view(np.uint16), v.cpu().numpy().view(np.uint16))
    pages = G.KvPages(g, *pool.args())
    for m in (1, 8):
        q = torch.randn((m, 32, dim), generator=r, device="cuda")
        out = torch.empty_like(q)
        assert g.attend_pages(pages, 0, q, ints([0, m]), 0.088, out, seqs=ints([1]), wait=True)
        want = g.attend(cache, 0, q.cpu().numpy(), m, 32, length - m, 0.088)
        err = np.linalg.norm(out.cpu().numpy().reshape(m, -1) - want) / np.linalg.norm(want)
        assert err <= 2e-5, err
    cache.close()


# --------------------------------------------------------------------------------------------------- rope

@pytest.mark.parametrize("ty,cache,out_ty", [("f32", "f16", "f32"), ("f32", "bf16", "bf16"), ("f16", "f16", "f16"), ("bf16", "bf16", "bf16"),
                                            ("bf16", "f16", "f32")])
@pytest.mark.parametrize("dim,rot,layout,scaling", [(128, 128, "half", "none"), (128, 64, "pairs", "yarn"), (64, 40, "half", "linear"),
                                                    (64, 64, "pairs", "none"), (96, 6, "pairs", "linear"), (256, 256, "half", "yarn"),
                                                    (128, 0, "half", "none"), (80, 80, "half", "yarn")])
def test_rope_append(G, g, ty, cache, out_ty, dim, rot, layout, scaling):
    rows, lens, page, kv, heads = [1, 37, 0, 4], [70000, 37, 5, 900], 32, 2, 6
    pool = Pool(2, sum(-(-l // page) for l in lens) + 1, page, kv, dim, cache, 5, 2200, seed=7)
    r = gen(7)
    slots = [3, 1, 0, 4]
    for s, l in zip(slots, lens):
        pool.fill(s, l, r, layer=1)
    before = pool.k.clone(), pool.v.clone()
    T = sum(rows)
    cu = np.cumsum([0] + rows).tolist()
    qkv = torch.randn((T + 2, heads + 2 * kv, dim), generator=r, device="cuda").to(TY[ty])
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    out = torch.full((T + 2, heads, dim), 7.0, device="cuda", dtype=TY[out_ty])
    opts = dict(scaling=scaling, factor=4.0, orig_ctx=4096)
    for norms, ff, positions in ((False, None, None), (True, np.linspace(1, 8, max(rot // 2, 1))[: rot // 2] if rot else None, torch.arange(T + 2, device="cuda").int() * 31)):
        w = [1 + 0.2 * torch.randn(dim, generator=r, device="cuda") for _ in range(2)] if norms else [None, None]
        rope = G.Rope(rot, layout=layout, base=500000.0, attn_factor=1.25, freq_factors=ff, **opts)
        pages = G.KvPages(g, *pool.args())
        assert g.rope_append(pages, 1, q, k, v, ints(cu), rope, out=out, seqs=ints(slots), positions=positions, q_norm=w[0], k_norm=w[1],
                             eps=1e-5, wait=True), g.last_decline
        f, mag = freqs64(rot, 500000.0, scaling, 4.0, 4096, attn=1.25, ff=None if ff is None else np.float32(ff)) if rot else (np.zeros(0), 1.0)
        pos = torch.cat([torch.arange(l - n, l) for n, l in zip(rows, lens)]).cuda()
        turn = pos if positions is None else positions[:T]
        want = [rotate64(q[:T], turn, f, mag, layout, w[0], 1e-5), rotate64(k[:T], turn, f, mag, layout, w[1], 1e-5), v[:T].double()]
        # rounding of the result; the rotation itself has 32-bit sine, cosine (2^-22), products and sums, the norm another few
        big = [x.abs().amax(-1, keepdim=True) * 2 for x in want]
        tol = lambda t, x, m: HALF[t] * x.abs() + 2.0 ** -20 * m + (2.0 ** -25 if t == "f16" else 0)  # noqa: E731
        assert float(((out[:T].double() - want[0]).abs() - tol(out_ty, want[0], big[0])).max()) <= 0
        assert bool((out[T:] == 7).all())
        new_k, new_v = pool.k.clone(), pool.v.clone()
        t = 0
        for s, n, l in zip(slots, rows, lens):
            for j in range(l - n, l):
                pg = int(pool.table[s, j // page])
                got_k, got_v = new_k[1, pg, j % page].double(), new_v[1, pg, j % page].double()
                assert float(((got_k - want[1][t]).abs() - tol(cache, want[1][t], big[1][t])).max()) <= 0
                assert float(((got_v - want[2][t]).abs() - tol(cache, want[2][t], torch.zeros(1, device="cuda"))).max()) <= 0
                new_k[1, pg, j % page], new_v[1, pg, j % page] = before[0][1, pg, j % page], before[1][1, pg, j % page]
                t += 1
        # everything else in the pool is as it was
        for x, y in ((new_k, before[0]), (new_v, before[1])):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_rope_in_place_and_without_queries(G, g):
    pool = Pool(1, 9, 16, 1, 64, "f16", 2, 8, seed=8)
    r = gen(8)
    pool.fill(0, 50, r)
    pages = G.KvPages(g, *pool.args())
    q = torch.randn((5, 4, 64), generator=r, device="cuda").half()
    k, v = torch.randn((5, 1, 64), generator=r, device="cuda").half(), torch.randn((5, 1, 64), generator=r, device="cuda").half()
    rope, cu = G.Rope(64), ints([0, 5])
    out = torch.empty_like(q)
    assert g.rope_append(pages, 0, q, k, v, cu, rope, out=out, wait=True)
    kept = pool.read(0)
    for x in pool.read(0):
        x.zero_()
    assert g.rope_append(pages, 0, None, k, v, cu, rope, wait=True)
    assert all(torch.equal(a, b) for a, b in zip(pool.read(0), kept))
    assert g.rope_append(pages, 0, q, k, v, cu, rope, wait=True)
    assert torch.equal(q, out)


def test_rope_drops_what_has_no_page(G, g):
    pool = Pool(1, 6, 16, 1, 64, "f16", 2, 3, seed=9)
    pool.k.zero_()
    pool.v.zero_()
    pool.table[0, :3] = ints([-1, 6, 2])
    pool.lens[0] = 48
    pages = G.KvPages(g, *pool.args())
    r = gen(9)
    x = [torch.randn((60, h, 64), generator=r, device="cuda").half() for h in (2, 1, 1)]
    out = torch.full_like(x[0], 7.0)
    assert g.rope_append(pages, 0, *x, ints([0, 60]), None, out=out, wait=True)   # 12 rows stand before position 0
    assert torch.equal(out, x[0])
    assert torch.equal(pool.v[0, 2], x[2][44:]) and not bool(pool.v[0, [0, 1, 3, 4, 5]].any())
    pool.lens[0] = 2 ** 31 - 1   # cut to the table's row
    assert g.rope_append(pages, 0, *x, ints([0, 60]), None, out=out, wait=True)
    assert not bool(pool.v[0, [0, 1, 3, 4, 5]].any())


# ------------------------------------------------------------------------------------------- the pages' upkeep

def same(pool, book):
    assert pool.refs.tolist() == book.refs
    for s, (pages, length) in enumerate(book.seqs):
        assert int(pool.lens[s]) == length
        assert pool.table[s, : len(pages)].tolist() == pages


@pytest.mark.parametrize("seed,order,dim,cache", [(1, (0, 1, 2, 3), 64, "f16"), (2, (1, 0, 3, 2), 128, "bf16"), (3, (3, 2, 1, 0), 8, "f16")])
def test_pages_follow_the_book(G, g, seed, order, dim, cache):
    """A few hundred random steps; after each the table, lengths and holders are the book's and every sequence still reads what
    it wrote, whoever it shares pages with."""
    rnd = random.Random(seed)
    n_pages, page, slots, width, layers, kv = 37, 8, 9, 14, 2, 2
    pool = Pool(layers, n_pages, page, kv, dim, cache, slots, width, order, 0, seed)
    pages, book = G.KvPages(g, *pool.args()), Book(n_pages, page, slots, width)
    text = [[] for _ in range(slots)]   # a number per position, stored in every layer and head
    counter = 0
    done = dict(short=0, copies=0, moves=0, long=0)
    for step in range(250):
        op = rnd.choice(["reserve", "reserve", "reserve", "fork", "release", "compact"])
        some = rnd.sample(range(slots), rnd.randint(1, slots))
        if op == "reserve":
            n_new = [rnd.choice([0, 1, 1, 2, page, 3 * page + 1]) for _ in some]
            short, copies = book.reserve(some, n_new)
            ok = g.pages_reserve(pages, some, n_new, wait=True)
            assert ok == (short == 0) and int(pages.short_by) == short
            if short:
                assert g.last_decline[0] == 6
                done["short" if short > 0 else "long"] += 1
            else:
                done["copies"] += len(copies)
                for s, n in zip(some, n_new):
                    for _ in range(n):
                        at = len(text[s])
                        pg = book.seqs[s][0][at // page]
                        counter += 1
                        pool.k[:, pg, at % page], pool.v[:, pg, at % page] = counter % 251, counter % 241
                        text[s].append(counter)
        elif op == "fork":
            half = max(1, len(some) // 2)
            dst = some[half:]
            src = [rnd.choice(some[:half]) for _ in dst]
            book.fork(src, dst)
            assert g.pages_fork(pages, src, dst)
            for a, b in zip(src, dst):
                text[b] = list(text[a])
        elif op == "release":
            keep = [rnd.choice([0, 0, rnd.randint(0, 40)]) for _ in some]
            book.release(some, keep)
            assert g.pages_release(pages, some, keep)
            for s, n in zip(some, keep):
                text[s] = text[s][:n]
        else:
            to, moved = book.compact()
            page_map = torch.full((n_pages,), 99, dtype=torch.int32, device="cuda")
            assert g.pages_compact(pages, page_map=page_map if rnd.random() < 0.7 else None)
            if int(page_map[0]) != 99:
                assert page_map.tolist() == to
            done["moves"] += len(moved)
        same(pool, book)
        for s in range(slots):
            for layer in range(layers):
                k, v = pool.read(s, layer)
                want = torch.tensor(text[s], device="cuda")
                assert torch.equal(k, (want % 251).to(k.dtype)[:, None, None].expand_as(k))
                assert torch.equal(v, (want % 241).to(v.dtype)[:, None, None].expand_as(v))
    done.pop("long")  # (which has its own case below)
    assert all(done.values()), done


def test_pages_many_sequences_and_pages(G, g):
    """More pages than one sweep of a block, a thousand sequences in one list, and rows of a table with room between them."""
    n_pages, page, slots, width = 5000, 8, 1024, 20
    pool = Pool(1, n_pages, page, 1, 8, "f16", slots, width, seed=4)
    pages, book = G.KvPages(g, *pool.args()), Book(n_pages, page, slots, width)
    rnd = random.Random(5)
    seqs = rnd.sample(range(slots), slots)
    for lo, hi in ((1, 30), (0, 3)):
        n_new = [rnd.randint(lo, hi) for _ in seqs]
        assert book.reserve(seqs, n_new)[0] == 0 and g.pages_reserve(pages, seqs, n_new)
        same(pool, book)
    dst = seqs[512:]
    book.fork(seqs[:512], dst), g.pages_fork(pages, seqs[:512], dst)
    same(pool, book)
    n_new = [rnd.randint(0, 9) for _ in seqs]
    assert book.reserve(seqs, n_new)[0] == 0 and g.pages_reserve(pages, seqs, n_new)
    same(pool, book)
    book.release(seqs[::2], [0] * 512), g.pages_release(pages, seqs[::2], [0] * 512)
    book.compact(), g.pages_compact(pages)
    same(pool, book)
    assert book.reserve([seqs[0]], [width * page + 1])[0] == -1 and not g.pages_reserve(pages, [seqs[0]], [width * page + 1])
    assert not g.pages_reserve(pages, [seqs[0]], [2 ** 31 - 1]) and int(pages.short_by) == -1
    same(pool, book)
    assert g.pages_reserve(pages, [], [])


def test_pages_with_a_spoilt_table(G, g):
    """Page numbers outside the pool and lengths outside the table change nothing outside it."""
    pool = Pool(1, 6, 8, 1, 8, "f16", 4, 3, seed=6)
    pages = G.KvPages(g, *pool.args())
    pool.table[:, :3] = ints([[-1, 6, 1], [0, 2, 2 ** 31 - 1], [3, 4, 5], [-2 ** 31, 7, 8]])
    pool.lens.copy_(ints([20, 2 ** 31 - 1, -9, 11]))
    pool.refs.copy_(ints([1, 1, 1, 0, 0, 0]))
    assert g.pages_reserve(pages, [0, 2, 3], [1, 1, 1], wait=True)
    assert g.pages_fork(pages, [1], [3])
    assert g.pages_release(pages, [0, 1, 3], [0, 4, 1])
    assert g.pages_compact(pages)
    torch.cuda.synchronize()
    assert int(pool.lens[1]) == 4 and int(pool.lens[3]) == 1


# --------------------------------------------------------------------------------------------- all of it together

@pytest.mark.parametrize("cache,rows_ty,dim,page", [("f16", "f16", 128, 16), ("bf16", "bf16", 64, 32), ("f16", "f32", 128, 64)])
def test_a_serving_loop(G, g, cache, rows_ty, dim, page):
    """Prompts in pieces, decoding, a fork, an end, a compaction, more decoding: every row of every step against attention over
    the sequence's whole history, which is kept apart."""
    layers, kv, heads, slots = 2, 2, 8, 5
    pool = Pool(layers, 4000 // page, page, kv, dim, cache, slots, 2000 // page, seed=11)
    pages = G.KvPages(g, *pool.args())
    rope, r, scale = G.Rope(dim // 2, layout="pairs", base=1e4, scaling="linear", factor=2.0), gen(11), dim ** -0.5
    f, mag = freqs64(dim // 2, 1e4, "linear", 2.0)
    hist = {}

    def step(seqs, rows):
        assert g.pages_reserve(pages, seqs, rows), g.last_decline
        T, cu = sum(rows), np.cumsum([0] + rows).tolist()
        for layer in range(layers):
            qkv = torch.randn((T, heads + 2 * kv, dim), generator=r, device="cuda").to(TY[rows_ty])
            q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
            turned = torch.empty((T, heads, dim), dtype=TY[rows_ty], device="cuda")
            out = torch.empty_like(turned)
            assert g.rope_append(pages, layer, q, k, v, ints(cu), rope, out=turned, seqs=ints(seqs))
            assert g.attend_pages(pages, layer, turned, ints(cu), scale, out, seqs=ints(seqs), wait=True)
            for i, s in enumerate(seqs):
                part = slice(cu[i], cu[i + 1])
                old = hist.setdefault((s, layer), (torch.zeros((0, kv, dim), device="cuda", dtype=TY[cache]),) * 2)
                at = torch.arange(old[0].shape[0], old[0].shape[0] + rows[i], device="cuda")
                got = pool.read(s, layer)
                want_k = rotate64(k[part], at, f, mag, "pairs")
                # the history is what the sequence read back when it was written: new rows are within a rounding, old ones untouched
                assert torch.equal(got[0][: len(old[0])], old[0]) and torch.equal(got[1][: len(old[1])], old[1])
                assert bool(((got[0][len(old[0]):].double() - want_k).abs() <= HALF[cache] * want_k.abs() + 2.0 ** -18 * want_k.abs().amax() + 2.0 ** -25).all())
                assert torch.equal(got[1][len(old[1]):], v[part].to(TY[cache]))
                hist[s, layer] = tuple(x.clone() for x in got)
                ref = attend64(turned[part], *hist[s, layer], scale)
                assert float(((out[part].double() - ref[0]).abs() - attend_bound(*ref, rows_ty)).max()) <= 0

    step([0, 2], [300, 45])
    step([0, 2, 3], [277, 1, 1])
    for _ in range(3):
        step([3, 0, 2], [1, 1, 1])
    assert g.pages_fork(pages, [0, 0], [1, 4])
    for layer in range(layers):
        hist[1, layer] = hist[4, layer] = hist[0, layer]
    step([0, 1, 4, 2], [1, 3, 1, 1])
    assert g.pages_release(pages, [0, 2], [0, 20])
    for layer in range(layers):
        hist[2, layer] = tuple(x[:20] for x in hist[2, layer])
        del hist[0, layer]
    assert g.pages_compact(pages)
    step([4, 1, 2, 0], [1, 1, 1, 130])
    step([0, 1, 2, 3, 4], [1, 1, 1, 1, 1])


def test_a_captured_step_is_replayed(G, g):
    """One decode step of three sequences in a CUDA graph: each replay adds a position and attends over one more; a second graph
    over another pool, replayed on another stream at the same time, does not disturb it."""
    def make(seed):
        pool = Pool(1, 40, 16, 2, 64, "f16", 3, 12, seed=seed)
        r = gen(seed)
        for s, l in enumerate((15, 90, 33)):
            pool.fill(s, l, r)
        x = [torch.randn((3, h, 64), generator=r, device="cuda").half() for h in (8, 2, 2)]
        return pool, G.KvPages(g, *pool.args()), x, torch.empty_like(x[0]), torch.empty_like(x[0])

    rope, cu = G.Rope(64), ints([0, 1, 2, 3])

    def step(pages, x, turned, out, **kw):
        assert g.pages_reserve(pages, [0, 1, 2], [1, 1, 1], wait=False, **kw)
        assert g.rope_append(pages, 0, *x, cu, rope, out=turned, **kw)
        assert g.attend_pages(pages, 0, turned, cu, 0.125, out, **kw)

    both = [make(21), make(22)]
    streams, graphs = [torch.cuda.Stream() for _ in both], []
    for (pool, pages, x, turned, out), st in zip(both, streams):
        step(pages, x, turned, out)   # once eagerly
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step(pages, x, turned, out)
        graphs.append(graph)
    for i in range(20):
        for b, st, graph in zip(both, streams, graphs):
            with torch.cuda.stream(st):
                b[2][0].mul_(0.9)
                b[2][1].mul_(1.1)
                graph.replay()
    torch.cuda.synchronize()
    for pool, pages, x, turned, out in both:
        assert pool.lens.tolist() == [36, 111, 54] and int(pages.short_by) == 0
        for s in range(3):
            k, v = pool.read(s)
            ref = attend64(turned[s:s + 1], k, v, 0.125)
            assert float(((out[s:s + 1].double() - ref[0]).abs() - attend_bound(*ref, "f16")).max()) <= 0


def test_captured_upkeep_is_replayed(G, g):
    """Fork, growth, release and compaction in one CUDA graph: its lists stay, the state moves on with every replay."""
    pool = Pool(2, 60, 8, 1, 64, "f16", 5, 12, seed=23)
    pages, book = G.KvPages(g, *pool.args()), Book(60, 8, 5, 12)
    assert g.pages_reserve(pages, [0, 1, 3], [13, 30, 5]) and book.reserve([0, 1, 3], [13, 30, 5])[0] == 0
    page_map = torch.zeros(60, dtype=torch.int32, device="cuda")

    def step():
        assert g.pages_fork(pages, [0, 1], [2, 4])
        assert g.pages_reserve(pages, [0, 2, 4], [3, 1, 9], wait=False)
        assert g.pages_release(pages, [1, 3], [21, 2])
        assert g.pages_compact(pages, page_map=page_map)

    def by_hand():
        book.fork([0, 1], [2, 4])
        assert book.reserve([0, 2, 4], [3, 1, 9])[0] == 0
        book.release([1, 3], [21, 2])
        return book.compact()[0]

    step()
    by_hand()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(6):
        graph.replay()
        to = by_hand()
        torch.cuda.synchronize()
        same(pool, book)
        assert page_map.tolist() == to and int(pages.short_by) == 0


def test_streams_and_counters(G, g):
    """Work goes to the stream it is given (here: after a producer on that stream) and is counted."""
    pool = Pool(1, 40, 16, 2, 128, "f16", 1, 40, seed=31)
    r = gen(31)
    k, v = pool.fill(0, 500, r)
    pages = G.KvPages(g, *pool.args())
    q, out = torch.zeros((1, 8, 128), device="cuda").half(), torch.zeros((1, 8, 128), device="cuda").half()
    want = torch.randn((1, 8, 128), generator=r, device="cuda").half()
    big = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    before = g.stats()[:2]
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        for _ in range(10):
            big = big @ big * 1e-4
        q.copy_(want)
        assert g.attend_pages(pages, 0, q, ints([0, 1]), 0.1, out)
    st.synchronize()
    ref = attend64(want, k, v, 0.1)
    assert float(((out.double() - ref[0]).abs() - attend_bound(*ref, "f16")).max()) <= 0
    after = g.stats()[:2]
    assert after[0] == before[0] + 1 and after[1] > before[1]
