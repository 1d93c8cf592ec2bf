"""The paged KV cache on a GPU, where its operators could go wrong: what hidden positions hold beside tiles that are cut over
many blocks, and what the calls report and leave behind."""
import math

import pytest
import torch

from tests.pages_util import TY, Pool, attend64, attend_bound

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


# ------------------------------------------------------------------------------- hidden values beside cut tiles

def hidden_case(G, g, rows, lens, spoils, *, cache, rows_ty, kv, group, dim, window=0, page=16, seed=60):
    """spoils: (sequence, position, value): V of that position, every head, one dimension.  The output is held against 64
    bits, with finite values in it beforehand and with NaN, and has the same bits both times."""
    ty, heads, n = rows_ty or cache, kv * group, len(rows)
    pool = Pool(1, sum(-(-x // page) for x in lens) + 1, page, kv, dim, cache, n, max(-(-x // page) for x in lens), seed=seed)
    r = gen(seed)
    for s, x in enumerate(lens):
        pool.fill(s, x, r)
    for s, j, x in spoils:
        pool.v[0, int(pool.table[s, j // page]), j % page, :, dim // 2 + 3] = x
    cu = [0]
    for x in rows:
        cu.append(cu[-1] + x)
    q = (torch.randn((cu[-1], heads, dim), generator=r, device="cuda") * 1.5).to(TY[ty])
    pages, scale, outs = G.KvPages(g, *pool.args()), dim ** -0.5, []
    for before in (7.0, math.nan):
        out = torch.full_like(q, before)
        assert g.attend_pages(pages, 0, q, ints(cu), scale, out, window=window, wait=True), g.last_decline
        outs.append(out)
    for s in range(n):
        part = slice(cu[s], cu[s + 1])
        k, v = pool.read(s)
        o, a, most = attend64(q[part], k, v, scale, True, window)
        got, fine = outs[0][part].double(), torch.isfinite(o)
        assert torch.equal(torch.isfinite(got), fine), (s, (~torch.isfinite(got) & fine).any(2).nonzero().tolist()[:9])
        assert float(((got - o).abs() - attend_bound(o, a, most, ty))[fine].max()) <= 0
    assert torch.equal(outs[0].view(torch.uint8), outs[1].view(torch.uint8))
    return outs[0]


KINDS = [("f16", None), ("bf16", None), ("f16", "f32")]


@pytest.mark.parametrize("cache,rows_ty", KINDS)
@pytest.mark.parametrize("dim,kv,group", [(128, 8, 4), (128, 8, 1), (64, 4, 4), (128, 2, 5), (64, 2, 8), (128, 1, 48)])
def test_drafts_do_not_see_a_later_drafts_infinity(G, g, cache, rows_ty, dim, kv, group):
    """Every tile is cut over several blocks; only the last of eight rows sees the infinity."""
    n, length = 5, 6000
    out = hidden_case(G, g, [8] * n, [length] * n, [(s, length - 1, math.inf if s % 2 else -math.inf) for s in range(n)], cache=cache, rows_ty=rows_ty,
                      kv=kv, group=group, dim=dim)
    assert bool(torch.isfinite(out.view(n, 8, -1)[:, :7]).all())


@pytest.mark.parametrize("cache,rows_ty", KINDS)
@pytest.mark.parametrize("dim,group", [(128, 1), (128, 4), (64, 5), (64, 8), (128, 16)])
@pytest.mark.parametrize("rows", [1, 5, 8])
def test_what_lies_before_the_window_does_not_matter(G, g, cache, rows_ty, dim, group, rows):
    """Cut tiles meet the infinity in their first block, where no row sees it; beside them a clean chunk of many rows."""
    lens, window = [5003, 4100, 700], 3000
    spoils = [(s, lens[s] - rows - window, x) for s, x in ((0, -math.inf), (1, math.nan))]
    for s, j, _ in spoils:   # (the position in front of the first row's window, in the same block of 128)
        assert j // 128 == (j + 1) // 128
    out = hidden_case(G, g, [rows, rows, 300], lens, spoils, cache=cache, rows_ty=rows_ty, kv=2, group=group, dim=dim, window=window)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("cache,rows_ty", KINDS)
@pytest.mark.parametrize("dim,group", [(128, 4), (64, 7)])
def test_a_long_chunk_does_not_see_behind_itself(G, g, cache, rows_ty, dim, group):
    """Tiles of 256 rows, cut; whole ones beside them in the same call."""
    out = hidden_case(G, g, [200, 1, 90], [9000, 60, 90], [(0, 8990, math.nan), (2, 89, math.inf)], cache=cache, rows_ty=rows_ty, kv=2, group=group, dim=dim)
    assert bool(torch.isfinite(out[:190]).all()) and bool(torch.isfinite(out[200:290]).all())


# ------------------------------------------------------------------------------------------- the pages' upkeep

@pytest.mark.parametrize("n", [15, 18])
def test_reserve_of_more_pages_than_32_bits_count(G, g, n):
    """Sequences of 2^30 - 8 positions each: 15 of them ask for fewer than 2^31 pages, 18 for more."""
    pages, page, width = 6, 8, 2 ** 27 - 1
    k, v = (torch.zeros((1, pages, page, 1, 8), dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.empty((n, width), dtype=torch.int32, device="cuda")
    lens, refs = ints([0] * n), ints([0, 1, 0, 0, 0, 0])
    pool = G.KvPages(g, k, v, table, lens, refs)
    assert not g.pages_reserve(pool, range(n), [width * page] * n) and g.last_decline[0] == 6
    assert int(pool.short_by) == min(n * width - 5, 2 ** 31 - 1)
    assert not bool(lens.any()) and refs.tolist() == [0, 1, 0, 0, 0, 0]
    assert g.pages_reserve(pool, range(n), [9] + [0] * (n - 1)) and table[0, :2].tolist() == [0, 2]


def test_an_earlier_calls_expired_wait_and_a_reservation(G, g):
    """work[1] is where attention leaves an expired wait (planted here).  A waited reservation that reports it has changed
    nothing, so it can be repeated; one that is not waited for does its work and leaves the report to the next waited call."""
    pool = Pool(1, 20, 16, 2, 64, "f16", 2, 8, seed=70)
    r = gen(70)
    pool.fill(0, 30, r)
    pages = G.KvPages(g, *pool.args())
    refs, table = pool.refs.clone(), pool.table.clone()
    pages.work[1] = 7
    with pytest.raises(G.GpuError) as e:
        g.pages_reserve(pages, [0, 1], [10, 5])
    assert e.value.code == -3 and int(pages.short_by) == -2
    assert pool.lens.tolist() == [30, 0] and torch.equal(pool.refs, refs) and torch.equal(pool.table, table)
    assert g.pages_reserve(pages, [0, 1], [10, 5]) and pool.lens.tolist() == [40, 5] and int(pages.short_by) == 0
    pages.work[1] = 7
    assert g.pages_reserve(pages, [0, 1], [1, 1], wait=False) and int(pages.short_by) == 0 and pool.lens.tolist() == [41, 6]
    x = [torch.randn((2, h, 64), generator=r, device="cuda").half() for h in (4, 2, 2)]
    turned = torch.empty_like(x[0])
    assert g.rope_append(pages, 0, *x, ints([0, 1, 2]), None, out=turned, wait=True) and torch.equal(turned, x[0])
    with pytest.raises(G.GpuError) as e:
        g.attend_pages(pages, 0, turned, ints([0, 1, 2]), 0.1, torch.empty_like(turned), wait=True)
    assert e.value.code == -3
    assert g.attend_pages(pages, 0, turned, ints([0, 1, 2]), 0.1, torch.empty_like(turned), wait=True)


def test_a_step_without_rows(G, g):
    pool = Pool(1, 4, 16, 2, 64, "f16", 2, 2, seed=71)
    pages = G.KvPages(g, *pool.args())
    q, k = (torch.empty((0, h, 64), dtype=torch.float16, device="cuda") for h in (4, 2))
    for cu, seqs in ((ints([0]), None), (ints([0, 0, 0]), ints([1, 0]))):
        assert g.rope_append(pages, 0, q, k, k, cu, G.Rope(64), seqs=seqs, wait=True)
        assert g.attend_pages(pages, 0, q, cu, 0.1, torch.empty_like(q), seqs=seqs, wait=True)
    assert g.pages_reserve(pages, [0, 1], [0, 0]) and not bool(pool.refs.any())


def test_a_pool_made_on_a_busy_stream_is_used_on_another(G, g):
    """Forks and their copies on a side stream, right after the pool was made on a stream with work in front of it."""
    pool = Pool(2, 40, 16, 2, 64, "f16", 9, 3, seed=72)
    r = gen(72)
    held = pool.fill(0, 25, r)
    pool.k[1], pool.v[1] = pool.k[0], pool.v[0]
    big = torch.randn((8192, 8192), device="cuda")
    torch.cuda.synchronize()
    for _ in range(8):
        big = big @ big * 1e-4
    pages, st = G.KvPages(g, *pool.args()), torch.cuda.Stream()
    kids = list(range(1, 9))
    assert g.pages_fork(pages, [0] * 8, kids, stream=st.cuda_stream)
    assert g.pages_reserve(pages, kids, [1] * 8, stream=st.cuda_stream, wait=False)
    torch.cuda.synchronize()
    assert int(pages.short_by) == 0 and pool.lens.tolist() == [25] + [26] * 8
    for s in kids:
        for layer in (0, 1):
            k, v = pool.read(s, layer)
            assert torch.equal(k[:25], held[0]) and torch.equal(v[:25], held[1])


def test_an_expired_wait_in_attention_is_reported_and_the_pool_lives_on(G):
    """Sixteen million rows of one sequence, nearly all before its position 0: the warp that looks for a block's share of the work
    walks 65536 tiles before it hands out the first one, milliseconds, and the others' waits for it run out under a budget
    of a cycle.  The call reports it, a second one with the ordinary budget is right."""
    g = G.Gpu(0)
    rows, length = 1 << 24, 40
    pool = Pool(1, 4, 16, 1, 64, "f16", 1, 3, seed=73)
    r = gen(73)
    k, v = pool.fill(0, length, r)
    pages = G.KvPages(g, *pool.args())
    row = torch.randn((1, 1, 64), generator=r, device="cuda").half()
    q, out = row.expand(rows, 1, 64), torch.full((rows, 1, 64), 7.0, dtype=torch.float16, device="cuda")
    call = lambda **kw: g.attend_pages(pages, 0, q, ints([0, rows]), 0.1, out, **kw)  # noqa: E731
    g.debug_set_wait_limit(1)
    with pytest.raises(G.GpuError) as e:
        call(wait=True)
    assert e.value.code == -3 and "site 10" in str(e.value)
    assert call(wait=False)
    with pytest.raises(G.GpuError) as e:
        g.pages_reserve(pages, [0], [1])
    assert e.value.code == -3 and int(pool.lens[0]) == length
    g.debug_set_wait_limit(0)
    assert call(wait=True)
    o, a, most = attend64(q[:length], k, v, 0.1)
    assert not bool(out[: rows - length].any())
    assert float(((out[rows - length:].double() - o).abs() - attend_bound(o, a, most, "f16")).max()) <= 0
    assert g.pages_reserve(pages, [0], [1]) and int(pool.lens[0]) == length + 1
    g.close()


# ------------------------------------------------------------------------------------------------- the largest batch

def test_a_step_of_as_many_sequences_as_a_batch_takes(G, g):
    """4096 sequences, in any order: prompts of 1 to 40 rows, then a token each; every hundredth is held against 64 bits."""
    n, page, dim, group = 4096, 8, 64, 2
    rows = torch.randint(1, 41, (n,), generator=torch.Generator().manual_seed(80))
    pool = Pool(1, int(((rows + 8) // page).sum()), page, 1, dim, "f16", n, 6, seed=80)
    pages, r, order = G.KvPages(g, *pool.args()), gen(80), torch.randperm(n, generator=torch.Generator().manual_seed(81))
    for step in (rows, torch.ones_like(rows)):
        for part in order.split(1024):
            assert g.pages_reserve(pages, part, step[part])
        mine = step[order]
        cu = torch.cat([torch.zeros(1, dtype=torch.int64), mine.cumsum(0)]).int().cuda()
        total = int(mine.sum())
        q, k, v = (torch.randn((total, h, dim), generator=r, device="cuda").half() for h in (group, 1, 1))
        out, seqs = torch.empty_like(q), order.int().cuda()
        assert g.rope_append(pages, 0, q, k, v, cu, None, seqs=seqs)
        assert g.attend_pages(pages, 0, q, cu, dim ** -0.5, out, seqs=seqs, wait=True)
        ends = cu.tolist()
        for i in list(range(0, n, 100)) + [n - 1]:
            part, (pk, pv) = slice(ends[i], ends[i + 1]), pool.read(int(order[i]))
            assert torch.equal(pk[-int(mine[i]):], k[part]) and torch.equal(pv[-int(mine[i]):], v[part])
            o, a, most = attend64(q[part], pk, pv, dim ** -0.5)
            assert float(((out[part].double() - o).abs() - attend_bound(o, a, most, "f16")).max()) <= 0
    assert pool.lens.tolist() == (rows + 1).tolist()
