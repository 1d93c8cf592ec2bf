"""The paged KV cache without a GPU: what its entry points refuse, the C layouts, and the test's own bookkeeping."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def gpu():
    from allpaka_b200 import build, gpu as G

    build.build()
    G.load_library()
    return G


class Tensor:
    """The face of a device tensor."""

    def __init__(self, *shape, dtype="float16", device=0, stride=None, ptr=1 << 20):
        self.shape, self.dtype, self._ptr = tuple(shape), f"torch.{dtype}", ptr
        self.device = type("D", (), dict(type="cuda", index=device, __str__=lambda s: f"cuda:{device}"))()
        if stride is None:
            stride, n = [], 1
            for x in reversed(shape):
                stride.insert(0, n)
                n *= x
            self._dense = True
        else:
            self._dense = False
        self._stride = tuple(stride)

    def stride(self, i=None):
        return self._stride if i is None else self._stride[i]

    def get_device(self):
        return self.device.index

    def is_contiguous(self):
        return self._dense

    def data_ptr(self):
        return self._ptr

    def numel(self):
        n = 1
        for x in self.shape:
            n *= x
        return n

    def new_zeros(self, n):
        return Tensor(n, dtype="int32")

    new_empty = new_zeros

    def __getitem__(self, i):
        return Tensor(dtype="int32")


@pytest.fixture
def ctx(gpu):
    """A context that no call may get as far as using: the refusals come before the first look at it."""
    g = gpu.Gpu.__new__(gpu.Gpu)
    g._l, g._device = gpu.load_library(), 0
    block = C.create_string_buffer(1 << 16)
    g._h = C.c_void_p(C.addressof(block))
    yield g
    g._h = None


def pool(gpu, g, layers=2, pages=10, page=16, kv=2, dim=128, dtype="float16", seqs=3, width=5, **kw):
    a = dict(k=Tensor(layers, pages, page, kv, dim, dtype=dtype), v=Tensor(layers, pages, page, kv, dim, dtype=dtype),
             table=Tensor(seqs, width, dtype="int32"), lens=Tensor(seqs, dtype="int32"), refs=Tensor(pages, dtype="int32"))
    return gpu.KvPages(g, **(a | kw))


def test_struct_sizes_against_the_compiler(gpu, tmp_path):
    src = tmp_path / "sz.c"
    src.write_text('#include "allpaka_b200.h"\n#include <stdio.h>\n#include <stddef.h>\n'
                   'int main(void){printf("%zu %zu %zu %zu %zu %zu %zu %u\\n", sizeof(apk_pages), sizeof(apk_rope), sizeof(apk_rope_req),'
                   ' sizeof(apk_attend_req), offsetof(apk_pages, work), offsetof(apk_rope_req, eps), offsetof(apk_attend_req, ws),'
                   ' APK_PAGES_WORK(10, 3));return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert (gpu._ATTEND_REQ.size, gpu._ROPE_REQ.size) == (C.sizeof(gpu._AttendReq), C.sizeof(gpu._RopeReq))
    assert got == [C.sizeof(gpu._Pages), C.sizeof(gpu._Rope), C.sizeof(gpu._RopeReq), C.sizeof(gpu._AttendReq), gpu._Pages.work.offset,
                   gpu._RopeReq.eps.offset, gpu._AttendReq.ws.offset, 64 + 4 * 3 + 3 * 10]


def test_a_pool_of_the_wrong_tensors(gpu, ctx):
    for bad in (dict(k=Tensor(2, 10, 16, 2, 128, dtype="float32")), dict(v=Tensor(2, 10, 16, 2, 64)), dict(k=Tensor(10, 16, 2, 128)),
                dict(v=Tensor(2, 10, 16, 2, 128, dtype="bfloat16")), dict(table=Tensor(3, 5, dtype="int64")), dict(lens=Tensor(4, dtype="int32")),
                dict(refs=Tensor(9, dtype="int32")), dict(k=Tensor(2, 10, 16, 2, 128, device=1)),
                dict(k=Tensor(2, 10, 16, 2, 128, stride=(1, 2, 20, 320, 640))), dict(table=Tensor(3, 5, dtype="int32", stride=(1, 3))),
                dict(lens=Tensor(3, dtype="int32", stride=(2,)))):
        with pytest.raises(ValueError):
            pool(gpu, ctx, **bad)


def test_a_table_whose_rows_overlap(gpu, ctx):
    """One row for all sequences (an expanded tensor): its storage ends long before the last row of a table would."""
    for stride in ((0, 1), (4, 1)):
        with pytest.raises(ValueError):
            pool(gpu, ctx, table=Tensor(3, 5, dtype="int32", stride=stride))
    one = pool(gpu, ctx, table=Tensor(1, 5, dtype="int32", stride=(0, 1)), lens=Tensor(1, dtype="int32"))
    assert one._c.table_stride == 5
    assert pool(gpu, ctx, table=Tensor(3, 5, dtype="int32", stride=(9, 1)))._c.table_stride == 9


@pytest.mark.parametrize("kw,code", [(dict(page=24), 3), (dict(page=4), 3), (dict(page=512), 3), (dict(dim=20), 3), (dict(dim=264), 3),
                                     (dict(k=Tensor(2, 10, 16, 2, 128, ptr=(1 << 20) + 8)), 3),
                                     (dict(k=Tensor(2, 10, 16, 2, 128, stride=(41000, 4100, 256, 128, 1))), 3), (dict(width=1 << 27), 3)])
def test_pools_that_are_declined(gpu, ctx, kw, code):
    p = pool(gpu, ctx, **kw)
    for call in (lambda: ctx.pages_reserve(p, [0], [1], stream=0), lambda: ctx.pages_fork(p, [0], [1], stream=0),
                 lambda: ctx.pages_release(p, [0], [1], stream=0), lambda: ctx.pages_compact(p, stream=0)):
        assert call() is False and ctx.last_decline[0] == code


def test_lists_that_are_refused(gpu, ctx):
    p = pool(gpu, ctx)
    for f, a, b in ((ctx.pages_reserve, [3], [1]), (ctx.pages_reserve, [-1], [1]), (ctx.pages_reserve, [0], [-1]), (ctx.pages_reserve, [1, 1], [1, 1]),
                    (ctx.pages_fork, [0], [0]), (ctx.pages_fork, [0, 1], [2, 2]), (ctx.pages_fork, [0, 1], [1, 2]), (ctx.pages_fork, [0], [3]),
                    (ctx.pages_fork, [-1], [2]), (ctx.pages_release, [0], [-1]), (ctx.pages_release, [2, 2], [0, 0]), (ctx.pages_release, [7], [0])):
        with pytest.raises(gpu.GpuError) as e:
            f(p, a, b, stream=0)
        assert e.value.code == -1
    for a, b in (([0], [1, 2]), ([0.5], [1]), ([2 ** 40], [1])):
        with pytest.raises(ValueError):
            ctx.pages_reserve(p, a, b, stream=0)
    big = pool(gpu, ctx, seqs=3000)
    assert ctx.pages_reserve(big, range(1025), [1] * 1025, stream=0) is False and ctx.last_decline[0] == 3
    assert ctx.pages_fork(p, [], [], stream=0) and ctx.pages_release(p, [], [], stream=0)   # nothing to do
    with pytest.raises(ValueError):
        ctx.pages_compact(p, page_map=Tensor(9, dtype="int32"), stream=0)
    other = pool(gpu, ctx)
    other.device = 1
    with pytest.raises(ValueError):
        ctx.pages_reserve(other, [0], [1], stream=0)


def attend(ctx, p, q=None, out=None, cu=None, layer=0, scale=0.1, **kw):
    q = q or Tensor(4, 8, 128)
    out = out or Tensor(*q.shape, dtype=q.dtype[6:], ptr=2 << 20)
    return ctx.attend_pages(p, layer, q, cu or Tensor(3, dtype="int32"), scale, out, stream=0, **kw)


def test_attention_requests_that_are_refused(gpu, ctx):
    p = pool(gpu, ctx)
    for kw in (dict(q=Tensor(4, 8, 64)), dict(q=Tensor(4, 8, 128, dtype="int32")), dict(out=Tensor(4, 8, 128, dtype="float32")), dict(out=Tensor(3, 8, 128)),
               dict(layer=2), dict(layer=-1), dict(cu=Tensor(3, dtype="int64")), dict(cu=Tensor(0, dtype="int32")), dict(seqs=Tensor(3, dtype="int32")),
               dict(window=-1), dict(q=Tensor(4, 8, 128, device=1)), dict(q=Tensor(4, 8, 128, stride=(1, 4, 32)))):
        with pytest.raises(ValueError):
            attend(ctx, p, **kw)
    for kw, code in ((dict(q=Tensor(4, 7, 128)), 3), (dict(q=Tensor(4, 130, 128)), 3), (dict(q=Tensor(4, 0, 128)), 3), (dict(q=Tensor(4, 8, 128, dtype="bfloat16")), 2),
                     (dict(q=Tensor(4, 8, 128, ptr=(1 << 20) + 8)), 3), (dict(q=Tensor(4, 8, 128, stride=(1028, 128, 1))), 3), (dict(window=1 << 30), 3),
                     (dict(cu=Tensor(5000, dtype="int32")), 3)):
        assert attend(ctx, p, **kw) is False and ctx.last_decline[0] == code, kw
    assert attend(ctx, pool(gpu, ctx, dim=96), q=Tensor(4, 8, 96)) is False and ctx.last_decline[0] == 3
    assert attend(ctx, pool(gpu, ctx, dtype="bfloat16"), q=Tensor(4, 8, 128, dtype="float32")) is False and ctx.last_decline[0] == 2
    for kw in (dict(scale=float("inf")), dict(scale=float("nan")), dict(out=Tensor(4, 8, 128))):
        with pytest.raises(gpu.GpuError) as e:
            attend(ctx, p, **kw)
        assert e.value.code == -1
    assert attend(ctx, p, q=Tensor(0, 8, 128)) and attend(ctx, p, cu=Tensor(1, dtype="int32"))   # no rows, no sequences


def test_batches_without_rows_are_nothing_to_do(gpu, ctx):
    """A tensor without elements has no address (0)."""
    p = pool(gpu, ctx)
    none = {h: Tensor(0, h, 128, ptr=0) for h in (8, 2)}
    for n in (1, 3):
        cu = Tensor(n, dtype="int32")
        assert attend(ctx, p, q=none[8], out=none[8], cu=cu)
        for q in (none[8], None):
            for out in (None, none[8]):
                assert ctx.rope_append(p, 0, q, none[2], none[2], cu, gpu.Rope(64), out=out, stream=0)
    with pytest.raises(ValueError):
        attend(ctx, p, q=none[8], out=Tensor(1, 8, 128))
    with pytest.raises(gpu.GpuError):   # rows without an address
        attend(ctx, p, q=Tensor(4, 8, 128, ptr=0))


def rope_call(ctx, p, rope, q=None, k=None, v=None, out=None, **kw):
    q, k, v = q or Tensor(4, 8, 128), k or Tensor(4, 2, 128), v or Tensor(4, 2, 128)
    return ctx.rope_append(p, 0, q, k, v, Tensor(3, dtype="int32"), rope, out=out or Tensor(4, 8, 128, ptr=2 << 20), stream=0, **kw)


def test_rotations_that_are_refused(gpu, ctx):
    p = pool(gpu, ctx)
    for kw in (dict(layout="third"), dict(scaling="more"), dict(freq_factors=[1.0, 2.0])):
        with pytest.raises(ValueError):
            gpu.Rope(64, **kw)
    for dim in (3, 130, 256):
        assert rope_call(ctx, p, gpu.Rope(dim)) is False and ctx.last_decline[0] == 3
    for r in (gpu.Rope(64, base=1.0), gpu.Rope(64, base=float("inf")), gpu.Rope(64, scaling="linear", factor=0.0), gpu.Rope(64, scaling="yarn", factor=2.0),
              gpu.Rope(64, scaling="yarn", factor=2.0, orig_ctx=4096, beta_slow=0.0), gpu.Rope(64, freq_factors=[0.0] * 32)):
        with pytest.raises(gpu.GpuError) as e:
            rope_call(ctx, p, r)
        assert e.value.code == -1
    for kw in (dict(k=Tensor(4, 3, 128)), dict(v=Tensor(5, 2, 128)), dict(q=Tensor(4, 8, 128, dtype="float32")), dict(q_norm=Tensor(64, dtype="float32")),
               dict(k_norm=Tensor(128)), dict(positions=Tensor(4, dtype="int64"))):
        with pytest.raises(ValueError):
            rope_call(ctx, p, gpu.Rope(64), **kw)
    assert rope_call(ctx, p, gpu.Rope(64), k=Tensor(4, 2, 128, ptr=(1 << 20) + 2)) is False and ctx.last_decline[0] == 3
    with pytest.raises(gpu.GpuError):
        rope_call(ctx, p, gpu.Rope(64), out=Tensor(4, 8, 128, dtype="float32"))   # in place, but of another type


def test_what_has_been_told_to_the_c_side_cannot_be_changed(gpu, ctx):
    """Neither a rotation nor a pool takes a later assignment that its calls would not follow."""
    import dataclasses

    rope = gpu.Rope(64, scaling="linear", factor=2.0, freq_factors=[1.0] * 32)
    for name in ("dim", "layout", "base", "scaling", "factor", "orig_ctx", "beta_fast", "beta_slow", "attn_factor", "freq_factors"):
        with pytest.raises(AttributeError):
            setattr(rope, name, getattr(rope, name))
    other = dataclasses.replace(rope, factor=4.0)
    assert (rope._c.factor, other._c.factor, other._c.rot_dim) == (2.0, 4.0, 64) and other._p == C.addressof(other._c) != rope._p
    p = pool(gpu, ctx)
    for name in ("k", "v", "table", "lens", "refs", "work", "short_by", "n_layers", "n_pages", "page", "n_kv_heads", "head_dim", "n_seqs", "width"):
        with pytest.raises(AttributeError):
            setattr(p, name, getattr(p, name))


def test_a_scale_beyond_32_bits_is_refused(gpu, ctx):
    """The kernels work in powers of two: it is the scale times log2(e) that has to be finite."""
    p = pool(gpu, ctx)
    for scale in (3e38, -3e38):
        with pytest.raises(gpu.GpuError) as e:
            attend(ctx, p, scale=scale)
        assert e.value.code == -1 and "scale" in str(e.value)
    assert attend(ctx, p, q=Tensor(0, 8, 128, ptr=0), scale=2e38)


def test_long_lists_that_are_refused(gpu, ctx):
    """A thousand sequences in any order: one named twice, or forked and written, wherever it stands."""
    import random

    p, rnd = pool(gpu, ctx, table=Tensor(3000, 5, dtype="int32"), lens=Tensor(3000, dtype="int32")), random.Random(3)
    some = rnd.sample(range(3000), 2048)
    src, dst = some[:1024], some[1024:]
    for i, j in ((0, 1023), (1023, 0), (511, 512), (7, 900)):
        twice, both = list(dst), list(src)
        twice[i] = dst[j]
        both[i] = dst[j]
        for call, word in ((lambda: ctx.pages_fork(p, src, twice, stream=0), "twice"), (lambda: ctx.pages_reserve(p, twice, [1] * 1024, stream=0), "twice"),
                           (lambda: ctx.pages_release(p, twice, [0] * 1024, stream=0), "twice"), (lambda: ctx.pages_fork(p, both, dst, stream=0), "both")):
            with pytest.raises(gpu.GpuError) as e:
                call()
            assert e.value.code == -1 and word in str(e.value) and str(dst[j]) in str(e.value)


def test_a_workspace_that_is_not_what_its_size_says(gpu, ctx):
    """An expanded tensor counts elements that it does not have."""
    p, small = pool(gpu, ctx), Tensor(1 << 28, dtype="uint8", stride=(0,))
    small.element_size = lambda: 1
    with pytest.raises(ValueError):
        attend(ctx, p, workspace=small)


def test_null_requests_are_refused(gpu):
    lib, block = gpu.load_library(), C.create_string_buffer(1 << 16)
    h = C.addressof(block)
    empty = gpu._Pages()
    assert lib.apk_rope_append(h, None, None, 0) == -1 and lib.apk_attend_pages(h, None, None, 0) == -1
    assert lib.apk_rope_append(None, C.byref(gpu._RopeReq()), None, 0) == -1 and lib.apk_attend_pages(h, C.byref(gpu._AttendReq()), None, 0) == -1
    assert lib.apk_pages_compact(h, None, None, None) == -1 and lib.apk_pages_compact(h, C.byref(empty), None, None) == -1
    assert lib.apk_pages_reserve(None, C.byref(empty), 0, None, None, None, 0) == -1
    assert b"null" in lib.apk_last_error(None)


def test_the_book_of_the_gpu_tests():
    """Copy on write, sharing and compaction on an example worked out by hand."""
    from tests.pages_util import Book

    b = Book(pages=8, page=4, slots=3, width=5)
    assert b.reserve([0], [6]) == (0, []) and b.seqs[0] == ([0, 1], 6)
    b.fork([0, 0], [1, 2])
    assert b.refs == [3, 3, 0, 0, 0, 0, 0, 0]
    # three holders write into page 1: two copies, the last of the list keeps it
    assert b.reserve([1, 0, 2], [1, 3, 0]) == (0, [(1, 2, 2), (1, 3, 2)])
    assert b.seqs == [([0, 3, 4], 9), ([0, 2], 7), ([0, 1], 6)] and b.refs == [3, 1, 1, 1, 1, 0, 0, 0]
    assert b.reserve([0, 1], [11, 5])[0] == 0 and b.seqs[0][0] == [0, 3, 4, 5, 6]
    assert b.reserve([2], [11]) == (3, []) and b.reserve([2], [15]) == (-1, [])
    b.release([0, 1], [0, 5])
    assert b.refs == [2, 1, 1, 0, 0, 0, 0, 0]
    b.release([2], [0])
    assert b.compact() == ([0, -1, 1, -1, -1, -1, -1, -1], [(2, 1)]) and b.seqs[1] == ([0, 1], 5)
