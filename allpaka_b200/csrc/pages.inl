// The paged KV cache: argument checks and launches of apk_rope_append, apk_attend_pages and apk_pages_*.
// Kernels in pages.cu and pages_attn.cu.  Included at the end of apk_b200.cu.
#include "pages.cuh"

#include <algorithm>
#include <cmath>

static_assert(APK_TY_F32 == PTY_F32 && APK_TY_F16 == PTY_F16 && APK_TY_BF16 == PTY_BF16, "type ids");
static_assert(APK_PAGES_MAX_LIST == PAGES_MAX_LIST && APK_PAGES_MAX_BATCH == PAGES_MAX_BATCH, "list lengths");

namespace {

// The caller's current device comes back when the call ends: these entry points work on the caller's own buffers
// and streams, beside the caller's other CUDA code.
struct DeviceScope {
    int old = -1;
    cudaError_t enter(int device) {
        cudaError_t e = cudaGetDevice(&old);
        if (e == cudaSuccess && old != device) e = cudaSetDevice(device);
        else old = -1;
        return e;
    }
    ~DeviceScope() {
        if (old >= 0) cudaSetDevice(old);
    }
};

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int pages_view(const char *what, const apk_pages *p, PagesDev *d) {
    if (!p || !p->k || !p->v || !p->table || !p->lens || !p->refs || !p->work)
        return fail(APK_ERR_INVALID_ARG, "%s: null pool or buffer", what);
    if (p->ty != APK_TY_F16 && p->ty != APK_TY_BF16)
        return fail(APK_DECLINE_UNSUPPORTED_TYPE, "%s: a pool of type %u (f16 and bf16 are supported)", what, p->ty);
    if (p->n_layers == 0 || p->n_pages == 0 || p->n_seqs == 0 || p->width == 0 || p->n_kv_heads == 0)
        return fail(APK_ERR_INVALID_ARG, "%s: an empty pool", what);
    if (p->page < 8 || p->page > 256 || (p->page & (p->page - 1)))
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: pages of %u positions (a power of two from 8 to 256 is supported)", what, p->page);
    if (p->head_dim == 0 || p->head_dim % 8 || p->head_dim > 256)
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: heads of %u dimensions (a multiple of 8 up to 256 is supported)", what, p->head_dim);
    const uint32_t big = 1u << 28;
    if (p->n_pages >= big || p->n_seqs >= big || p->n_layers > 65535 || p->n_kv_heads > 65535 ||
        (uint64_t)p->width * p->page >= (1u << 30) || p->table_stride < p->width)
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: %u pages, %u sequences of %u pages in rows of %llu", what, p->n_pages, p->n_seqs,
                    p->width, (unsigned long long)p->table_stride);
    if (!aligned16(p->k) || !aligned16(p->v)) return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: pages that do not start on 16 bytes", what);
    for (int i = 0; i < 4; ++i) {
        if (p->k_stride[i] % 8 || p->v_stride[i] % 8 || p->k_stride[i] >= (1ull << 38) || p->v_stride[i] >= (1ull << 38))
            return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: strides of the pages are multiples of 8 elements", what);
        d->ks[i] = (long long)p->k_stride[i];
        d->vs[i] = (long long)p->v_stride[i];
    }
    d->k = (uint16_t *)p->k;
    d->v = (uint16_t *)p->v;
    d->table = p->table;
    d->table_stride = (long long)p->table_stride;
    d->lens = p->lens;
    d->refs = p->refs;
    d->work = p->work;
    d->n_seqs = (int)p->n_seqs;
    d->width = (int)p->width;
    d->n_layers = (int)p->n_layers;
    d->n_pages = (int)p->n_pages;
    d->page = (int)p->page;
    d->shift = 0;
    while ((1 << d->shift) < d->page) ++d->shift;
    d->kv = (int)p->n_kv_heads;
    d->dim = (int)p->head_dim;
    d->bf16 = p->ty == APK_TY_BF16;
    return APK_OK;
}

int pages_batch(const char *what, const int32_t *cu, const int32_t *seqs, uint32_t n, uint32_t n_rows, BatchDev *b) {
    if (!cu) return fail(APK_ERR_INVALID_ARG, "%s: null row offsets", what);
    if (n > APK_PAGES_MAX_BATCH || n_rows >= (1u << 28))
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: %u rows of %u sequences (at most %u sequences)", what, n_rows, n, APK_PAGES_MAX_BATCH);
    b->cu = cu;
    b->seqs = seqs;
    b->n = (int)n;
    b->rows = (int)n_rows;
    return APK_OK;
}

// Rows of heads: 16-byte aligned start, strides that keep it.
int check_rows(const char *what, const char *name, const void *p, uint32_t ty, const uint64_t stride[2]) {
    const uint64_t unit = ty == APK_TY_F32 ? 4 : 8;
    if (ty != APK_TY_F32 && ty != APK_TY_F16 && ty != APK_TY_BF16)
        return fail(APK_DECLINE_UNSUPPORTED_TYPE, "%s: %s of type %u (f32, f16 and bf16 are supported)", what, name, ty);
    if (!aligned16(p) || stride[0] % unit || stride[1] % unit || stride[0] >= (1ull << 38) || stride[1] >= (1ull << 38))
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: rows of %s do not start on 16 bytes", what, name);
    return APK_OK;
}

int pages_list(const char *what, const apk_pages *p, uint32_t n, const int32_t *a, const int32_t *b, SlotList *l) {
    if (n && (!a || !b)) return fail(APK_ERR_INVALID_ARG, "%s: null list", what);
    if (n > APK_PAGES_MAX_LIST)
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: %u sequences in one call (at most %u)", what, n, APK_PAGES_MAX_LIST);
    for (uint32_t i = 0; i < n; ++i) {
        if (a[i] < 0 || (uint32_t)a[i] >= p->n_seqs)
            return fail(APK_ERR_INVALID_ARG, "%s: sequence %d of %u", what, a[i], p->n_seqs);
        l->a[i] = a[i];
        l->b[i] = b[i];
    }
    l->n = (int)n;
    return APK_OK;
}

// A list that names a sequence twice has no order that its kernel could keep.  `sorted` receives the n <= PAGES_MAX_LIST
// entries in order (compared pair by pair, a fork of 1024 took half a millisecond).
int pages_distinct(const char *what, const int32_t *a, uint32_t n, int32_t *sorted) {
    std::copy(a, a + n, sorted);
    std::sort(sorted, sorted + n);
    const int32_t *twice = std::adjacent_find(sorted, sorted + n);
    return twice == sorted + n ? APK_OK : fail(APK_ERR_INVALID_ARG, "%s: sequence %d is named twice", what, *twice);
}

// What a waited call reports: the words of work[] after its kernels.  A reservation reports an expired wait only where it has
// changed nothing on that account: its caller repeats what ends in an error.
int pages_wait(const char *what, const PagesDev &P, cudaStream_t st, bool reserve) {
    int w[2] = {0, 0};
    CUDA_TRY(cudaMemcpyAsync(w, P.work, sizeof w, cudaMemcpyDeviceToHost, st));
    CUDA_TRY(cudaStreamSynchronize(st));
    if (reserve ? w[PW_SHORT] == PW_UNTRIED : w[PW_ERR] != 0) {
        CUDA_TRY(cudaMemsetAsync(P.work + PW_ERR, 0, sizeof(int), st));
        CUDA_TRY(cudaStreamSynchronize(st));
        return fail(APK_ERR_TIMEOUT, "%s: device-side wait expired (site %d)", what, w[PW_ERR]);
    }
    if (reserve && w[PW_SHORT] < 0) return fail(APK_DECLINE_INVALID_STATE, "%s: a sequence would outgrow its row of the page table", what);
    if (reserve && w[PW_SHORT] > 0) return fail(APK_DECLINE_INVALID_STATE, "%s: the pool is %d pages short", what, w[PW_SHORT]);
    return APK_OK;
}

int pages_done(apk_ctx *c, cudaError_t e, int launches, const char *what) {
    if (e != cudaSuccess) return fail(APK_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    std::lock_guard<std::mutex> g(c->mu);
    c->st.launches += (uint64_t)launches;
    c->st.calls++;
    return APK_OK;
}

// Radians a position of every rotated pair, and the factor on sine and cosine (apk_rope in the header).
int rope_frequencies(const char *what, const apk_rope *r, uint32_t dim, RopeParams *p) {
    const double two_pi = 6.283185307179586476925286766559;
    p->rot = 0;
    p->mag = 1.f;
    if (!r || r->rot_dim == 0) return APK_OK;
    if (r->rot_dim % 2 || r->rot_dim > dim)
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: %u of %u dimensions rotated (an even number is supported)", what, r->rot_dim, dim);
    if (r->layout > APK_ROPE_PAIRS || r->scaling > APK_ROPE_YARN) return fail(APK_ERR_INVALID_ARG, "%s: layout %u, scaling %u", what, r->layout, r->scaling);
    const bool yarn = r->scaling == APK_ROPE_YARN;
    if (!(r->base > 1.f) || !std::isfinite(r->base) || (r->scaling && (!(r->factor > 0.f) || !std::isfinite(r->factor))) ||
        (yarn && (r->orig_ctx == 0 || !(r->beta_fast > 0.f) || !(r->beta_slow > 0.f))))
        return fail(APK_ERR_INVALID_ARG, "%s: base %g, factor %g, context %u", what, r->base, r->factor, r->orig_ctx);
    const int half = (int)r->rot_dim / 2;
    const double rot = r->rot_dim, base = r->base, factor = r->scaling ? r->factor : 1.0;
    double lo = 0, hi = 0, mag = r->attn_factor;
    if (yarn) {
        // the pair that turns b times over the original context
        auto pair = [&](double b) { return rot * std::log(r->orig_ctx / (b * two_pi)) / (2.0 * std::log(base)); };
        lo = std::max(std::floor(pair(r->beta_fast)), 0.0);
        hi = std::min(std::ceil(pair(r->beta_slow)), rot - 1.0);
        if (factor > 1.0) mag *= 0.1 * std::log(factor) + 1.0;
    }
    // one power, then products: 128 of them are off by 2^-46 at most, 1e-8 of a turn at position 2^20
    const double ratio = std::pow(base, -2.0 / rot);
    double power = 1.0;
    for (int i = 0; i < half; ++i, power *= ratio) {
        double f = power;
        if (r->freq_factors) {
            if (!(r->freq_factors[i] > 0.f)) return fail(APK_ERR_INVALID_ARG, "%s: frequency factor %d is %g", what, i, r->freq_factors[i]);
            f /= r->freq_factors[i];
        }
        if (yarn) {
            const double ramp = std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 1e-3)));
            f = f / factor * ramp + f * (1.0 - ramp);
        } else {
            f /= factor;
        }
        p->turn[i] = f / two_pi;
    }
    p->rot = (int)r->rot_dim;
    p->pairs = r->layout == APK_ROPE_PAIRS;
    p->mag = (float)mag;
    return APK_OK;
}

}  // namespace

extern "C" {

int apk_rope_append(apk_ctx *c, const apk_rope_req *r, void *stream, int wait) {
    const char *what = "rope_append";
    if (!c || !r) return fail(APK_ERR_INVALID_ARG, "%s: null argument", what);
    RopeParams p{};
    APK_TRY(pages_view(what, r->pages, &p.P));
    APK_TRY(pages_batch(what, r->cu, r->seqs, r->n, r->n_rows, &p.B));
    const bool none = r->n == 0 || r->n_rows == 0;   // (rows that are not there may have no address)
    if (!none && (!r->k || !r->v || (r->q && !r->out))) return fail(APK_ERR_INVALID_ARG, "%s: null rows", what);
    if (r->layer >= r->pages->n_layers) return fail(APK_ERR_INVALID_ARG, "%s: layer %u of %u", what, r->layer, r->pages->n_layers);
    APK_TRY(check_rows(what, "k", r->k, r->ty, r->k_stride));
    APK_TRY(check_rows(what, "v", r->v, r->ty, r->v_stride));
    if (r->q) {
        if (r->n_heads == 0 || r->n_heads > 65535) return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: %u heads", what, r->n_heads);
        APK_TRY(check_rows(what, "q", r->q, r->ty, r->q_stride));
        APK_TRY(check_rows(what, "out", r->out, r->out_ty, r->out_stride));
        if (!none && r->out == r->q && (r->out_ty != r->ty || r->out_stride[0] != r->q_stride[0] || r->out_stride[1] != r->q_stride[1]))
            return fail(APK_ERR_INVALID_ARG, "%s: out in place of q has its type and strides", what);
    }
    if ((r->q_norm || r->k_norm) && !(r->eps >= 0.f)) return fail(APK_ERR_INVALID_ARG, "%s: eps %g", what, r->eps);
    APK_TRY(rope_frequencies(what, r->rope, r->pages->head_dim, &p));
    p.layer = (int)r->layer;
    p.q = r->q; p.k = r->k; p.v = r->v; p.out = r->out;
    p.ty = (int)r->ty;
    p.out_ty = (int)r->out_ty;
    p.heads = r->q ? (int)r->n_heads : 0;
    for (int i = 0; i < 2; ++i) {
        p.qs[i] = (long long)r->q_stride[i]; p.ks[i] = (long long)r->k_stride[i];
        p.vs[i] = (long long)r->v_stride[i]; p.os[i] = (long long)r->out_stride[i];
    }
    p.positions = r->positions;
    p.q_norm = r->q_norm;
    p.k_norm = r->k_norm;
    p.eps = r->eps;
    if (none) return APK_OK;
    DeviceScope dev;
    CUDA_TRY(dev.enter(c->device));
    int launches = 0;
    const cudaError_t e = launch_rope_append(p, c->n_sm, (cudaStream_t)stream, &launches);
    APK_TRY(pages_done(c, e, launches, what));
    // (it has no waits of its own to report, and one in place may not be repeated)
    if (wait) CUDA_TRY(cudaStreamSynchronize((cudaStream_t)stream));
    return APK_OK;
}

}  // extern "C"

namespace {

int attend_view(const apk_attend_req *r, AttendParams *q) {
    const char *what = "attend_pages";
    AttendParams &p = *q;
    APK_TRY(pages_view(what, r->pages, &p.P));
    APK_TRY(pages_batch(what, r->cu, r->seqs, r->n, r->n_rows, &p.B));
    const bool none = r->n == 0 || r->n_rows == 0;   // (rows that are not there may have no address)
    if (!none && (!r->q || !r->out)) return fail(APK_ERR_INVALID_ARG, "%s: null rows", what);
    if (r->layer >= r->pages->n_layers) return fail(APK_ERR_INVALID_ARG, "%s: layer %u of %u", what, r->layer, r->pages->n_layers);
    APK_TRY(check_rows(what, "q", r->q, r->ty, r->q_stride));
    APK_TRY(check_rows(what, "out", r->out, r->ty, r->out_stride));
    if (r->ty != r->pages->ty && !(r->ty == APK_TY_F32 && r->pages->ty == APK_TY_F16))
        return fail(APK_DECLINE_UNSUPPORTED_TYPE, "%s: rows of type %u over pages of type %u (the pages' type, or f32 over f16)", what, r->ty, r->pages->ty);
    if (r->pages->head_dim != 64 && r->pages->head_dim != 128)
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: heads of %u dimensions (64 and 128 are supported)", what, r->pages->head_dim);
    if (!none && r->out == r->q) return fail(APK_ERR_INVALID_ARG, "%s: out in place of q", what);
    const uint32_t kv = r->pages->n_kv_heads;
    if (r->n_heads == 0 || r->n_heads % kv || r->n_heads / kv > 64)
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: %u heads over %u kv heads (whole groups of at most 64)", what, r->n_heads, kv);
    p.scale_log2 = r->scale * 1.44269504088896340736f;
    if (!std::isfinite(p.scale_log2)) return fail(APK_ERR_INVALID_ARG, "%s: scale %g", what, r->scale);
    if (r->window >= (1u << 30)) return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: a window of %u", what, r->window);
    p.layer = (int)r->layer;
    p.q = r->q; p.out = r->out;
    p.ty = (int)r->ty;
    for (int i = 0; i < 2; ++i) { p.qs[i] = (long long)r->q_stride[i]; p.os[i] = (long long)r->out_stride[i]; }
    p.heads = (int)r->n_heads;
    p.group = (int)(r->n_heads / kv);
    p.causal = r->causal != 0;
    p.window = (int)r->window;
    // the kernels count (kv head, tile of rows, 128 positions) in 32 bits
    const uint64_t tiles = (uint64_t)r->n_rows / (128u / (uint32_t)p.group) + r->n;
    if (tiles * (2 * ((uint64_t)r->pages->width * r->pages->page / 128 + 1) + 8) * kv >= (1ull << 30))
        return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: %u rows of %u sequences over tables of %u pages are too much for one call", what, r->n_rows, r->n, r->pages->width);
    return APK_OK;
}

}  // namespace

extern "C" {

size_t apk_attend_pages_ws(apk_ctx *c, const apk_attend_req *r) {
    AttendParams p{};
    if (!c || !r || attend_view(r, &p) != APK_OK) return 0;
    return attend_ws_bytes(p, c->n_sm);
}

int apk_attend_pages(apk_ctx *c, const apk_attend_req *r, void *stream, int wait) {
    const char *what = "attend_pages";
    if (!c || !r) return fail(APK_ERR_INVALID_ARG, "%s: null argument", what);
    AttendParams p{};
    APK_TRY(attend_view(r, &p));
    if (r->n == 0 || r->n_rows == 0) return APK_OK;
    const size_t need = attend_ws_bytes(p, c->n_sm);
    if (need && (!r->ws || r->ws_bytes < need || ((uintptr_t)r->ws & 255)))
        return fail(APK_ERR_INVALID_ARG, "%s: a workspace of %zu bytes (%zu are needed, 256-byte aligned)", what, r->ws ? r->ws_bytes : (size_t)0, need);
    DeviceScope dev;
    CUDA_TRY(dev.enter(c->device));
    int launches = 0;
    const cudaError_t e = launch_attend(p, c->n_sm, r->ws, c->wait_limit, (cudaStream_t)stream, &launches);
    if (e == cudaErrorNotSupported) return fail(APK_DECLINE_UNSUPPORTED_SHAPE, "%s: strides of the pages that a tensor map cannot express", what);
    APK_TRY(pages_done(c, e, launches, what));
    return wait ? pages_wait(what, p.P, (cudaStream_t)stream, false) : APK_OK;
}

int apk_pages_reserve(apk_ctx *c, const apk_pages *pages, uint32_t n, const int32_t *seqs, const int32_t *n_new, void *stream, int wait) {
    const char *what = "pages_reserve";
    if (!c) return fail(APK_ERR_INVALID_ARG, "%s: null argument", what);
    PagesDev P{};
    SlotList l;
    APK_TRY(pages_view(what, pages, &P));
    APK_TRY(pages_list(what, pages, n, seqs, n_new, &l));
    int32_t sorted[PAGES_MAX_LIST];
    APK_TRY(pages_distinct(what, seqs, n, sorted));
    for (uint32_t i = 0; i < n; ++i)
        if (n_new[i] < 0) return fail(APK_ERR_INVALID_ARG, "%s: %d new positions", what, n_new[i]);
    DeviceScope dev;
    CUDA_TRY(dev.enter(c->device));
    int launches = 0;
    const cudaError_t e = launch_pages_reserve(P, l, wait != 0, c->n_sm, (cudaStream_t)stream, &launches);
    APK_TRY(pages_done(c, e, launches, what));
    return wait ? pages_wait(what, P, (cudaStream_t)stream, true) : APK_OK;
}

int apk_pages_fork(apk_ctx *c, const apk_pages *pages, uint32_t n, const int32_t *src, const int32_t *dst, void *stream) {
    const char *what = "pages_fork";
    if (!c) return fail(APK_ERR_INVALID_ARG, "%s: null argument", what);
    PagesDev P{};
    SlotList l;
    APK_TRY(pages_view(what, pages, &P));
    APK_TRY(pages_list(what, pages, n, dst, src, &l));
    APK_TRY(pages_list(what, pages, n, src, dst, &l));
    int32_t sorted[PAGES_MAX_LIST];
    APK_TRY(pages_distinct(what, dst, n, sorted));
    for (uint32_t i = 0; i < n; ++i)
        if (std::binary_search(sorted, sorted + n, src[i])) return fail(APK_ERR_INVALID_ARG, "%s: sequence %d is both forked and written", what, src[i]);
    if (n == 0) return APK_OK;
    DeviceScope dev;
    CUDA_TRY(dev.enter(c->device));
    int launches = 0;
    const cudaError_t e = launch_pages_fork(P, l, (cudaStream_t)stream, &launches);
    return pages_done(c, e, launches, what);
}

int apk_pages_release(apk_ctx *c, const apk_pages *pages, uint32_t n, const int32_t *seqs, const int32_t *keep, void *stream) {
    const char *what = "pages_release";
    if (!c) return fail(APK_ERR_INVALID_ARG, "%s: null argument", what);
    PagesDev P{};
    SlotList l;
    APK_TRY(pages_view(what, pages, &P));
    APK_TRY(pages_list(what, pages, n, seqs, keep, &l));
    int32_t sorted[PAGES_MAX_LIST];
    APK_TRY(pages_distinct(what, seqs, n, sorted));
    for (uint32_t i = 0; i < n; ++i)
        if (keep[i] < 0) return fail(APK_ERR_INVALID_ARG, "%s: %d positions kept", what, keep[i]);
    if (n == 0) return APK_OK;
    DeviceScope dev;
    CUDA_TRY(dev.enter(c->device));
    int launches = 0;
    const cudaError_t e = launch_pages_release(P, l, (cudaStream_t)stream, &launches);
    return pages_done(c, e, launches, what);
}

int apk_pages_compact(apk_ctx *c, const apk_pages *pages, int32_t *page_map, void *stream) {
    const char *what = "pages_compact";
    if (!c) return fail(APK_ERR_INVALID_ARG, "%s: null argument", what);
    PagesDev P{};
    APK_TRY(pages_view(what, pages, &P));
    DeviceScope dev;
    CUDA_TRY(dev.enter(c->device));
    int launches = 0;
    const cudaError_t e = launch_pages_compact(P, page_map, c->n_sm, (cudaStream_t)stream, &launches);
    return pages_done(c, e, launches, what);
}

}  // extern "C"
