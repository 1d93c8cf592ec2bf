// Kernels that write the paged KV cache: rotary positions with the store into pages, and the pages' upkeep.
#include "pages.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace apk {
namespace {

template <int TY> struct Elem;
template <> struct Elem<PTY_F32> { typedef float T; };
template <> struct Elem<PTY_F16> { typedef __half T; };
template <> struct Elem<PTY_BF16> { typedef __nv_bfloat16 T; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// One rounding to nearest even, at the store.
__device__ __forceinline__ void put(void *p, long long i, int ty, float x) {
    if (ty == PTY_F32) ((float *)p)[i] = x;
    else if (ty == PTY_F16) ((__half *)p)[i] = __float2half_rn(x);
    else ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(x);
}

// ---------------------------------------------------------------------------------------------- rope_append

// One block per row of the batch.  Angles: position * turns(pair) in 64 bits, whole turns taken off, then sine and
// cosine of the rest in 32 bits: at a position of 2^20 a 32-bit product would already be 2^-4 radians off.
template <int TY>
__global__ void __launch_bounds__(256) rope_append_kernel(const __grid_constant__ RopeParams p) {
    typedef typename Elem<TY>::T T;
    __shared__ float2 cs[128];
    const int t = blockIdx.x;
    const int i = batch_find(p.B, t);
    if (i < 0) return;
    const SeqRows s = batch_seq(p.P, p.B, i);
    const int pos = s.len - s.rows + (t - s.first);
    const int rp = p.positions ? p.positions[t] : pos;
    for (int j = threadIdx.x; j < p.rot / 2; j += blockDim.x) {
        const double a = (double)rp * p.turn[j];
        float sn, cn;
        sincospif((float)(2.0 * (a - rint(a))), &sn, &cn);
        cs[j] = make_float2(cn * p.mag, sn * p.mag);
    }
    __syncthreads();
    const int page = pos >= 0 && pos < s.len ? page_of(p.P, s.slot, pos) : -1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.P.dim;
    const int n_rows = p.heads + 2 * p.P.kv;
    for (int r = warp; r < n_rows; r += 8) {
        const int kind = r < p.heads ? 0 : (r < p.heads + p.P.kv ? 1 : 2);
        const int h = kind == 0 ? r : (kind == 1 ? r - p.heads : r - p.heads - p.P.kv);
        if (kind && page < 0) continue;
        const T *src;
        void *dst;
        long long at;
        int ty;
        const int slot_in = pos & (p.P.page - 1);
        if (kind == 0) {
            if (!p.q) continue;
            src = (const T *)p.q + t * p.qs[0] + h * p.qs[1];
            dst = p.out; at = t * p.os[0] + h * p.os[1]; ty = p.out_ty;
        } else if (kind == 1) {
            src = (const T *)p.k + t * p.ks[0] + h * p.ks[1];
            dst = p.P.k; at = p.layer * p.P.ks[0] + page * p.P.ks[1] + slot_in * p.P.ks[2] + h * p.P.ks[3];
            ty = p.P.bf16 ? PTY_BF16 : PTY_F16;
        } else {
            src = (const T *)p.v + t * p.vs[0] + h * p.vs[1];
            dst = p.P.v; at = p.layer * p.P.vs[0] + page * p.P.vs[1] + slot_in * p.P.vs[2] + h * p.P.vs[3];
            ty = p.P.bf16 ? PTY_BF16 : PTY_F16;
        }
        if (kind == 2) {
            for (int d = lane; d < D; d += 32) put(dst, at + d, ty, to_f32(src[d]));
            continue;
        }
        const float *w = kind == 0 ? p.q_norm : p.k_norm;
        float rs = 1.f;
        if (w) {
            float ss = 0.f;
            for (int d = lane; d < D; d += 32) { const float x = to_f32(src[d]); ss += x * x; }
            for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
            rs = rsqrtf(ss / (float)D + p.eps);
        }
        const int half = p.rot / 2;
        for (int j = lane; j < half; j += 32) {
            const int da = p.pairs ? 2 * j : j, db = p.pairs ? 2 * j + 1 : j + half;
            float a = to_f32(src[da]), b = to_f32(src[db]);
            if (w) { a = a * rs * w[da]; b = b * rs * w[db]; }
            put(dst, at + da, ty, a * cs[j].x - b * cs[j].y);
            put(dst, at + db, ty, b * cs[j].x + a * cs[j].y);
        }
        for (int d = p.rot + lane; d < D; d += 32) {
            float x = to_f32(src[d]);
            if (w) x = x * rs * w[d];
            put(dst, at + d, ty, x);
        }
    }
}

// ------------------------------------------------------------------------------------------- the pages' upkeep

__device__ __forceinline__ int pages_for(const PagesDev &P, long long len) { return (int)((len + P.page - 1) >> P.shift); }

// Sums of refs[] are the same in whatever order the blocks come: integers.
__device__ __forceinline__ void drop_pages(const PagesDev &P, int slot, int from, int to) {
    const int *row = P.table + (long long)slot * P.table_stride;
    for (int c = from + threadIdx.x; c < to; c += blockDim.x) {
        const int pg = row[c];
        if ((unsigned)pg < (unsigned)P.n_pages) atomicSub(&P.refs[pg], 1);
    }
}

// dst takes over src's pages and length in place of what it held: one block per pair.  The host has checked that no
// slot is named twice as a destination and none is a source too.
__global__ void __launch_bounds__(256) pages_fork_kernel(const __grid_constant__ PagesDev P, const __grid_constant__ SlotList l) {
    const int src = l.a[blockIdx.x], dst = l.b[blockIdx.x];
    const int len = pages_len(P, src), n = pages_for(P, len);
    drop_pages(P, dst, 0, pages_for(P, pages_len(P, dst)));
    __syncthreads();
    const int *from = P.table + (long long)src * P.table_stride;
    int *to = P.table + (long long)dst * P.table_stride;
    for (int c = threadIdx.x; c < n; c += blockDim.x) {
        const int pg = from[c];
        to[c] = pg;
        if ((unsigned)pg < (unsigned)P.n_pages) atomicAdd(&P.refs[pg], 1);
    }
    if (threadIdx.x == 0) P.lens[dst] = len;
}

// The sequence keeps its first b positions; the pages behind them lose a holder.
__global__ void __launch_bounds__(256) pages_release_kernel(const __grid_constant__ PagesDev P, const __grid_constant__ SlotList l) {
    const int slot = l.a[blockIdx.x];
    const int len = pages_len(P, slot), keep = min(len, l.b[blockIdx.x]);
    drop_pages(P, slot, pages_for(P, keep), pages_for(P, len));
    __syncthreads();
    if (threadIdx.x == 0) P.lens[slot] = keep;
}

// Inclusive sum over the 1024 threads of a block.
__device__ __forceinline__ int block_scan(int x, int *sh /*32*/) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = sh[lane];
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(~0u, w, o);
            if (lane >= o) w += y;
        }
        sh[lane] = w;
    }
    __syncthreads();
    return x + (warp ? sh[warp - 1] : 0);
}

// Room for b more positions in each listed sequence: thread i looks after entry i.  A sequence that is about to write
// into a last page which others hold too gets a copy of it; in the order of the list, so the last of several holders
// keeps the original.  All or nothing: with too few pages nothing changes and work[PW_SHORT] says how many are missing.
__global__ void __launch_bounds__(PAGES_MAX_LIST) pages_reserve_kernel(const __grid_constant__ PagesDev P, const __grid_constant__ SlotList l) {
    __shared__ int sh[32], last_of[PAGES_MAX_LIST], first_of[PAGES_MAX_LIST], n_copies, too_long;
    const int i = threadIdx.x;
    int *const list = P.work + PW_LIST;
    int *const fresh = list + 4 * P.n_seqs;
    if (i == 0) n_copies = too_long = 0;
    int slot = 0, old = 0, have = 0, want = 0, last = -1;
    if (i < l.n) {
        slot = l.a[i];
        old = pages_len(P, slot);
        have = pages_for(P, old);
        const long long len = (long long)old + l.b[i];
        want = len > ((long long)P.width << P.shift) ? P.width + 1 : pages_for(P, len);
        if ((old & (P.page - 1)) && l.b[i] > 0) last = page_of(P, slot, old - 1);
    }
    last_of[i] = last;
    __syncthreads();
    if (want > P.width) too_long = 1;
    int copy = 0;
    if (last >= 0 && P.refs[last] > 1) {
        int before = 0;
        for (int j = 0; j < i; ++j) before += last_of[j] == last;
        copy = P.refs[last] - before > 1;
    }
    const int need = i < l.n ? want - have + copy : 0;
    const int end = block_scan(need, sh);
    const int total = sh[31];
    first_of[i] = end - need;
    __syncthreads();
    if (too_long) {
        if (i == 0) { P.work[PW_SHORT] = -1; P.work[PW_COPIES] = 0; }
        return;
    }
    // the `total` lowest free pages, in order
    int got = 0;
    for (int base = 0; base < P.n_pages && got < total; base += PAGES_MAX_LIST) {
        const int pg = base + i, is_free = pg < P.n_pages && P.refs[pg] == 0;
        const int at = got + block_scan(is_free, sh);
        if (is_free && at <= total) fresh[at - 1] = pg;
        got += sh[31];
        __syncthreads();
    }
    if (got < total) {
        if (i == 0) { P.work[PW_SHORT] = total - got; P.work[PW_COPIES] = 0; }
        return;
    }
    __syncthreads();
    if (i < l.n) {
        int *row = P.table + (long long)slot * P.table_stride;
        int at = first_of[i];
        if (copy) {
            const int pg = fresh[at++];
            row[have - 1] = pg;
            P.refs[pg] = 1;
            atomicSub(&P.refs[last], 1);
            int *e = list + 4 * atomicAdd(&n_copies, 1);  // (the copies are independent of one another: any order)
            e[0] = last; e[1] = pg; e[2] = old & (P.page - 1);
        }
        for (int c = have; c < want; ++c) {
            const int pg = fresh[at++];
            row[c] = pg;
            P.refs[pg] = 1;
        }
        P.lens[slot] = old + l.b[i];
    }
    __syncthreads();
    if (i == 0) { P.work[PW_SHORT] = 0; P.work[PW_COPIES] = n_copies; }
}

// The copy list, in every layer, K and V: 16 bytes a thread and turn.
__device__ __forceinline__ void copy_pages(const PagesDev &P, const int *list, int n, int block, int blocks) {
    const int vecs = P.dim / 8;
    for (int u = block; u < n * P.n_layers * 2; u += blocks) {
        const int e = u / (P.n_layers * 2), lk = u % (P.n_layers * 2), layer = lk >> 1;
        const int src = list[4 * e], dst = list[4 * e + 1], tok = list[4 * e + 2];
        const long long *st = lk & 1 ? P.vs : P.ks;
        uint16_t *base = (lk & 1 ? P.v : P.k) + layer * st[0];
        const int total = tok * P.kv * vecs;
        for (int x = threadIdx.x; x < total; x += blockDim.x) {
            const int d = x % vecs, y = x / vecs, h = y % P.kv, t = y / P.kv;
            const long long off = t * st[2] + h * st[3] + d * 8;
            *(uint4 *)(base + dst * st[1] + off) = *(const uint4 *)(base + src * st[1] + off);
        }
    }
}

__global__ void __launch_bounds__(256) pages_copy_kernel(const __grid_constant__ PagesDev P) {
    copy_pages(P, P.work + PW_LIST, min(P.work[PW_COPIES], P.n_seqs), blockIdx.x, gridDim.x);
}

// Where every page goes: live pages whose number is not below the number of live pages move into the free pages
// below it, both in ascending order.  map = new number, -1 for a free page.  One block.
__global__ void __launch_bounds__(1024) pages_plan_kernel(const __grid_constant__ PagesDev P, int *map) {
    __shared__ int sh[32];
    const int i = threadIdx.x;
    int live = 0;
    for (int pg = i; pg < P.n_pages; pg += 1024) live += P.refs[pg] > 0;
    block_scan(live, sh);
    const int count = sh[31];
    int *const holes = P.work + PW_LIST + 4 * P.n_seqs, *const movers = holes + P.n_pages;
    int nh = 0, nm = 0;
    for (int base = 0; base < P.n_pages; base += 1024) {
        const int pg = base + i, in = pg < P.n_pages, lv = in && P.refs[pg] > 0;
        const int hole = in && !lv && pg < count, mover = lv && pg >= count;
        const int h = nh + block_scan(hole, sh);
        nh += sh[31];
        const int m = nm + block_scan(mover, sh);
        nm += sh[31];
        if (hole) holes[h - 1] = pg;
        if (mover) movers[m - 1] = pg;
        if (in) map[pg] = lv ? pg : -1;
        __syncthreads();
    }
    // as many holes as movers: both are the live pages' share of the upper part
    for (int e = i; e < nm; e += 1024) {
        const int from = movers[e], to = holes[e];
        map[from] = to;
        P.refs[to] = P.refs[from];
        P.refs[from] = 0;
    }
    if (i == 0) P.work[PW_COPIES] = nm;
}

__global__ void __launch_bounds__(256) pages_move_kernel(const __grid_constant__ PagesDev P, const int *map) {
    const int *holes = P.work + PW_LIST + 4 * P.n_seqs, *movers = holes + P.n_pages;
    for (int s = blockIdx.x; s < P.n_seqs; s += gridDim.x) {
        int *row = P.table + (long long)s * P.table_stride;
        const int n = pages_for(P, pages_len(P, s));
        for (int c = threadIdx.x; c < n; c += blockDim.x) {
            const int pg = row[c];
            if ((unsigned)pg < (unsigned)P.n_pages && map[pg] >= 0) row[c] = map[pg];
        }
    }
    const int n = P.work[PW_COPIES], vecs = P.dim / 8;
    for (int u = blockIdx.x; u < n * P.n_layers * 2; u += gridDim.x) {
        const int e = u / (P.n_layers * 2), lk = u % (P.n_layers * 2), layer = lk >> 1;
        const int src = movers[e], dst = holes[e];
        const long long *st = lk & 1 ? P.vs : P.ks;
        uint16_t *base = (lk & 1 ? P.v : P.k) + layer * st[0];
        const int total = P.page * P.kv * vecs;
        for (int x = threadIdx.x; x < total; x += blockDim.x) {
            const int d = x % vecs, y = x / vecs, h = y % P.kv, t = y / P.kv;
            const long long off = t * st[2] + h * st[3] + d * 8;
            *(uint4 *)(base + dst * st[1] + off) = *(const uint4 *)(base + src * st[1] + off);
        }
    }
}

}  // namespace

cudaError_t launch_rope_append(const RopeParams &p, int, cudaStream_t st, int *launches) {
    if (p.ty == PTY_F32) rope_append_kernel<PTY_F32><<<p.B.rows, 256, 0, st>>>(p);
    else if (p.ty == PTY_F16) rope_append_kernel<PTY_F16><<<p.B.rows, 256, 0, st>>>(p);
    else rope_append_kernel<PTY_BF16><<<p.B.rows, 256, 0, st>>>(p);
    *launches += 1;
    return cudaGetLastError();
}

cudaError_t launch_pages_fork(const PagesDev &P, const SlotList &l, cudaStream_t st, int *launches) {
    pages_fork_kernel<<<l.n, 256, 0, st>>>(P, l);
    *launches += 1;
    return cudaGetLastError();
}

cudaError_t launch_pages_release(const PagesDev &P, const SlotList &l, cudaStream_t st, int *launches) {
    pages_release_kernel<<<l.n, 256, 0, st>>>(P, l);
    *launches += 1;
    return cudaGetLastError();
}

cudaError_t launch_pages_reserve(const PagesDev &P, const SlotList &l, int n_sm, cudaStream_t st, int *launches) {
    pages_reserve_kernel<<<1, PAGES_MAX_LIST, 0, st>>>(P, l);
    *launches += 1;
    if (l.n) {
        pages_copy_kernel<<<(unsigned)std::min<long long>(4 * n_sm, (long long)l.n * P.n_layers * 2), 256, 0, st>>>(P);
        *launches += 1;
    }
    return cudaGetLastError();
}

cudaError_t launch_pages_compact(const PagesDev &P, int *page_map, int n_sm, cudaStream_t st, int *launches) {
    if (!page_map) page_map = P.work + PW_LIST + 4 * P.n_seqs + 2 * P.n_pages;
    pages_plan_kernel<<<1, 1024, 0, st>>>(P, page_map);
    pages_move_kernel<<<4 * n_sm, 256, 0, st>>>(P, page_map);
    *launches += 2;
    return cudaGetLastError();
}

}  // namespace apk
