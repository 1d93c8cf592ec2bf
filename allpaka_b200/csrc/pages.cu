// Kernels that write the paged KV cache: rotary positions with the store into pages, and the pages' upkeep.
#include "pages.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

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

// Where a row of the batch belongs: its position in its sequence and where that is stored (-1: nowhere; -2: the row is nobody's).
struct RopeAt { int pos, page; };
constexpr int ROPE_MOST = 8;   // rows that a block takes at a time

// The places and the sines and cosines of a block's rows, side by side: a warp looks for a row's sequence, 32 offsets at a time
// instead of a chain of loads.  Angles: position * turns(pair) in 64 bits, whole turns taken off, then sine and cosine of the rest
// in 32 bits: at a position of 2^20 a 32-bit product would already be 2^-4 radians off.  Pair j lies at cs[rope_slot(j)]: the
// threads of a head, which hold eight neighbouring pairs each, read 8-byte neighbours.
__device__ __forceinline__ int rope_slot(int j) { return (j & 7) * 16 + (j >> 3); }
__device__ __forceinline__ void rope_places(const RopeParams &p, int t0, int rows, RopeAt *at, int *turn_at, float2 *cs) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < rows) {
        const int t = t0 + warp;
        int before = 0;   // sequences that begin at row t or before
        for (int i0 = 0; i0 < p.B.n; i0 += 32) before += __popc(__ballot_sync(~0u, i0 + lane < p.B.n && p.B.cu[i0 + lane] <= t));
        RopeAt r = {0, -2};
        int rp = 0;
        if (before > 0 && t < p.B.cu[before]) {
            const SeqRows s = batch_seq(p.P, p.B, before - 1);
            r.pos = s.len - s.rows + (t - s.first);
            rp = p.positions ? p.positions[t] : r.pos;
            r.page = r.pos >= 0 && r.pos < s.len ? page_of(p.P, s.slot, r.pos) : -1;
        }
        if (lane == 0) { at[warp] = r; turn_at[warp] = rp; }
    }
    __syncthreads();
    const int half = p.rot / 2;
    for (int i = threadIdx.x; i < rows * half; i += 256) {
        const int row = i / half, j = i - row * half;
        const double a = (double)turn_at[row] * p.turn[j];
        float sn, cn;
        sincospif((float)(2.0 * (a - rint(a))), &sn, &cn);
        cs[row * 128 + rope_slot(j)] = make_float2(cn * p.mag, sn * p.mag);
    }
    __syncthreads();
}

__device__ __forceinline__ void rope_turn(float &a, float &b, float2 z) {
    const float x = a * z.x - b * z.y, y = b * z.x + a * z.y;
    a = x;
    b = y;
}

// Sixteen values of a row at two offsets, as they are stored, and as 32-bit values.
template <int TY> struct Raw16 { uint4 v[TY == PTY_F32 ? 4 : 2]; };
template <int TY>
__device__ __forceinline__ void load16(Raw16<TY> &x, const typename Elem<TY>::T *src, int o0, int o1) {
    if constexpr (TY == PTY_F32) {
        x.v[0] = __ldcs((const uint4 *)(src + o0)); x.v[1] = __ldcs((const uint4 *)(src + o0 + 4));
        x.v[2] = __ldcs((const uint4 *)(src + o1)); x.v[3] = __ldcs((const uint4 *)(src + o1 + 4));
    } else {
        x.v[0] = __ldcs((const uint4 *)(src + o0));
        x.v[1] = __ldcs((const uint4 *)(src + o1));
    }
}
template <int TY>
__device__ __forceinline__ void widen16(const Raw16<TY> &x, float *y) {
#pragma unroll
    for (int h = 0; h < (TY == PTY_F32 ? 4 : 2); ++h) {
        const uint32_t u[4] = {x.v[h].x, x.v[h].y, x.v[h].z, x.v[h].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (TY == PTY_F32) {
                y[4 * h + e] = __uint_as_float(u[e]);
            } else {
                float2 f;
                if constexpr (TY == PTY_F16) f = __half22float2(*(const __half2 *)&u[e]);
                else f = __bfloat1622float2(*(const __nv_bfloat162 *)&u[e]);
                y[8 * h + 2 * e] = f.x;
                y[8 * h + 2 * e + 1] = f.y;
            }
        }
    }
}
__device__ __forceinline__ void store8(void *p, long long at, int ty, const float *x) {
    if (ty == PTY_F32) {
        *(float4 *)((float *)p + at) = *(const float4 *)x;
        *(float4 *)((float *)p + at + 4) = *(const float4 *)(x + 4);
        return;
    }
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (ty == PTY_F16) { const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]); u[e] = *(const uint32_t *)&h; }
        else { const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]); u[e] = *(const uint32_t *)&h; }
    }
    *(uint4 *)((uint16_t *)p + at) = make_uint4(u[0], u[1], u[2], u[3]);
}

// Heads of 16 * LANES dimensions, rotated in whole groups of 16: LANES threads a head, 16 values each (8 pairs, or 16 that pass
// through), so that every access is 16 bytes wide.  Bound by the bytes; what stands in the way is latency: finding a row's place
// and its angles is a chain of four loads and 64-bit arithmetic, about 2 us, so a block takes eight rows of its share at a time,
// works their places out together, and has its first loads under way before it begins; three blocks share a multiprocessor.
// A warp stays with its row (rows that are fewer than warps get several each), so that what belongs to a row is worked out once:
// spread over the block instead, a prompt of 8192 rows took 90 us with a third of the instructions spent on addresses.
template <int TY, int LANES>
__global__ void __launch_bounds__(256, 3) rope_append_wide_kernel(const __grid_constant__ RopeParams p) {
    typedef typename Elem<TY>::T T;
    constexpr int AHEAD = TY == PTY_F32 ? 1 : 2, SIDE = 32 / LANES;   // loads of a group; heads that a warp works on side by side
    __shared__ float2 cs[ROPE_MOST * 128];
    __shared__ RopeAt place[ROPE_MOST];
    __shared__ int turn_at[ROPE_MOST];
    pages_let_next();
    pages_wait_front();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, u = lane % LANES, heads = p.heads + 2 * p.P.kv;
    const bool turned = u < p.rot / 16;
    const int o0 = turned && !p.pairs ? u * 8 : u * 16, o1 = turned && !p.pairs ? p.rot / 2 + u * 8 : u * 16 + 8;
    const int cache = p.P.bf16 ? PTY_BF16 : PTY_F16;
    const int end = (int)((long long)p.B.rows * (blockIdx.x + 1) / gridDim.x);
    for (int t0 = (int)((long long)p.B.rows * blockIdx.x / gridDim.x); t0 < end; t0 += ROPE_MOST) {
        const int rows = min(ROPE_MOST, end - t0);
        const int per_row = rows > 4 ? 1 : (rows > 2 ? 2 : (rows > 1 ? 4 : 8));   // warps a row
        const int row = warp / per_row, step = per_row * SIDE, first = (warp % per_row) * SIDE + lane / LANES;
        const long long t = t0 + min(row, rows - 1);
        const T *const q = (const T *)p.q + t * p.qs[0], *const k = (const T *)p.k + t * p.ks[0], *const v = (const T *)p.v + t * p.vs[0];
        Raw16<TY> ping[AHEAD], pong[AHEAD];   // one is on its way while the other is worked on
        auto load = [&](Raw16<TY> *raw, int r0) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int r = r0 + a * step + first;
                if (row >= rows || r >= heads) continue;
                load16<TY>(raw[a], r < p.heads ? q + r * p.qs[1] : (r < p.heads + p.P.kv ? k + (r - p.heads) * p.ks[1] : v + (r - p.heads - p.P.kv) * p.vs[1]), o0, o1);
            }
        };
        load(ping, 0);
        rope_places(p, t0, rows, place, turn_at, cs);
        const RopeAt at = place[min(row, rows - 1)];
        const bool mine = row < rows && at.page != -2;
        const long long in = at.pos & (p.P.page - 1), out_at = t * p.os[0];
        const long long k_at = p.layer * p.P.ks[0] + at.page * p.P.ks[1] + in * p.P.ks[2], v_at = p.layer * p.P.vs[0] + at.page * p.P.vs[1] + in * p.P.vs[2];
        const float2 *const z = cs + min(row, rows - 1) * 128 + u;
        auto work = [&](const Raw16<TY> *raw, int r0) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (r0 + a * step >= heads) break;   // (the whole warp)
                const int r = r0 + a * step + first;
                float y[16];
                widen16<TY>(raw[a], y);
                const int kind = r < p.heads ? 0 : (r < p.heads + p.P.kv ? 1 : 2);
                if (p.q_norm || p.k_norm) {
                    const float *w = kind == 0 ? p.q_norm : (kind == 1 ? p.k_norm : nullptr);
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 16; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
                    for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
                    if (w) {
                        const float rs = rsqrtf(ss / (float)p.P.dim + p.eps);
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const float4 g = __ldg((const float4 *)(w + (e < 8 ? o0 + e : o1 + e - 8)));
                            y[e] *= rs * g.x; y[e + 1] *= rs * g.y; y[e + 2] *= rs * g.z; y[e + 3] *= rs * g.w;
                        }
                    }
                }
                if (kind < 2 && turned) {
                    if (p.pairs) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) rope_turn(y[2 * e], y[2 * e + 1], z[16 * e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) rope_turn(y[e], y[8 + e], z[16 * e]);
                    }
                }
                if (!mine || r >= heads || (kind && at.page < 0)) continue;
                void *dst = p.out;
                long long to = out_at + r * p.os[1];
                if (kind == 1) { dst = p.P.k; to = k_at + (r - p.heads) * p.P.ks[3]; }
                if (kind == 2) { dst = p.P.v; to = v_at + (r - p.heads - p.P.kv) * p.P.vs[3]; }
                const int ty = kind ? cache : p.out_ty;
                store8(dst, to + o0, ty, y);
                store8(dst, to + o1, ty, y + 8);
            }
        };
        for (int r0 = 0; r0 < heads; r0 += 2 * AHEAD * step) {
            load(pong, r0 + AHEAD * step);
            work(ping, r0);
            load(ping, r0 + 2 * AHEAD * step);
            work(pong, r0 + AHEAD * step);
        }
        __syncthreads();   // (the places and angles are read until here)
    }
}

// Any other head: a warp per head, value by value.
template <int TY>
__global__ void __launch_bounds__(256) rope_append_kernel(const __grid_constant__ RopeParams p) {
    typedef typename Elem<TY>::T T;
    __shared__ float2 cs[128];
    __shared__ RopeAt place;
    __shared__ int turn_at;
    pages_let_next();
    pages_wait_front();
    const int t = blockIdx.x;
    rope_places(p, t, 1, &place, &turn_at, cs);
    const int pos = place.pos, page = place.page;
    if (page == -2) return;
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
            const float2 z = cs[rope_slot(j)];
            put(dst, at + da, ty, a * z.x - b * z.y);
            put(dst, at + db, ty, b * z.x + a * z.y);
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
    pages_let_next();
    pages_wait_front();
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
    pages_let_next();
    pages_wait_front();
    const int slot = l.a[blockIdx.x];
    const int len = pages_len(P, slot), keep = min(len, l.b[blockIdx.x]);
    drop_pages(P, slot, pages_for(P, keep), pages_for(P, len));
    __syncthreads();
    if (threadIdx.x == 0) P.lens[slot] = keep;
}

// Inclusive sum over the 1024 threads of a block.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T *sh /*32*/) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    if (warp == 0) {
        T w = sh[lane];
        for (int o = 1; o < 32; o <<= 1) {
            const T y = __shfl_up_sync(~0u, w, o);
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
// heed: with an expired wait of an earlier call to report, nothing changes either.
__global__ void __launch_bounds__(PAGES_MAX_LIST) pages_reserve_kernel(const __grid_constant__ PagesDev P, const __grid_constant__ SlotList l, int heed) {
    __shared__ int sh[32], last_of[PAGES_MAX_LIST], first_of[PAGES_MAX_LIST], n_copies, too_long;
    __shared__ long long needs[32];
    const int i = threadIdx.x;
    int *const list = P.work + PW_LIST;
    int *const fresh = list + 4 * P.n_seqs;
    pages_let_next();
    pages_wait_front();
    if (heed && P.work[PW_ERR]) {
        if (i == 0) { P.work[PW_SHORT] = PW_UNTRIED; P.work[PW_COPIES] = 0; }
        return;
    }
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
    const long long end = block_scan((long long)need, needs);   // (64 bits: 1024 sequences of up to 2^27 pages)
    const long long total = needs[31];
    first_of[i] = (int)(end - need);   // (used only where all of them are there)
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
        if (i == 0) { P.work[PW_SHORT] = (int)min(total - got, (long long)INT_MAX); P.work[PW_COPIES] = 0; }
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

// Copies of pages' positions in every layer, K and V.  A piece is 1024 16-byte vectors, four a thread, all asked for before the
// first is stored; pieces are dealt out over all blocks.  copy(e, src, dst, positions): what entry e is.
template <typename Copy>
__device__ __forceinline__ void copy_pages(const PagesDev &P, int n, const Copy &copy) {
    const int vecs = P.dim / 8, per_pos = P.kv * vecs, pieces = (P.page * per_pos + 1023) / 1024;
    const bool flat = P.ks[3] == P.dim && P.vs[3] == P.dim && P.ks[2] == (long long)P.kv * P.dim && P.vs[2] == (long long)P.kv * P.dim;
    for (long long u = blockIdx.x; u < (long long)n * P.n_layers * 2 * pieces; u += gridDim.x) {
        const int piece = (int)(u % pieces), lk = (int)(u / pieces) % (2 * P.n_layers), e = (int)(u / pieces) / (2 * P.n_layers);
        int src, dst, positions;
        copy(e, src, dst, positions);
        const int total = positions * per_pos;
        const long long *st = lk & 1 ? P.vs : P.ks;
        uint16_t *base = (lk & 1 ? P.v : P.k) + (lk >> 1) * st[0];
        const uint16_t *from = base + src * st[1];
        uint16_t *to = base + dst * st[1];
        uint4 v[4];
        long long off[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = piece * 1024 + i * 256 + threadIdx.x;
            if (flat) {
                off[i] = (long long)x * 8;
            } else {
                const int d = x % vecs, y = x / vecs;
                off[i] = (y / P.kv) * st[2] + (y % P.kv) * st[3] + d * 8;
            }
            if (x < total) v[i] = __ldcs((const uint4 *)(from + off[i]));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (piece * 1024 + i * 256 + threadIdx.x < total) __stcs((uint4 *)(to + off[i]), v[i]);
    }
}

__global__ void __launch_bounds__(256) pages_copy_kernel(const __grid_constant__ PagesDev P) {
    pages_let_next();
    pages_wait_front();
    const int *list = P.work + PW_LIST;
    copy_pages(P, min(P.work[PW_COPIES], P.n_seqs), [&](int e, int &src, int &dst, int &positions) {
        src = list[4 * e];
        dst = list[4 * e + 1];
        positions = list[4 * e + 2];
    });
}

// Where every page goes: live pages whose number is not below the number of live pages move into the free pages
// below it, both in ascending order.  map = new number, -1 for a free page.  One block.
__global__ void __launch_bounds__(1024) pages_plan_kernel(const __grid_constant__ PagesDev P, int *map) {
    __shared__ int sh[32];
    const int i = threadIdx.x;
    pages_let_next();
    pages_wait_front();
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
    pages_let_next();
    pages_wait_front();
    const int *holes = P.work + PW_LIST + 4 * P.n_seqs, *movers = holes + P.n_pages;
    for (int s = blockIdx.x; s < P.n_seqs; s += gridDim.x) {
        int *row = P.table + (long long)s * P.table_stride;
        const int n = pages_for(P, pages_len(P, s));
        for (int c = threadIdx.x; c < n; c += blockDim.x) {
            const int pg = row[c];
            if ((unsigned)pg < (unsigned)P.n_pages && map[pg] >= 0) row[c] = map[pg];
        }
    }
    copy_pages(P, P.work[PW_COPIES], [&](int e, int &src, int &dst, int &positions) {
        src = movers[e];
        dst = holes[e];
        positions = P.page;
    });
}

// Blocks for n copies: eight a multiprocessor at most, each with something to do.
unsigned copy_blocks(const PagesDev &P, long long n, int n_sm) {
    const long long pieces = (P.page * P.kv * (P.dim / 8) + 1023) / 1024;
    return (unsigned)std::max<long long>(1, std::min<long long>(8 * n_sm, n * P.n_layers * 2 * pieces));
}

}  // namespace

template <int TY>
cudaError_t launch_rope(const RopeParams &p, int n_sm, cudaStream_t st) {
    // weights are read 16 bytes at a time; their start is the caller's
    const bool weights = (((uintptr_t)p.q_norm | (uintptr_t)p.k_norm) & 15) == 0;
    if (p.rot % 16 == 0 && weights && (p.P.dim == 64 || p.P.dim == 128 || p.P.dim == 256)) {
        const dim3 grid(std::min(p.B.rows, 3 * n_sm));
        if (p.P.dim == 64) return launch_front(rope_append_wide_kernel<TY, 4>, grid, 256, 0, st, p);
        if (p.P.dim == 128) return launch_front(rope_append_wide_kernel<TY, 8>, grid, 256, 0, st, p);
        return launch_front(rope_append_wide_kernel<TY, 16>, grid, 256, 0, st, p);
    }
    return launch_front(rope_append_kernel<TY>, dim3(p.B.rows), 256, 0, st, p);
}

cudaError_t launch_rope_append(const RopeParams &p, int n_sm, cudaStream_t st, int *launches) {
    *launches += 1;
    if (p.ty == PTY_F32) return launch_rope<PTY_F32>(p, n_sm, st);
    if (p.ty == PTY_F16) return launch_rope<PTY_F16>(p, n_sm, st);
    return launch_rope<PTY_BF16>(p, n_sm, st);
}

cudaError_t launch_pages_fork(const PagesDev &P, const SlotList &l, cudaStream_t st, int *launches) {
    *launches += 1;
    return launch_front(pages_fork_kernel, dim3(l.n), 256, 0, st, P, l);
}

cudaError_t launch_pages_release(const PagesDev &P, const SlotList &l, cudaStream_t st, int *launches) {
    *launches += 1;
    return launch_front(pages_release_kernel, dim3(l.n), 256, 0, st, P, l);
}

cudaError_t launch_pages_reserve(const PagesDev &P, const SlotList &l, int heed, int n_sm, cudaStream_t st, int *launches) {
    *launches += 1;
    cudaError_t e = launch_front(pages_reserve_kernel, dim3(1), PAGES_MAX_LIST, 0, st, P, l, heed);
    if (e != cudaSuccess || l.n == 0) return e;
    *launches += 1;
    return launch_front(pages_copy_kernel, dim3(copy_blocks(P, l.n, n_sm)), 256, 0, st, P);
}

cudaError_t launch_pages_compact(const PagesDev &P, int *page_map, int n_sm, cudaStream_t st, int *launches) {
    if (!page_map) page_map = P.work + PW_LIST + 4 * P.n_seqs + 2 * P.n_pages;
    *launches += 2;
    cudaError_t e = launch_front(pages_plan_kernel, dim3(1), 1024, 0, st, P, page_map);
    if (e != cudaSuccess) return e;
    return launch_front(pages_move_kernel, dim3(copy_blocks(P, P.n_pages / 2 + 1, n_sm)), 256, 0, st, P, (const int *)page_map);
}

}  // namespace apk
