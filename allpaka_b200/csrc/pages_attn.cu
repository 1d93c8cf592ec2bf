// Attention of new rows over a paged KV cache.
//
#include "pages.cuh"
#include "pages_tc.cuh"

#include <cuda.h>
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
__device__ __forceinline__ void from_f32(float *p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// Positions that the row at `pos` sees: [lo, hi).
__host__ __device__ __forceinline__ void row_span(const AttendParams &p, int len, int pos, int &lo, int &hi) {
    hi = p.causal ? min(pos + 1, len) : len;
    lo = p.window ? max(0, pos - p.window + 1) : 0;
}

// o = sum_j p_j v_j / sum_j p_j, p_j = 2^(scale_log2 q.k_j - m), m the running maximum: one pass over the positions.
// One warp per (row, head), the head's dimensions over the lanes.  A position that is not visible is not read at all,
// so nothing that it holds (infinities, NaN, what an earlier sequence left) reaches a result.
template <int D, typename T, typename C>
__device__ __noinline__ void attend_row(const AttendParams &p, const SeqRows &s, int t, int h, int lane) {
    constexpr int E = D / 32;
    const int kvh = h / p.group;
    int lo, hi;
    row_span(p, s.len, s.len - s.rows + (t - s.first), lo, hi);
    const T *q = (const T *)p.q + t * p.qs[0] + h * p.qs[1];
    float qr[E], o[E];
    for (int e = 0; e < E; ++e) { qr[e] = to_f32(q[lane * E + e]); o[e] = 0.f; }
    float m = -INFINITY, l = 0.f;
    const C *kb = (const C *)p.P.k + p.layer * p.P.ks[0] + kvh * p.P.ks[3] + lane * E;
    const C *vb = (const C *)p.P.v + p.layer * p.P.vs[0] + kvh * p.P.vs[3] + lane * E;
    for (int j0 = lo; j0 < hi;) {
        const int pg = page_of(p.P, s.slot, j0), in = j0 & (p.P.page - 1);
        const int n = min(min(p.P.page - in, hi - j0), 8);
        if (pg >= 0) {
            const C *kp = kb + pg * p.P.ks[1] + in * p.P.ks[2], *vp = vb + pg * p.P.vs[1] + in * p.P.vs[2];
            float sc[8], mx = m;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float d = 0.f;
                if (j < n)
                    for (int e = 0; e < E; ++e) d += qr[e] * to_f32(kp[j * p.P.ks[2] + e]);
                for (int x = 16; x; x >>= 1) d += __shfl_xor_sync(~0u, d, x);
                sc[j] = j < n ? d * p.scale_log2 : -INFINITY;
                mx = fmaxf(mx, sc[j]);
            }
            const float base = mx == -INFINITY ? 0.f : mx, c = exp2f(m - base);
            l *= c;
            for (int e = 0; e < E; ++e) o[e] *= c;
            m = mx;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) {
                    const float w = exp2f(sc[j] - base);
                    l += w;
                    for (int e = 0; e < E; ++e) o[e] += w * to_f32(vp[j * p.P.vs[2] + e]);
                }
        }
        j0 += n;
    }
    T *out = (T *)p.out + t * p.os[0] + h * p.os[1] + lane * E;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    for (int e = 0; e < E; ++e) from_f32(out + e, o[e] * inv);
}

// ----------------------------------------------------------------------------------------------- tensor cores
//
// A tile is one kv head and up to 256 query rows of one sequence (tokens x heads of the GQA group), its work the
// 128-position blocks of K and V that its rows see.  One CTA per SM; the blocks of all tiles in a row are cut into equal
// contiguous ranges, one per CTA, so long and short sequences, chunks and single tokens load every SM alike.  A tile that
// a cut runs through leaves partial results (unnormalised rows, maximum, sum) in the workspace, which
// attend_join_kernel merges in a fixed order.
//
// Ten warps: two groups of four for the softmax (thread = row = TMEM lane), one that issues TMA copies, one that issues
// the tensor instructions.  S = Q K^T (both from shared memory) goes to TMEM; the softmax group turns its 128 x 128
// scores into 16-bit weights P over the same TMEM columns; O += P V takes P from TMEM and V from shared memory
// (transposed by its descriptor).
//   wide tile (more than 128 rows): group w works on rows 128w.. and shares every K and V block with the other;
//   narrow tile (one token of a few heads, mostly): both groups hold the same rows, group w takes every second block,
//   and group 0 joins the two results, which lie on the same TMEM lanes.
// The maximum that the weights refer to moves only when a row's grows by more than 2^8 (LAZY): until then weights are at
// most 2^8 (x 2^7 for f16, whose range is 2^-24 .. 2^16), and O keeps its scale.
//
// 32-bit rows (over f16 pages): a query, scaled by a power of two of its own, and a weight are each the sum of two f16
// values, 22 bits; every product is done for both.  The tensor cores' sums are truncated at about 24 bits, and over the
// blocks of a long sequence that would add up to 2^-15: so O of a block starts from 0, and group 1 adds it to its registers
// in 32 bits, while group 0 does the softmax of every block (tiles are narrow, two score and two O buffers).

constexpr int TC_THREADS = 384;      // warps 0-7 softmax, 8 copies, 9 tensor instructions, 10 and 11 only complete the third register group
constexpr int TC_STAGES = 4;
constexpr int TC_BLOCK = 128;         // positions a block
constexpr int TC_OVERHEAD = 2;        // what opening and closing a tile costs, in blocks
constexpr int TC_MIN_UNITS = 4;       // least range of a CTA
constexpr int TC_MOST = 1 << 30;      // units of a call (the host has bounded a proper batch's)
constexpr float TC_LAZY = 8.f;

struct TcParams {
    AttendParams a;
    int n_ctas, ws_rows;    // rows of a partial result in the workspace: 256, or fewer where no tile can have more
    int *meta;              // [n_ctas][8]
    float *ml;              // [n_ctas][2][ws_rows][2]
    float *part;            // [n_ctas][2][ws_rows][D]
    long long wait_limit;
};

struct TcGeom { int tq, step; };  // tokens per 128 rows, per tile
__host__ __device__ __forceinline__ TcGeom tc_geom(const AttendParams &p) {
    const int tq = 128 / p.group;
    return {tq, p.ty == PTY_F32 ? tq : 2 * tq};
}

struct TcTile {
    int seq, t, h;          // batch index, tile of the sequence, kv head
    int base;               // the tile's first unit
    int nt;                 // tiles of the sequence
    SeqRows s;
    int tok0, ntok, k0, nb; // first token (of the sequence), tokens, first block, blocks
};

__host__ __device__ __forceinline__ void tc_span(const AttendParams &p, const TcGeom &g, TcTile &x) {
    x.tok0 = x.t * g.step;
    x.ntok = min(x.s.rows - x.tok0, g.step);
    const int pos = x.s.len - x.s.rows + x.tok0;
    int lo, hi, unused;
    row_span(p, x.s.len, pos, lo, unused);
    row_span(p, x.s.len, pos + x.ntok - 1, unused, hi);
    x.k0 = lo / TC_BLOCK;
    x.nb = hi > lo ? (hi + TC_BLOCK - 1) / TC_BLOCK - x.k0 : 0;
}

__host__ __device__ __forceinline__ void tc_open(const AttendParams &p, const TcGeom &g, TcTile &x) {
    while (x.seq < p.B.n) {
        x.s = batch_seq(p.P, p.B, x.seq);
        x.nt = (x.s.rows + g.step - 1) / g.step;
        if (x.nt > 0) break;
        x.seq++;
    }
    if (x.seq < p.B.n) tc_span(p, g, x);
}

__host__ __device__ __forceinline__ void tc_next(const AttendParams &p, const TcGeom &g, TcTile &x) {
    x.base += x.nb + TC_OVERHEAD;
    if (++x.h < p.P.kv) return;
    x.h = 0;
    if (++x.t < x.nt) {
        tc_span(p, g, x);
        return;
    }
    x.t = 0;
    x.seq++;
    tc_open(p, g, x);
}

// Where the cut before unit u falls: a tile and a block.  A cut that would leave a single block on one side moves to
// the tile's edge.
__host__ __device__ inline void tc_cut(const AttendParams &p, const TcGeom &g, const int *prefix, int total, int u, int *out) {
    TcTile x;
    x.t = x.h = 0;
    int block = 0;
    if (u >= total) {
        x.seq = p.B.n;
        x.base = total;
    } else {
        int lo = 0, hi = p.B.n;  // the last sequence with prefix <= u; it has units, since its successor's prefix is larger
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= u) lo = mid;
            else hi = mid;
        }
        x.seq = lo;
        x.base = prefix[lo];
        tc_open(p, g, x);
        while ((long long)x.base + (long long)(x.nb + TC_OVERHEAD) * p.P.kv <= u) {
            x.base += (x.nb + TC_OVERHEAD) * p.P.kv;
            ++x.t;
            tc_span(p, g, x);
        }
        x.h = (u - x.base) / (x.nb + TC_OVERHEAD);
        x.base += x.h * (x.nb + TC_OVERHEAD);
        block = u - x.base - TC_OVERHEAD;
        if (u == x.base || block <= 1) {
            block = 0;
        } else if (block >= x.nb - 1) {
            tc_next(p, g, x);
            block = 0;
        }
    }
    out[0] = x.seq; out[1] = x.t; out[2] = x.h; out[3] = block; out[4] = x.base;
}

// The segments of a CTA's range, in order.  Every warp walks them for itself, in shared memory (the registers belong to
// the scores): its first lane takes the step.
struct TcWalk {
    TcTile x;
    int j0, j1;   // blocks of the tile
    __host__ __device__ __forceinline__ bool check(const AttendParams &p, const int *end) {
        if (x.seq >= p.B.n) return false;
        if (x.seq == end[0] && x.t == end[1] && x.h == end[2]) {
            j1 = end[3];
            return j1 > j0;
        }
        j1 = x.nb;
        return x.seq < end[0] || (x.seq == end[0] && (x.t < end[1] || (x.t == end[1] && x.h < end[2])));
    }
    __host__ __device__ __forceinline__ bool start(const AttendParams &p, const TcGeom &g, const int *begin, const int *end) {
        x.seq = begin[0]; x.t = begin[1]; x.h = begin[2]; x.base = begin[4];
        j0 = begin[3];
        tc_open(p, g, x);
        return check(p, end);
    }
    __host__ __device__ __forceinline__ bool next(const AttendParams &p, const TcGeom &g, const int *end) {
        if (x.seq == end[0] && x.t == end[1] && x.h == end[2]) return false;
        tc_next(p, g, x);
        j0 = 0;
        return check(p, end);
    }
};

struct TcShared {
    uint64_t full[TC_STAGES], empty[TC_STAGES], q_full, s_full[2], p_full[2], o_full[2], o_free[2], drain;
    uint32_t tmem;
    int dead, odd;          // a wait ran out; a result is not finite
    int begin[8], end[8];   // the CTA's range: sequence, tile, head, block, and the tile's first unit
    float ml[128][2];       // narrow tiles: maxima and sums of the other group
    float by[2][128];       // 32-bit rows: what a block's new maximum makes of the sums so far
    float unit[128];        // 32-bit rows: a row's power of two
    TcWalk walk[10];
    int prefix[1];          // [n + 1] units before each sequence
};

// Order in which a narrow tile's n blocks of K and V pass through the ring: K0 K1 V0 K2 V1 ... (wide: K0 V0 K1 V1 ...)
__host__ __device__ __forceinline__ int tc_slot_k(bool wide, int j) { return wide ? 2 * j : (j < 2 ? j : 2 * j - 1); }
__host__ __device__ __forceinline__ int tc_slot_v(bool wide, int j, int n) { return wide ? 2 * j + 1 : (j < n - 1 ? 2 * j + 2 : 2 * n - 1); }

__device__ __forceinline__ bool tc_wait(TcShared &sh, uint64_t *bar, uint32_t parity, const TcParams &p, int site) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*(volatile int *)&sh.dead) return false;
    if (mbar_wait_bounded(bar, parity, p.wait_limit)) return true;
    *(volatile int *)&sh.dead = 1;
    atomicCAS(&p.a.P.work[PW_ERR], 0, site);
    return false;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float a, float b) {  // a in the low half
    uint32_t r;
    if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ float2 unpack16(uint32_t x) { return __half22float2(*(const __half2 *)&x); }
// Values that a load into registers has delivered may not be used before its wait: ties the registers to this place.
__device__ __forceinline__ void pin32(uint32_t *r) {
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i])::"memory");
}
__device__ __forceinline__ bool softmax_bar_or(bool x) {  // the 256 threads of both groups
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)x) : "memory");
    return r != 0;
}

__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u); }

template <int D, int TY>
__global__ void __launch_bounds__(TC_THREADS, 1)
attend_tc_kernel(const __grid_constant__ TcParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int PANELS = D / 64;
    constexpr bool BF = TY == PTY_BF16, F32 = TY == PTY_F32;
    constexpr int PARTS = F32 ? 2 : 1;
    constexpr uint32_t TILE = TC_BLOCK * D * 2;    // bytes of a Q tile or of a block of K or V
    constexpr uint32_t O_COL = 256;                // TMEM columns: S0 S1 O0 O1
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *const qs = smem, *const ring = smem + 2 * TILE;
    TcShared &sh = *(TcShared *)(ring + TC_STAGES * TILE);
    const AttendParams &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const TcGeom g = tc_geom(a);

    if (tid == 0) {
        for (int i = 0; i < TC_STAGES; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 1); }
        mbar_init(&sh.q_full, 8);
        for (int i = 0; i < 2; ++i) { mbar_init(&sh.s_full[i], 1); mbar_init(&sh.p_full[i], 4); mbar_init(&sh.o_full[i], 1); mbar_init(&sh.o_free[i], 4); }
        mbar_init(&sh.drain, 1);
        sh.dead = sh.odd = 0;
        fence_mbar_init();
    }
    if (warp == 9) tm_alloc(&sh.tmem, 512);

    // units of every sequence, then their running sum
    {
        const int n = a.B.n;
        const bool lanes = n < 64;  // few sequences: a warp each, its lanes over the tiles; many: a thread each
        for (int i = lanes ? warp : tid; i < n; i += lanes ? TC_THREADS / 32 : TC_THREADS) {
            TcTile x;
            x.s = batch_seq(a.P, a.B, i);
            const int nt = (x.s.rows + g.step - 1) / g.step;
            int units = 0;
            for (x.t = lanes ? lane : 0; x.t < nt; x.t += lanes ? 32 : 1) {
                tc_span(a, g, x);
                units = min(units + x.nb + TC_OVERHEAD, TC_MOST);
            }
            if (lanes)
                for (int o = 16; o; o >>= 1) units = min(units + __shfl_xor_sync(~0u, units, o), TC_MOST);
            if (!lanes || lane == 0) sh.prefix[i + 1] = (int)min((long long)units * a.P.kv, (long long)TC_MOST);
        }
        __syncthreads();
        if (warp == 0) {
            int run = 0;
            for (int i0 = 0; i0 < n; i0 += 32) {
                int v = i0 + lane < n ? sh.prefix[i0 + lane + 1] : 0;
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(~0u, v, o);
                    if (lane >= o) v = min(v + y, TC_MOST);
                }
                v = min(run + v, TC_MOST);
                if (i0 + lane < n) sh.prefix[i0 + lane + 1] = v;
                run = __shfl_sync(~0u, v, 31);
            }
            if (lane == 0) sh.prefix[0] = 0;
        }
        __syncthreads();
    }
    // (offsets that overlap could claim more rows than there are: such a batch is left alone)
    const int total = sh.prefix[a.B.n] < TC_MOST ? sh.prefix[a.B.n] : 0;
    const int per = max((int)(((long long)total + p.n_ctas - 1) / p.n_ctas), TC_MIN_UNITS);
    const int cta = blockIdx.x;
    if (tid == 0 || tid == 32) {
        const long long u = (long long)(cta + (tid ? 1 : 0)) * per;
        tc_cut(a, g, sh.prefix, total, (int)(u < total ? u : total), tid ? sh.end : sh.begin);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t idesc_qk = tc_idesc(BF, 128, 128, false), idesc_pv = tc_idesc(BF, 128, D, true);

    // Register shares of the three groups of four warps: 2 x 208 + 80 <= 3 x 168, what the block was launched with.
    TcWalk &wk = sh.walk[min(warp, 9)];
    auto step = [&](bool first) {   // to the warp's first or next segment
        __syncwarp();
        int more = 0;
        if (lane == 0) more = first ? wk.start(a, g, sh.begin, sh.end) : wk.next(a, g, sh.end);
        __syncwarp();
        return __shfl_sync(~0u, more, 0) != 0;
    };
    int ring0 = 0;                        // ring entries before this segment

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp == 8) {
        // ------------------------------------------------------------------ TMA
        const int boxes = max(1, TC_BLOCK >> a.P.shift), rows = min(a.P.page, TC_BLOCK);
        bool ok = true;
        int filled = 0;
        for (bool more = step(true); more; more = step(false)) {
            const int n = wk.j1 - wk.j0;
            const bool wide = wk.x.ntok > g.tq;
            for (int e = 0; e < 2 * n; ++e) {
                // entry e of the segment: a block of K or of V
                bool is_v;
                int j;
                if (wide) { is_v = e & 1; j = e >> 1; }
                else if (e < 2 && e < n) { is_v = false; j = e; }
                else if (e == 2 * n - 1) { is_v = true; j = n - 1; }
                else { is_v = !(e & 1); j = is_v ? (e - 2) >> 1 : (e + 1) >> 1; }
                const int pos = (wk.x.k0 + wk.j0 + j) * TC_BLOCK;
                const int idx = ring0 + e, st = idx % TC_STAGES;
                // a page that does not exist (or lies behind the sequence) is asked for outside the pool: zeros arrive
                const int box = lane / PANELS, panel = lane % PANELS;
                const int at = pos + box * rows;
                int pg = a.P.n_pages;
                if (box < boxes && at < wk.x.s.len) {
                    pg = page_of(a.P, wk.x.s.slot, at);
                    if (pg < 0) pg = a.P.n_pages;
                }
                ok = __all_sync(~0u, tc_wait(sh, &sh.empty[st], ((idx / TC_STAGES) & 1) ^ 1, p, 1));
                if (!ok) break;
                filled = idx + 1;
                uint8_t *dst = ring + st * TILE;
                if (lane == 0) mbar_arrive_expect_tx(&sh.full[st], TILE);
                __syncwarp();
                if (box < boxes)
                    tma_load_4d(dst + panel * (TC_BLOCK * 128) + box * rows * 128, is_v ? &vmap : &kmap, panel * 64, at & (a.P.page - 1), wk.x.h, pg, &sh.full[st]);
            }
            if (!ok) break;
            ring0 += 2 * n;
        }
        // every copy that was asked for has arrived before the block ends
        for (int idx = max(0, filled - TC_STAGES); idx < filled; ++idx)
            (void)mbar_wait_bounded(&sh.full[idx % TC_STAGES], (idx / TC_STAGES) & 1, p.wait_limit);
    } else if (warp == 9) {
        // -------------------------------------------------------- tensor instructions: one thread
        if (lane == 0) {
            uint32_t ph_q = 0, ph_p[2] = {0, 0};
            bool ok = true;
            const uint32_t q_addr = smem_u32(qs), r_addr = smem_u32(ring);
            auto qk = [&](int w, int tile, int st) {
                const uint32_t qa = q_addr + tile * TILE, ka = r_addr + st * TILE;
                // (low parts first: a sum is truncated where it is, and theirs are small)
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t off = (k >> 2) * (TC_BLOCK * 128) + (k & 3) * 32;
                        tc_mma_ss(tmem + w * 128, tc_desc(qa + part * TILE + off, 16), tc_desc(ka + off, 16), idesc_qk, part < PARTS - 1 || k > 0);
                    }
                tc_commit(&sh.s_full[w]);
            };
            auto pv = [&](int w, int st, bool add) {
                const uint32_t va = r_addr + st * TILE;
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                    for (int k = 0; k < TC_BLOCK / 16; ++k)
                        tc_mma_ts(tmem + O_COL + w * D, tmem + w * 128 + part * 64 + k * 8, tc_desc(va + k * 2048, TC_BLOCK * 128), idesc_pv,
                                  add || part < PARTS - 1 || k > 0);
            };
            auto full = [&](int idx) { return tc_wait(sh, &sh.full[idx % TC_STAGES], (idx / TC_STAGES) & 1, p, 2); };
            auto weights = [&](int w) {
                const bool r = tc_wait(sh, &sh.p_full[w], ph_p[w], p, 3);
                ph_p[w] ^= 1;
                tc_fence_after();
                return r;
            };
            for (bool more = wk.start(a, g, sh.begin, sh.end); ok && more; more = wk.next(a, g, sh.end)) {
                const int n = wk.j1 - wk.j0;
                if (n == 0) continue;
                const bool wide = wk.x.ntok > g.tq;
                if (!(ok = tc_wait(sh, &sh.q_full, ph_q, p, 4))) break;
                ph_q ^= 1;
                if (!F32 && wide) {
                    if (!(ok = full(ring0))) break;
                    tc_fence_after();
                    qk(0, 0, ring0 % TC_STAGES);
                    qk(1, 1, ring0 % TC_STAGES);
                    tc_commit(&sh.empty[ring0 % TC_STAGES]);
                    for (int j = 0; j < n; ++j) {
                        const int v = ring0 + 2 * j + 1, kn = v + 1;
                        if (!(ok = full(v) && weights(0))) break;
                        pv(0, v % TC_STAGES, j > 0);
                        if (j + 1 < n) {
                            if (!(ok = full(kn))) break;
                            tc_fence_after();
                            qk(0, 0, kn % TC_STAGES);
                        } else {
                            tc_commit(&sh.o_full[0]);
                        }
                        if (!(ok = weights(1))) break;
                        pv(1, v % TC_STAGES, j > 0);
                        tc_commit(&sh.empty[v % TC_STAGES]);
                        if (j + 1 < n) {
                            qk(1, 1, kn % TC_STAGES);
                            tc_commit(&sh.empty[kn % TC_STAGES]);
                        } else {
                            tc_commit(&sh.o_full[1]);
                        }
                    }
                } else {
                    for (int j = 0; j < 2 && j < n; ++j) {
                        if (!(ok = full(ring0 + j))) break;
                        tc_fence_after();
                        qk(j, 0, (ring0 + j) % TC_STAGES);
                        tc_commit(&sh.empty[(ring0 + j) % TC_STAGES]);
                    }
                    for (int j = 0; ok && j < n; ++j) {
                        const int w = j & 1, v = ring0 + tc_slot_v(false, j, n), kn = ring0 + tc_slot_k(false, j + 2);
                        if (!(ok = full(v) && weights(w))) break;
                        pv(w, v % TC_STAGES, !F32 && j > 1);
                        tc_commit(&sh.empty[v % TC_STAGES]);
                        if (F32) tc_commit(&sh.o_full[w]);
                        if (j + 2 < n) {
                            if (!(ok = full(kn))) break;
                            tc_fence_after();
                            qk(w, 0, kn % TC_STAGES);
                            tc_commit(&sh.empty[kn % TC_STAGES]);
                        } else if (!F32) {
                            tc_commit(&sh.o_full[w]);
                        }
                    }
                }
                ring0 += 2 * n;
            }
        }
        __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ------------------------------------------------------------------ softmax
        // (after a wait that ran out the groups go on through their barriers, without the work)
        const int w = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // TMEM lane base of the warp, in the address's upper half
        const uint32_t ts = tmem + lanes + w * 128, to = tmem + lanes + O_COL + w * D;
        const bool flip = a.scale_log2 < 0.f;                // a negative scale turns the queries round
        const float c = fmaxf(fabsf(a.scale_log2), 1e-30f);  // (a scale of 0: hidden positions still get 2^-inf)
        const float shift = BF ? 0.f : 7.f;
        uint32_t ph_s = 0, ph_b = 0, ph_o[2] = {0, 0};
        bool ok = true, meta = false;
        auto wait = [&](uint64_t *bar, uint32_t parity, int site) { ok = __all_sync(~0u, ok && tc_wait(sh, bar, parity, p, site)); return ok; };
        for (bool more = step(true); more; more = step(false)) {
            const TcTile &x = wk.x;
            const int n = wk.j1 - wk.j0, k_first = x.k0 + wk.j0;
            const bool wide = x.ntok > g.tq;
            const bool whole = wk.j0 == 0 && wk.j1 == x.nb;
            // the row that this thread looks after
            const int tok = x.tok0 + (wide ? w * g.tq : 0) + r / a.group;
            const bool mine = r < g.tq * a.group && tok < x.tok0 + x.ntok;
            const int row = x.s.first + tok, head = x.h * a.group + r % a.group;
            int lo = 0, hi = 0;
            if (mine) row_span(a, x.s.len, x.s.len - x.s.rows + tok, lo, hi);
            // pages that are not there: looked for once a segment
            bool odd = false;
            for (int c0 = (k_first * TC_BLOCK >> a.P.shift) + tid; (c0 << a.P.shift) < min((k_first + n) * TC_BLOCK, x.s.len); c0 += 256)
                odd |= page_of(a.P, x.s.slot, c0 << a.P.shift) < 0;
            odd = softmax_bar_or(odd);   // (also: both groups have left the segment before)
            if (n > 0 && ok) {
                const int rows = min(x.ntok, g.tq) * a.group;
                const int tok_a = x.tok0 + (wide ? w * g.tq : 0);
                const int n_rows = wide && w ? (x.ntok - g.tq) * a.group : rows;
                const int nth = wide ? 128 : 256, me = wide ? r : tid;
                uint8_t *q_tile = qs + (wide ? w * TILE : 0);
                if constexpr (F32) {
                    constexpr int E = D / 32;
                    for (int rr = warp; rr < n_rows; rr += 8) {
                        const float *src = (const float *)a.q + (long long)(x.s.first + tok_a + rr / a.group) * a.qs[0] +
                                           (long long)(x.h * a.group + rr % a.group) * a.qs[1] + lane * E;
                        float v[E], mx = 0.f;
#pragma unroll
                        for (int e = 0; e < E; ++e) { v[e] = src[e]; mx = fmaxf(mx, fabsf(v[e])); }
                        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
                        // the row's largest value lands in [2^13, 2^14): what is 2^-27 of it still has 11 bits
                        const int ex = mx < INFINITY ? max((int)(__float_as_uint(mx) >> 23) - 127, -100) : 0;
                        const float by = __uint_as_float((uint32_t)(127 + 13 - ex) << 23) * (flip ? -1.f : 1.f);
                        if (lane == 0) sh.unit[rr] = __uint_as_float((uint32_t)max(127 - 13 + ex, 1) << 23);
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float u0 = v[e] * by, u1 = v[e + 1] * by;
                            const uint32_t hi = pack16<false>(u0, u1);
                            const float2 h = unpack16(hi);
                            const int d = lane * E + e;
                            uint8_t *at = q_tile + (d >> 6) * (TC_BLOCK * 128) + sw128(rr, (d >> 3) & 7) + (d & 7) * 2;
                            *(uint32_t *)at = hi;
                            *(uint32_t *)(at + TILE) = pack16<false>(u0 - h.x, u1 - h.y);
                        }
                    }
                } else
                for (int i = me; i < n_rows * (D / 8); i += nth) {
                    const int rr = i / (D / 8), ch = i % (D / 8);
                    const uint16_t *src = (const uint16_t *)a.q + (long long)(x.s.first + tok_a + rr / a.group) * a.qs[0] +
                                          (long long)(x.h * a.group + rr % a.group) * a.qs[1] + ch * 8;
                    uint4 v = *(const uint4 *)src;
                    if (flip) { v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u; }
                    *(uint4 *)(q_tile + (ch >> 3) * (TC_BLOCK * 128) + sw128(rr, ch & 7)) = v;
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.q_full);
            }
            float m = -INFINITY, l = 0.f;   // m: of the scaled scores, what the weights refer to
            const bool warp_mine = __any_sync(~0u, mine);
            // scores of positions that the row does not see
            auto hide = [&](float *f, int pos) {
                                    if (odd || __any_sync(~0u, mine && (pos < lo || pos + TC_BLOCK > hi))) {
                                        uint32_t see[4];   // a bit per position
                #pragma unroll
                                        for (int k = 0; k < 4; ++k) see[k] = bits_below(hi - pos - 32 * k) & ~bits_below(lo - pos - 32 * k);
                                        if (odd)
                                            for (int at = pos; at < min(pos + TC_BLOCK, x.s.len); at += min(a.P.page, 32))
                                                if (page_of(a.P, x.s.slot, at) < 0) {
                                                    const uint32_t gone = bits_below(min(a.P.page, 32)) << (at & 31);
                #pragma unroll
                                                    for (int k = 0; k < 4; ++k)
                                                        if (((at - pos) >> 5) == k) see[k] &= ~gone;
                                                }
                #pragma unroll
                                        for (int k = 0; k < 128; ++k)
                                            if (!((see[k >> 5] >> (k & 31)) & 1u)) f[k] = -INFINITY;
                                    }
            };
            // What lies behind the sequence in its last page takes part in the product with weight 0: it may not be NaN.
            auto clear_tail = [&](int j, int pos) {
                const int idx = ring0 + tc_slot_v(wide, j, n);
                if (!wait(&sh.full[idx % TC_STAGES], (idx / TC_STAGES) & 1, 6)) return false;
                if (pos + r >= x.s.len) {
                    uint8_t *v = ring + (idx % TC_STAGES) * TILE + r * 128;
#pragma unroll
                    for (int k = 0; k < PANELS * 8; ++k) *(uint4 *)(v + (k >> 3) * (TC_BLOCK * 128) + (k & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
                return true;
            };
            const int slot = 2 * cta + (wk.j0 == 0 ? 1 : 0);
            if constexpr (F32) {
                softmax_bar_or(false);   // the rows' powers of two are written
                const float cr = c * sh.unit[r];
                if (w == 0) {
                    for (int j = 0; j < n && ok; ++j) {
                        const int b = j & 1, pos = (k_first + j) * TC_BLOCK;
                        if (!wait(&sh.s_full[b], ph_b >> b & 1, 5)) break;
                        // (the sums of the block before last have been taken: its O buffer and its factor are free)
                        if (!wait(&sh.o_free[b], (ph_b >> b & 1) ^ 1, 9)) break;
                        ph_b ^= 1 << b;
                        tc_fence_after();
                        if (warp_mine) {
                            const uint32_t tb = tmem + lanes + b * 128;
                            uint32_t s[128], hi[64], lw[64];
                            tm_ld32(tb, s); tm_ld32(tb + 32, s + 32); tm_ld32(tb + 64, s + 64); tm_ld32(tb + 96, s + 96);
                            tm_wait_ld();
                            pin32(s); pin32(s + 32); pin32(s + 64); pin32(s + 96);
                            float *f = (float *)s;
                            hide(f, pos);
                            float mx[4] = {f[0], f[1], f[2], f[3]};
#pragma unroll
                            for (int k = 4; k < 128; ++k) mx[k & 3] = fmaxf(mx[k & 3], f[k]);
                            const float to_m = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * cr);
                            const float by = m == -INFINITY ? 0.f : ex2(m - to_m);
                            m = to_m;
                            sh.by[b][r] = by;
                            const float off = m == -INFINITY ? 0.f : -m;
                            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int k = 0; k < 128; k += 2) {
                                // weights up to 2^14 (f16 ends at 2^16); as a factor: in the exponent it would cost the argument bits
                                const float p0 = 16384.f * ex2(fmaf(f[k], cr, off)), p1 = 16384.f * ex2(fmaf(f[k + 1], cr, off));
                                sum[(k >> 1) & 3] += p0 + p1;
                                hi[k >> 1] = pack16<false>(p0, p1);
                                const float2 h = unpack16(hi[k >> 1]);
                                lw[k >> 1] = pack16<false>(p0 - h.x, p1 - h.y);
                            }
                            l = l * by + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                            tm_st32(tb, hi); tm_st32(tb + 32, hi + 32); tm_st32(tb + 64, lw); tm_st32(tb + 96, lw + 32);
                            tm_wait_st();
                        }
                        if (pos + TC_BLOCK > x.s.len && !clear_tail(j, pos)) break;
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.p_full[b]);
                    }
                    sh.ml[r][0] = m;
                    sh.ml[r][1] = l;
                    softmax_bar_or(false);
                } else {
                    float acc[D];
#pragma unroll
                    for (int k = 0; k < D; ++k) acc[k] = 0.f;
                    for (int j = 0; j < n && ok; ++j) {
                        const int b = j & 1;
                        if (!wait(&sh.p_full[b], ph_b >> b & 1, 7)) break;   // (the factor)
                        if (!wait(&sh.o_full[b], ph_b >> b & 1, 8)) break;
                        ph_b ^= 1 << b;
                        tc_fence_after();
                        if (warp_mine) {
                            const float by = sh.by[b][r];
#pragma unroll
                            for (int h = 0; h < D; h += 32) {
                                uint32_t o[32];
                                tm_ld32(tmem + lanes + O_COL + b * D + h, o);
                                tm_wait_ld();
                                pin32(o);
#pragma unroll
                                for (int k = 0; k < 32; ++k) acc[h + k] = fmaf(acc[h + k], by, __uint_as_float(o[k]));
                            }
                        }
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.o_free[b]);
                    }
                    softmax_bar_or(false);
                    const float top = sh.ml[r][0], lt = sh.ml[r][1], inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);
                    float *dst = whole ? (float *)a.out + row * a.os[0] + head * a.os[1] : p.part + ((long long)slot * p.ws_rows + r) * D;
                    float size = 0.f;
                    if (mine && ok) {
#pragma unroll
                        for (int k = 0; k < D; k += 4) {
                            const float u = whole ? inv : 1.f;
                            const float4 y = make_float4(acc[k] * u, acc[k + 1] * u, acc[k + 2] * u, acc[k + 3] * u);
                            size += (fabsf(y.x) + fabsf(y.y)) + (fabsf(y.z) + fabsf(y.w));
                            *(float4 *)(dst + k) = y;
                        }
                        if (!whole) *(float2 *)(p.ml + ((long long)slot * p.ws_rows + r) * 2) = make_float2(top, lt);
                        else if (!(size < INFINITY)) sh.odd = 1;   // (see attend_join_kernel)
                    }
                }
                ring0 += 2 * n;
            } else {
            const int cnt = wide ? n : (n - w + 1) >> 1;
            for (int i = 0; i < cnt && ok; ++i) {
                const int j = wide ? i : 2 * i + w, pos = (k_first + j) * TC_BLOCK;
                if (!wait(&sh.s_full[w], ph_s, 5)) break;
                ph_s ^= 1;
                tc_fence_after();
                if (warp_mine) {
                    uint32_t s[128];
                    tm_ld32(ts, s); tm_ld32(ts + 32, s + 32); tm_ld32(ts + 64, s + 64); tm_ld32(ts + 96, s + 96);
                    tm_wait_ld();
                    pin32(s); pin32(s + 32); pin32(s + 64); pin32(s + 96);
                    float *f = (float *)s;
                    hide(f, pos);
                    float mx = f[0];
#pragma unroll
                    for (int k = 1; k < 128; ++k) mx = fmaxf(mx, f[k]);
                    mx *= c;
                    const bool grow = mx > m + TC_LAZY;      // (from -inf: with the first visible position)
                    if (__any_sync(~0u, grow)) {
                        const float to_m = grow ? mx : m;
                        const float by = m == -INFINITY ? 0.f : ex2(m - to_m);
                        m = to_m;
                        l *= by;
                        if (i > 0) {
                            // this group's products so far are complete: they were issued before the scores
#pragma unroll
                            for (int h = 0; h < D; h += 32) {
                                uint32_t o[32];
                                tm_ld32(to + h, o);
                                tm_wait_ld();
                                pin32(o);
#pragma unroll
                                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * by);
                                tm_st32(to + h, o);
                            }
                        }
                    }
                    const float off = shift - (m == -INFINITY ? 0.f : m);
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < 128; k += 2) {
                        const float p0 = ex2(fmaf(f[k], c, off)), p1 = ex2(fmaf(f[k + 1], c, off));
                        sum[(k >> 1) & 3] += p0 + p1;
                        s[k >> 1] = pack16<BF>(p0, p1);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tm_st32(ts, s);
                    tm_st32(ts + 32, s + 32);
                    tm_wait_st();
                }
                if (pos + TC_BLOCK > x.s.len && !clear_tail(j, pos)) break;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[w]);
            }
            ring0 += 2 * n;

            // ---- the segment's result
            float m1 = -INFINITY, l1 = 0.f;
            if (!wide && n > 0) {
                if (w == 1) { sh.ml[r][0] = m; sh.ml[r][1] = l; }
                softmax_bar_or(false);
                if (w == 0) { m1 = sh.ml[r][0]; l1 = sh.ml[r][1]; }
            }
            if (w == 0 || wide) {
                if (n > 0) {
                    wait(&sh.o_full[w], ph_o[w], 7);
                    ph_o[w] ^= 1;
                }
                if (w == 0 && (wide ? n > 0 : n > 1)) {
                    if (!wide) wait(&sh.o_full[1], ph_o[1], 8);
                    ph_o[1] ^= 1;
                }
                tc_fence_after();
                const bool two = !wide && n > 1;
                const float top = fmaxf(m, m1);
                const float b0 = m == -INFINITY ? 0.f : ex2(m - top), b1 = m1 == -INFINITY ? 0.f : ex2(m1 - top);
                const float lt = l * b0 + l1 * b1;
                const float inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);
                float size = 0.f;
                const int wr = wide ? w * 128 + r : r;
                const bool part = mine && !whole;
                if (warp_mine && ok) {
                    uint16_t *out = (uint16_t *)a.out + row * a.os[0] + head * a.os[1];
                    float *pt = p.part + ((long long)slot * p.ws_rows + wr) * D;
#pragma unroll
                    for (int h = 0; h < D; h += 32) {
                        uint32_t o[32];
                        float *f = (float *)o;
                        if (n > 0) {
                            tm_ld32(to + h, o);
                            tm_wait_ld();
                            pin32(o);
                        } else {
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = 0;
                        }
                        // (a group whose maximum is still -inf has weights of 0 only, and its O holds zeros)
#pragma unroll
                        for (int k = 0; k < 32; ++k) f[k] *= b0;
                        if (two) {
                            uint32_t o1[32];
                            tm_ld32(to + D + h, o1);
                            tm_wait_ld();
                            pin32(o1);
#pragma unroll
                            for (int k = 0; k < 32; ++k) f[k] = fmaf(__uint_as_float(o1[k]), b1, f[k]);
                        }
                        if (part) {
#pragma unroll
                            for (int k = 0; k < 32; k += 4) *(float4 *)(pt + h + k) = make_float4(f[k], f[k + 1], f[k + 2], f[k + 3]);
                        } else if (mine) {
#pragma unroll
                            for (int k = 0; k < 32; ++k) { f[k] *= inv; size += fabsf(f[k]); }
#pragma unroll
                            for (int k = 0; k < 32; k += 8)
                                *(uint4 *)(out + h + k) = make_uint4(pack16<BF>(f[k], f[k + 1]), pack16<BF>(f[k + 2], f[k + 3]),
                                                                     pack16<BF>(f[k + 4], f[k + 5]), pack16<BF>(f[k + 6], f[k + 7]));
                        }
                    }
                    if (part) *(float2 *)(p.ml + ((long long)slot * p.ws_rows + wr) * 2) = make_float2(top, lt);
                    if (mine && whole && !(size < INFINITY)) sh.odd = 1;   // (see attend_join_kernel)
                }
            } else if (n > 1) {
                ph_o[1] ^= 1;
            }
            }
            // the first of a cut tile's pieces says how many follow
            if (!whole && wk.j0 == 0) {
                meta = true;
                if (tid == 0) {
                    const int first = x.base + TC_OVERHEAD + 2, last = x.base + TC_OVERHEAD + x.nb - 2;   // cuts that stay inside the tile
                    int *mt = p.meta + cta * 8;
                    mt[0] = last / per - (first - 1) / per;
                    mt[1] = x.seq; mt[2] = x.tok0; mt[3] = x.ntok; mt[4] = x.h; mt[5] = wide;
                }
            }
            tc_fence_before();
        }
        if (!meta && tid == 0) p.meta[cta * 8] = 0;
    }

    // ---- close: no copy and no tensor instruction may be in flight when the CTA ends
    __syncthreads();
    if (tid == 0) p.meta[cta * 8 + 6] = sh.odd;
    if (warp == 9) {
        if (lane == 0) {
            tc_commit(&sh.drain);
            (void)mbar_wait_bounded(&sh.drain, 0, p.wait_limit);
        }
        __syncwarp();
        tc_fence_after();
        tm_dealloc(tmem, 512);
    }
}

// Merges the pieces of a cut tile: block c those of the tile whose first piece CTA c has left.  Piece 0 lies in slot 1 of CTA c,
// the others in slot 0 of the CTAs behind it.  A warp per row, in the order of the pieces.
// An infinity or NaN in V at a position that some rows of a tile do not see has met their weight of 0 in the product.  Such
// rows show it by not being finite; they are done over here, position by position.
template <int D, int TY>
__global__ void __launch_bounds__(512) attend_join_kernel(const __grid_constant__ TcParams p) {
    constexpr int E = D / 32;
    typedef typename Elem<TY>::T T;
    typedef typename Elem<TY == PTY_BF16 ? PTY_BF16 : PTY_F16>::T C;
    const AttendParams &a = p.a;
    const int *mt = p.meta + blockIdx.x * 8;
    const int more = mt[0];
    int odd = 0;
    for (int i = threadIdx.x; i < p.n_ctas; i += blockDim.x) odd |= p.meta[i * 8 + 6];
    if (__syncthreads_or(odd)) {
        for (long long u = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * 16 + (threadIdx.x >> 5); u < (long long)a.B.rows * a.heads;
             u += (long long)gridDim.x * gridDim.y * 16) {
            const int t = (int)(u / a.heads), hd = (int)(u % a.heads), i = batch_find(a.B, t);
            if (i < 0) continue;
            const T *o = (const T *)a.out + t * a.os[0] + hd * a.os[1] + (threadIdx.x & 31) * E;
            float size = 0.f;
            for (int e = 0; e < E; ++e) size += fabsf(to_f32(o[e]));
            if (__any_sync(~0u, !(size < INFINITY))) attend_row<D, T, C>(a, batch_seq(a.P, a.B, i), t, hd, threadIdx.x & 31);
        }
    }
    if (more <= 0 || more >= p.n_ctas - (int)blockIdx.x) return;
    const int seq = mt[1], tok0 = mt[2], ntok = mt[3], h = mt[4], wide = mt[5];
    const SeqRows s = batch_seq(a.P, a.B, seq);
    const int tq = 128 / a.group, lane = threadIdx.x & 31;
    const int n_rows = wide ? 256 : ntok * a.group;
    for (int r = blockIdx.y * 16 + (threadIdx.x >> 5); r < n_rows; r += 16 * gridDim.y) {
        const int half = r >> 7, rr = r & 127, tok = (wide ? half * tq : 0) + rr / a.group;
        if (rr >= tq * a.group || tok >= ntok) continue;
        auto at = [&](int piece) { return (long long)(piece ? 2 * ((int)blockIdx.x + piece) : 2 * (int)blockIdx.x + 1) * p.ws_rows + r; };
        float top = -INFINITY, l = 0.f, o[E];
        for (int i = lane; i <= more; i += 32) top = fmaxf(top, p.ml[at(i) * 2]);
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
        for (int e = 0; e < E; ++e) o[e] = 0.f;
        for (int i = 0; i <= more; ++i) {
            const float2 ml = *(const float2 *)(p.ml + at(i) * 2);
            if (ml.x == -INFINITY) continue;
            const float b = ex2(ml.x - top);
            l += b * ml.y;
            const float *src = p.part + at(i) * D + lane * E;
            for (int e = 0; e < E; ++e) o[e] = fmaf(b, src[e], o[e]);
        }
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        float size = 0.f;
        for (int e = 0; e < E; ++e) { o[e] *= inv; size += fabsf(o[e]); }
        const int row = s.first + tok0 + tok, head = h * a.group + rr % a.group;
        T *out = (T *)a.out + row * a.os[0] + head * a.os[1] + lane * E;
        for (int e = 0; e < E; ++e) from_f32(out + e, o[e]);
        if (__any_sync(~0u, !(size < INFINITY))) {
            __syncwarp();
            attend_row<D, T, C>(a, s, row, head, lane);
        }
    }
}

// ------------------------------------------------------------------------------------------------ launches

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) fn = nullptr;
        return (EncodeTiled)fn;
    }();
    return f;
}

// K or V of one layer as (dimension, position, kv head, page); boxes of 64 dimensions x the positions of a page.
bool page_map(CUtensorMap *m, const PagesDev &P, const uint16_t *base, const long long *st) {
    const cuuint64_t dims[4] = {(cuuint64_t)P.dim, (cuuint64_t)P.page, (cuuint64_t)P.kv, (cuuint64_t)P.n_pages};
    // (an axis of length 1 has no stride of its own)
    const cuuint64_t row = (cuuint64_t)P.dim * 2;
    const cuuint64_t strides[3] = {(cuuint64_t)st[2] * 2, P.kv == 1 ? row : (cuuint64_t)st[3] * 2, P.n_pages == 1 ? row : (cuuint64_t)st[1] * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)std::min(P.page, TC_BLOCK), 1, 1}, one[4] = {1, 1, 1, 1};
    const EncodeTiled f = encode_tiled();
    return f && f(m, P.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, (void *)base, dims, strides, box, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct TcSize { size_t meta, ml, part; int rows; };
TcSize tc_size(const AttendParams &p, int n_sm) {
    TcSize s;
    const TcGeom g = tc_geom(p);
    s.rows = p.B.rows > g.tq ? (g.step > g.tq ? 256 : 128) : p.B.rows * p.group;
    s.meta = ((size_t)n_sm * 8 * 4 + 255) / 256 * 256;
    s.ml = ((size_t)n_sm * 2 * s.rows * 2 * 4 + 255) / 256 * 256;
    s.part = (size_t)n_sm * 2 * s.rows * p.P.dim * 4;
    return s;
}

template <int D, int TY>
cudaError_t launch_tc(const AttendParams &p, int n_sm, void *ws, long long wait_limit, cudaStream_t st, int *launches) {
    constexpr int smem = 1024 + (2 + TC_STAGES) * TC_BLOCK * D * 2 + (int)sizeof(TcShared) + 4 * PAGES_MAX_BATCH;
    static_assert(smem <= 232448, "shared memory of a block");
    CUtensorMap km, vm;
    if (!page_map(&km, p.P, p.P.k + p.layer * p.P.ks[0], p.P.ks) || !page_map(&vm, p.P, p.P.v + p.layer * p.P.vs[0], p.P.vs)) return cudaErrorNotSupported;
    const TcSize z = tc_size(p, n_sm);
    TcParams q{};
    q.a = p;
    q.n_ctas = n_sm;
    q.ws_rows = z.rows;
    q.meta = (int *)ws;
    q.ml = (float *)((char *)ws + z.meta);
    q.part = (float *)((char *)ws + z.meta + z.ml);
    q.wait_limit = wait_limit;
    // (the limit belongs to the kernel on the current device; setting it again costs a few hundred nanoseconds)
    cudaError_t e = cudaFuncSetAttribute(attend_tc_kernel<D, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    attend_tc_kernel<D, TY><<<n_sm, TC_THREADS, smem, st>>>(q, km, vm);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    attend_join_kernel<D, TY><<<dim3(n_sm, z.rows == 256 ? 4 : 1), 512, 0, st>>>(q);
    *launches += 2;
    return cudaGetLastError();
}

}  // namespace

size_t attend_ws_bytes(const AttendParams &p, int n_sm) {
    const TcSize z = tc_size(p, n_sm);
    return z.meta + z.ml + z.part;
}

cudaError_t launch_attend(const AttendParams &p, int n_sm, void *ws, long long wait_limit, cudaStream_t st, int *launches) {
    const bool d128 = p.P.dim == 128;
    if (p.ty == PTY_F32) return (d128 ? launch_tc<128, PTY_F32> : launch_tc<64, PTY_F32>)(p, n_sm, ws, wait_limit, st, launches);
    if (p.ty == PTY_BF16) return (d128 ? launch_tc<128, PTY_BF16> : launch_tc<64, PTY_BF16>)(p, n_sm, ws, wait_limit, st, launches);
    return (d128 ? launch_tc<128, PTY_F16> : launch_tc<64, PTY_F16>)(p, n_sm, ws, wait_limit, st, launches);
}

}  // namespace apk
