// Attention of new rows over a paged KV cache.
//
#include "pages.cuh"
#include "pages_tc.cuh"

#include <cuda.h>
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
// Two groups of four warps for the softmax (thread = row = TMEM lane), a warp that walks the CTA's range and hands out its
// segments, one that issues TMA copies, one that issues the tensor instructions.  S = Q K^T (both from shared memory) goes
// to TMEM; the softmax group turns its 128 x 128 scores into 16-bit weights P over the same TMEM columns; O += P V takes P
// from TMEM and V from shared memory (transposed by its descriptor).
//   wide tile (more than 128 rows): group w works on rows 128w.. and shares every K and V block with the other;
//   narrow tile (one token of a few heads, mostly): both groups hold the same rows, group w takes every second block,
//   and group 0 joins the two results, which lie on the same TMEM lanes.  Up to 32 rows lie in TMEM four times, and each
//   copy weighs a quarter of a block's positions: one warp would otherwise do it all.
// The maximum that the weights refer to moves only when a row's grows by more than 2^8 (LAZY): until then weights are at
// most 2^8 (x 2^7 for f16, whose range is 2^-24 .. 2^16), and O keeps its scale.
//
// 16-bit rows: a weight is rounded to the rows' type, by half a step at most (f16 2^-11, bf16 2^-8, relative), because the
// tensor instruction takes V and the weights in one type; maxima and the weights' sum stay in 32 bits and take the weight before
// its rounding.  A second part, as below, would double the products with V and the weights' registers.  Against 64 bits the
// results are off by 2.3e-4 to 2.9e-4 (f16; 2.1e-4 with weights in 32 bits, which is the result's own rounding) and 2.0e-3 to
// 2.3e-3 (bf16; 1.7e-3).  O is summed over a CTA's whole range in TMEM, where sums are truncated at about 24 bits: with V = 1
// everywhere most f16 results came out one step (2^-11) low over 2^20 positions a CTA, one in a thousand over 2^19, none over 2^17.
//
// 32-bit rows (over f16 pages): a query, scaled by a power of two of its own, and a weight are each the sum of two f16
// values, 22 bits; every product is done for both.  The tensor cores' sums are truncated at about 24 bits, and over the
// blocks of a long sequence that would add up to 2^-15: so O of a block starts from 0, and group 1 adds it to its registers
// in 32 bits, while group 0 does the softmax of every block (tiles are narrow, two score and two O buffers).
//
// What bounds it, and what it measured (loops of single calls, from the best of several B200s to the slowest).  Single tokens:
// the bytes of K and V; 64 sessions of 200 to 8192 positions (577 MB) 105 to 128 us, 4.5 to 5.5 TB/s or 0.70 to 0.85 of the
// measured copy rate; one of 131077 positions 93 to 105 us, 0.79 to 0.89; the rest is 15 us of opening, joining and cold code.
// Chunks: a group's chain scores -> weights (1.1 us for 128 x 128: the exponentials alone are 0.6) ->
// both products (0.6) -> scores, with 0.5 us of hand-overs in between; two groups in turn keep the tensor cores half busy:
// 4096 rows over 8192 positions 444 to 496 us, 833 to 930 TFLOP/s.  TMEM is full (two times 128 columns of scores and of O), so there is
// no third group and no second score buffer; 64-position steps with two of them took 600 us.
// 32-bit rows: the tensor cores' time for every product done twice, 1.7 us a block.

constexpr int TC_THREADS = 384;      // warps 0-7 softmax, 8 copies, 9 tensor instructions, 10 walks the segments, 11 completes the third register group
constexpr int TC_MOST_STAGES = 8;     // blocks of K or V in the ring: 512 / D, 128 KB
constexpr int TC_BLOCK = 128;         // positions a block
// Units of work: a block of a narrow tile is one, of a wide tile two; opening and closing a tile costs as much as TC_OPEN blocks of
// its own.  (64 sessions of 200 to 8192 positions: 122 us with 2, 116 with 3, 109 with 4, 110 with 6; a 4096-row chunk 454, 454, 447, 443.)
constexpr int TC_OPEN = 4;
constexpr int TC_MIN_UNITS = 2;       // least range of a CTA
constexpr int TC_FEW = 4;             // fewer units a CTA than this, without the opening: it is not counted, so that all CTAs have a share
constexpr int TC_MOST = 1 << 30;      // units of a call (the host has bounded a proper batch's)
constexpr int TC_SEGS = 4;            // segments that are known ahead
constexpr int TC_INFO = 256;          // sequences that a block keeps a copy of
constexpr long long TC_DRAIN = 1ll << 31;  // cycles that a block waits for its own copies and products at its end, whatever the waits' budget
constexpr float TC_LAZY = 8.f;

struct TcParams {
    AttendParams a;
    int n_ctas, ws_rows;    // rows of a partial result in the workspace: 256, or fewer where no tile can have more
    int *meta;              // [n_ctas][8]
    float *ml;              // [n_ctas][2][ws_rows][2]
    float *part;            // [n_ctas][2][ws_rows][D]
    long long wait_limit;
};

// Everything that says how a call's work is cut.
struct TcBatch {
    const AttendParams &p;
    int tq, step;           // tokens per 128 rows, per tile
    const SeqRows *info;    // the first TC_INFO sequences, where a copy is at hand
    int open = TC_OPEN;     // blocks that opening a tile counts for
    __host__ __device__ __forceinline__ TcBatch(const AttendParams &p_, const SeqRows *i)
        : p(p_), tq(128 / p_.group), step(p_.ty == PTY_F32 ? 128 / p_.group : 2 * (128 / p_.group)), info(i) {}
    __host__ __device__ __forceinline__ SeqRows seq(int i) const { return info && i < TC_INFO ? info[i] : batch_seq(p.P, p.B, i); }
};

struct TcTile {
    int seq, t, h;          // batch index, tile of the sequence, kv head
    int base;               // the tile's first unit
    int nt;                 // tiles of the sequence
    SeqRows s;
    int tok0, ntok, k0, nb; // first token (of the sequence), tokens, first block, blocks
    int per_block, opening; // units
    __host__ __device__ __forceinline__ int units() const { return nb * per_block + opening; }
};

__host__ __device__ __forceinline__ void tc_span(const TcBatch &c, TcTile &x) {
    x.tok0 = x.t * c.step;
    x.ntok = min(x.s.rows - x.tok0, c.step);
    const int pos = x.s.len - x.s.rows + x.tok0;
    int lo, hi, unused;
    row_span(c.p, x.s.len, pos, lo, unused);
    row_span(c.p, x.s.len, pos + x.ntok - 1, unused, hi);
    x.k0 = lo / TC_BLOCK;
    x.nb = hi > lo ? (hi + TC_BLOCK - 1) / TC_BLOCK - x.k0 : 0;
    x.per_block = x.ntok > c.tq ? 2 : 1;
    x.opening = max(c.open * x.per_block, x.nb == 0 ? 1 : 0);   // (a tile without blocks has its rows to clear)
}

__host__ __device__ __forceinline__ void tc_open(const TcBatch &c, TcTile &x) {
    while (x.seq < c.p.B.n) {
        x.s = c.seq(x.seq);
        x.nt = (x.s.rows + c.step - 1) / c.step;
        if (x.nt > 0) break;
        x.seq++;
    }
    if (x.seq < c.p.B.n) tc_span(c, x);
}

__host__ __device__ __forceinline__ void tc_next(const TcBatch &c, TcTile &x) {
    x.base += x.units();
    if (++x.h < c.p.P.kv) return;
    x.h = 0;
    if (++x.t < x.nt) {
        tc_span(c, x);
        return;
    }
    x.t = 0;
    x.seq++;
    tc_open(c, x);
}

// Fewest blocks of a piece of a cut tile: its rows are loaded, stored and joined once more, which costs a narrow tile about one
// block's time and a wide one (up to 256 rows of partial sums) several.  (Mixed chunks 39 us with 4 for wide ones, 37 with 6 or 8.)
__host__ __device__ __forceinline__ int tc_edge(const TcBatch &c, const TcTile &x) { return x.ntok > c.tq ? 6 : 2; }

// Where the cut before unit u falls: a tile and a block of it (returned).  A cut too near to a tile's edge moves there.
__host__ __device__ inline int tc_cut(const TcBatch &c, const int *prefix, int total, int u, TcTile &x) {
    x.t = x.h = 0;
    int block = 0;
    if (u >= total) {
        x.seq = c.p.B.n;
        x.base = total;
    } else {
        int lo = 0, hi = c.p.B.n;  // the last sequence with prefix <= u; it has units, since its successor's prefix is larger
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= u) lo = mid;
            else hi = mid;
        }
        x.seq = lo;
        x.base = prefix[lo];
        tc_open(c, x);
        while ((long long)x.base + (long long)x.units() * c.p.P.kv <= u) {
            x.base += x.units() * c.p.P.kv;
            ++x.t;
            tc_span(c, x);
        }
        x.h = (u - x.base) / x.units();
        x.base += x.h * x.units();
        block = u > x.base + x.opening ? (u - x.base - x.opening) / x.per_block : 0;
        if (block < tc_edge(c, x)) {
            block = 0;
        } else if (block > x.nb - tc_edge(c, x)) {
            tc_next(c, x);
            block = 0;
        }
    }
    return block;
}

// The segments of a CTA's range, in order.
struct TcWalk {
    TcTile x;
    int j0, j1;                      // blocks of the tile
    int e_seq, e_t, e_h, e_block;    // where the range ends
    __host__ __device__ __forceinline__ bool check(const TcBatch &c) {
        if (x.seq >= c.p.B.n) return false;
        if (x.seq == e_seq && x.t == e_t && x.h == e_h) {
            j1 = e_block;
            return j1 > j0;
        }
        j1 = x.nb;
        return x.seq < e_seq || (x.seq == e_seq && (x.t < e_t || (x.t == e_t && x.h < e_h)));
    }
    __host__ __device__ __forceinline__ bool next(const TcBatch &c) {
        if (x.seq == e_seq && x.t == e_t && x.h == e_h) return false;
        tc_next(c, x);
        j0 = 0;
        return check(c);
    }
};

// One segment, as the walking warp hands it to the others.
struct TcSegment {
    SeqRows s;
    int h, tok0, ntok;      // kv head, first token of the sequence, tokens
    int first, n;           // first block of the sequence, blocks; n < 0: there are no more segments
    int base, nb, j0;       // the tile's first unit and blocks; the segment's first block of the tile
};

struct TcShared {
    uint64_t full[TC_MOST_STAGES], empty[TC_MOST_STAGES], seg_full[TC_SEGS], seg_empty[TC_SEGS], q_full, s_full[2], p_full[2], o_full[2], o_free[2], both, half, drain;
    uint32_t tmem;
    int dead, odd;          // a wait ran out; a result is not finite
    int gone[2][8];         // per warp: a page of the segment is not there
    float ml[128][2];       // maxima and sums that one softmax group hands to the other
    float red[128][2];      // ... and the lanes of one group to one another
    float by[2][128];       // 32-bit rows: what a block's new maximum makes of the sums so far
    float unit[128];        // 32-bit rows: a row's power of two
    TcSegment seg[TC_SEGS];
    SeqRows info[TC_INFO];
    int prefix[1];          // [n + 1] units before each sequence
};

// Order in which a narrow tile's n blocks of K and V pass through the ring: K0 K1 V0 K2 V1 ... (wide: K0 V0 K1 V1 ...)
__host__ __device__ __forceinline__ int tc_slot_k(bool wide, int j) { return wide ? 2 * j : (j < 2 ? j : 2 * j - 1); }
__host__ __device__ __forceinline__ int tc_slot_v(bool wide, int j, int n) { return wide ? 2 * j + 1 : (j < n - 1 ? 2 * j + 2 : 2 * n - 1); }

// A bounded wait; the first to run out is recorded, and nobody else waits for long after it.
__device__ __forceinline__ bool tc_wait_on(TcShared &sh, uint64_t *bar, uint32_t parity, int *err, long long limit, int site) {
    if (*(volatile int *)&sh.dead) return false;
    if (mbar_wait_bounded(bar, parity, limit)) return true;
    *(volatile int *)&sh.dead = 1;
    atomicCAS(err, 0, site);
    return false;
}
__device__ __forceinline__ bool tc_wait(TcShared &sh, uint64_t *bar, uint32_t parity, const TcParams &p, int site) {
    return mbar_try_wait(bar, parity) || tc_wait_on(sh, bar, parity, &p.a.P.work[PW_ERR], p.wait_limit, site);
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
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u); }

__device__ __forceinline__ void tm_ld(uint32_t addr, uint32_t *r) {
    tm_ld32(addr, r);
    tm_wait_ld();
    pin32(r);
}

// What a softmax thread knows of its row in a segment.
struct TcRow {
    int lo, hi;        // positions that it sees
    bool mine, odd;    // the thread has a row; the segment has pages that are not there
};

// Scores of 32 positions from `pos` on (a multiple of 32) that the row does not see.
__device__ __forceinline__ void tc_hide(const AttendParams &a, const SeqRows &s, const TcRow &row, int pos, float *f) {
    uint32_t see = bits_below(row.hi - pos) & ~bits_below(row.lo - pos);   // a bit per position
    if (row.odd)
        for (int at = pos; at < min(pos + 32, s.len); at += min(a.P.page, 32))
            if (page_of(a.P, s.slot, at) < 0) see &= ~(bits_below(min(a.P.page, 32)) << (at & 31));
#pragma unroll
    for (int k = 0; k < 32; ++k)
        if (!((see >> k) & 1u)) f[k] = -INFINITY;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <int N>
__device__ __forceinline__ float tc_max(const float *f) {
    float mx[4] = {f[0], f[1], f[2], f[3]};
#pragma unroll
    for (int k = 4; k + 8 <= N; k += 8)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], f[k + 2 * i], f[k + 2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) mx[i] = fmaxf(mx[i], f[N - 4 + i]);
    return max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
}

// Two 32-bit values at a time
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 one_by_one(uint64_t x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// N scores into N / 2 columns of weights; returns the weights' sum.
template <int N, bool BF>
__device__ __forceinline__ float tc_exp16(const float *f, float c, float off, uint32_t *w) {
    const uint64_t c2 = two(c, c), off2 = two(off, off);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        const float2 x = one_by_one(fma2(two(f[k], f[k + 1]), c2, off2));
        const float p0 = ex2(x.x), p1 = ex2(x.y);
        sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], two(p0, p1));
        w[k >> 1] = pack16<BF>(p0, p1);
    }
    const float2 t = one_by_one(add2(sum[0], sum[1]));
    return t.x + t.y;
}
// (and their second parts)
__device__ __forceinline__ float tc_exp32(const float *f, float c, float off, uint32_t *hi, uint32_t *lw) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 32; k += 2) {
        // weights up to 2^14 (f16 ends at 2^16); as a factor: in the exponent it would cost the argument bits
        const float p0 = 16384.f * ex2(fmaf(f[k], c, off)), p1 = 16384.f * ex2(fmaf(f[k + 1], c, off));
        sum[(k >> 1) & 3] += p0 + p1;
        hi[k >> 1] = pack16<false>(p0, p1);
        const float2 h = unpack16(hi[k >> 1]);
        lw[k >> 1] = pack16<false>(p0 - h.x, p1 - h.y);
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// A warp's quarter of the weight columns; the other quarters, whose positions other lanes weigh, get 0.
__device__ __forceinline__ void tc_put_quarter(uint32_t to, int part, const uint32_t *w) {
    uint32_t none[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) none[i] = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (q == part) tm_st16(to + q * 16, w);
        else tm_st16(to + q * 16, none);
    }
}

// What a group's sums O at `to` become where the maximum of a row has moved.
template <int D>
__device__ __forceinline__ void tc_rescale(uint32_t to, float by) {
#pragma unroll 1
    for (int h = 0; h < D; h += 32) {
        uint32_t o[32];
        tm_ld(to + h, o);
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * by);
        tm_st32(to + h, o);
    }
}

// A block of scores (TMEM columns at `ts`) becomes 16-bit weights in the same columns.  m: what the weights refer to, l: their sum;
// `first`: there are no sums O yet.  A quarter (part >= 0): the thread weighs 32 of the positions.
// 128 scores stay in registers from their one load on: reading them again chunk by chunk costs six trips to TMEM a block instead
// of one (a 4096-row chunk over 8192 positions: 604 us).  For the same reason nothing here may spill: with this much shared memory
// there is next to no L1 for it.
template <int D, bool BF>
__device__ __forceinline__ void tc_weights16(const AttendParams &a, const SeqRows &s, const TcRow &row, uint32_t ts, uint32_t to, int part, int pos, bool first,
                                             float c, float &m, float &l) {
    const float shift = BF ? 0.f : 7.f;
    auto moved = [&](float mx) {      // a row's maximum, and what becomes of m, l and O
        mx *= c;
        const bool grow = row.mine && mx > m + TC_LAZY;      // (from -inf: with the first visible position)
        if (__any_sync(~0u, grow)) {
            const float to_m = grow ? mx : m;
            const float by = m == -INFINITY ? 0.f : ex2(m - to_m);
            m = to_m;
            l *= by;
            // (this group's products so far are complete: they were issued before the scores)
            if (!first) tc_rescale<D>(to, by);
        }
        return shift - (m == -INFINITY ? 0.f : m);
    };
    if (part >= 0) {
        uint32_t x[32], w[16];
        float *const f = (float *)x;
        const int p0 = pos + part * 32;
        tm_ld(ts + part * 32, x);
        if (row.odd || __any_sync(~0u, row.mine && (p0 < row.lo || p0 + 32 > row.hi))) tc_hide(a, s, row, p0, f);
        const float off = moved(tc_max<32>(f));
        l += tc_exp16<32, BF>(f, c, off, w);
        tc_put_quarter(ts, part, w);
    } else {
        uint32_t x[128], w[64];
        float *const f = (float *)x;
        tm_ld32(ts, x); tm_ld32(ts + 32, x + 32); tm_ld32(ts + 64, x + 64); tm_ld32(ts + 96, x + 96);
        tm_wait_ld();
        pin32(x); pin32(x + 32); pin32(x + 64); pin32(x + 96);
        if (row.odd || __any_sync(~0u, row.mine && (pos < row.lo || pos + 128 > row.hi))) {
#pragma unroll
            for (int h = 0; h < 128; h += 32) tc_hide(a, s, row, pos + h, f + h);
        }
        const float off = moved(tc_max<128>(f));
        l += tc_exp16<128, BF>(f, c, off, w);
        tm_st32(ts, w);
        tm_st32(ts + 32, w + 32);
    }
    tm_wait_st();
}

// The same for 32-bit rows: weights as two f16 parts, the maximum moves with every block; returns what that makes of the sums so far.
__device__ __forceinline__ float tc_weights32(const AttendParams &a, const SeqRows &s, const TcRow &row, uint32_t ts, int part, int pos, float c, float &m, float &l) {
    uint32_t x[32], hi[16], lw[64];
    float *const f = (float *)x;
    const int p0 = part < 0 ? pos : pos + part * 32;
    const bool edge = row.odd || __any_sync(~0u, row.mine && (p0 < row.lo || p0 + (part < 0 ? 128 : 32) > row.hi));
    float mx = -INFINITY;
    if (part >= 0) {
        tm_ld(ts + part * 32, x);
        if (edge) tc_hide(a, s, row, p0, f);
        mx = tc_max<32>(f);
    } else {
#pragma unroll
        for (int h = 0; h < 128; h += 32) {
            tm_ld(ts + h, x);
            if (edge) tc_hide(a, s, row, pos + h, f);
            mx = fmaxf(mx, tc_max<32>(f));
        }
    }
    const float to_m = fmaxf(m, mx * c);
    const float by = m == -INFINITY ? 0.f : ex2(m - to_m);
    m = to_m;
    l *= by;
    const float off = m == -INFINITY ? 0.f : -m;
    if (part >= 0) {
        l += tc_exp32(f, c, off, hi, lw);
        tc_put_quarter(ts, part, hi);
        tc_put_quarter(ts + 64, part, lw);
    } else {
#pragma unroll
        for (int h = 0; h < 128; h += 32) {
            tm_ld(ts + h, x);
            if (edge) tc_hide(a, s, row, pos + h, f);
            l += tc_exp32(f, c, off, hi, lw + h / 2);
            tm_st16(ts + h / 2, hi);
        }
        tm_st32(ts + 64, lw);   // (over scores: only once all have been read)
        tm_st32(ts + 96, lw + 32);
    }
    tm_wait_st();
    return by;
}

// Four values of a finished row.
template <int TY>
__device__ __forceinline__ void put4(void *out, long long at, float4 y) {
    if constexpr (TY == PTY_F32) *(float4 *)((float *)out + at) = y;
    else *(uint2 *)((uint16_t *)out + at) = make_uint2(pack16<TY == PTY_BF16>(y.x, y.y), pack16<TY == PTY_BF16>(y.z, y.w));
}

template <int D, int TY>
__global__ void __launch_bounds__(TC_THREADS, 1)
attend_tc_kernel(const __grid_constant__ TcParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int PANELS = D / 64;
    constexpr bool BF = TY == PTY_BF16, F32 = TY == PTY_F32;
    constexpr int PARTS = F32 ? 2 : 1;
    constexpr uint32_t TILE = TC_BLOCK * D * 2;    // bytes of a Q tile or of a block of K or V
    constexpr int STAGES = 512 / D;
    constexpr uint32_t O_COL = 256;                // TMEM columns: S0 S1 O0 O1
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *const qs = smem, *const ring = smem + 2 * TILE;
    TcShared &sh = *(TcShared *)(ring + STAGES * TILE);
    const AttendParams &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tq = 128 / a.group;

    pages_let_next();   // (attend_join_kernel waits for this grid's end)
    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 1); }
        for (int i = 0; i < TC_SEGS; ++i) { mbar_init(&sh.seg_full[i], 1); mbar_init(&sh.seg_empty[i], 10); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sh.s_full[i], 1); mbar_init(&sh.p_full[i], 4); mbar_init(&sh.o_full[i], 1); mbar_init(&sh.o_free[i], 4); }
        mbar_init(&sh.q_full, 8);
        mbar_init(&sh.both, 8);
        mbar_init(&sh.half, 4);
        mbar_init(&sh.drain, 1);
        sh.dead = sh.odd = 0;
        for (int i = 0; i < 16; ++i) sh.gone[i >> 3][i & 7] = 0;
        fence_mbar_init();
    }
    if (warp == 9) tm_alloc(&sh.tmem, 512);
    if (tid == 256) {
        tma_prefetch_map(&kmap);
        tma_prefetch_map(&vmap);
    }
    pages_wait_front();
    for (int i = tid; i < min(a.B.n, TC_INFO); i += TC_THREADS) sh.info[i] = batch_seq(a.P, a.B, i);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int cta = blockIdx.x;
    const uint32_t tmem = sh.tmem;
    const uint32_t idesc_qk = tc_idesc(BF, 128, 128, false), idesc_pv = tc_idesc(BF, 128, D, true);
    int ring0 = 0, n_seg = 0;             // ring entries before this segment, segments so far
    bool ok = true;
    auto segment = [&]() -> const TcSegment & { return sh.seg[n_seg % TC_SEGS]; };
    auto seg_wait = [&] { return tc_wait(sh, &sh.seg_full[n_seg % TC_SEGS], (n_seg / TC_SEGS) & 1, p, 10); };

    // Register shares of the three groups of four warps: 2 x 208 + 80 <= 3 x 168, what the block was launched with.
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp == 8) {
            // ------------------------------------------------------------------ TMA
            const int box_shift = max(0, 7 - a.P.shift), boxes = 1 << box_shift, rows = min(a.P.page, TC_BLOCK), ahead = 32 >> box_shift;
            const int box = lane / PANELS, panel = lane % PANELS;
            int filled = 0;
            while ((ok = __all_sync(~0u, seg_wait()))) {
                const TcSegment &x = segment();
                const int n = x.n;
                if (n < 0) break;
                const bool wide = x.ntok > tq;
                // page numbers of `ahead` blocks from block from[.] on, one a lane; K and V move through them apart.  A page that does
                // not exist (or lies behind the sequence) is asked for outside the pool: zeros arrive
                int from[2] = {INT_MIN, INT_MIN}, pages[2];
#pragma unroll 1
                for (int e = 0; e < 2 * n; ++e) {
                    // entry e of the segment: a block of K or of V
                    bool is_v;
                    int j;
                    if (wide) { is_v = e & 1; j = e >> 1; }
                    else if (e < 2 && e < n) { is_v = false; j = e; }
                    else if (e == 2 * n - 1) { is_v = true; j = n - 1; }
                    else { is_v = !(e & 1); j = is_v ? (e - 2) >> 1 : (e + 1) >> 1; }
                    const int pos = (x.first + j) * TC_BLOCK;
                    const int idx = ring0 + e, st = idx % STAGES;
                    int pg = 0;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv)
                        if (kv == (int)is_v) {
                            if (from[kv] == INT_MIN || j >= from[kv] + ahead) {
                                from[kv] = j;
                                const int at = pos + (lane >> box_shift) * TC_BLOCK + (lane & (boxes - 1)) * rows;
                                pages[kv] = at < x.s.len ? page_of(a.P, x.s.slot, at) : -1;
                                if (pages[kv] < 0) pages[kv] = a.P.n_pages;
                            }
                            pg = __shfl_sync(~0u, pages[kv], ((j - from[kv]) << box_shift) + min(box, boxes - 1));
                        }
                    ok = __all_sync(~0u, tc_wait(sh, &sh.empty[st], ((idx / STAGES) & 1) ^ 1, p, 1));
                    if (!ok) break;
                    filled = idx + 1;
                    uint8_t *dst = ring + st * TILE;
                    if (lane == 0) mbar_arrive_expect_tx(&sh.full[st], TILE);
                    __syncwarp();
                    if (box < boxes)
                        tma_load_4d(dst + panel * (TC_BLOCK * 128) + box * rows * 128, is_v ? &vmap : &kmap, panel * 64, (pos + box * rows) & (a.P.page - 1), x.h, pg,
                                    &sh.full[st]);
                }
                if (!ok) break;
                ring0 += 2 * n;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.seg_empty[n_seg % TC_SEGS]);
                ++n_seg;
            }
            // every copy that was asked for has arrived before the block ends
            for (int idx = max(0, filled - STAGES); idx < filled; ++idx)
                (void)mbar_wait_bounded(&sh.full[idx % STAGES], (idx / STAGES) & 1, TC_DRAIN);
        } else if (warp == 9) {
            // -------------------------------------------------------- tensor instructions: issued by one thread of a warp that stays
            // together, so that their operands are the warp's and not the thread's (one thread alone took 85 cycles for each)
            const bool leader = elect_one();
            uint32_t ph_q = 0, ph_p = 0;
            const uint32_t q_addr = smem_u32(qs), r_addr = smem_u32(ring);
            while ((ok = __all_sync(~0u, seg_wait()))) {
                const int n = __shfl_sync(~0u, segment().n, 0);
                if (n < 0) break;
                const bool wide = !F32 && __shfl_sync(~0u, segment().ntok, 0) > tq;
                __syncwarp();
                if (leader) mbar_arrive(&sh.seg_empty[n_seg % TC_SEGS]);
                ++n_seg;
                if (n == 0) continue;
                if (!(ok = __all_sync(~0u, tc_wait(sh, &sh.q_full, ph_q, p, 4)))) break;
                ph_q ^= 1;
                // Step i is the product with V of one group and the scores of its next block: wide, both groups for every block (group
                // i & 1, block i / 2); narrow, the groups in turn (block i).  The first two steps have scores only.
                const int steps = wide ? 2 * n : n;
#pragma unroll 1
                for (int i = -2; i < steps; ++i) {
                    const int w = i & 1;
                    const bool last = i + 2 >= steps, both = !wide || w;   // both: no other group needs the block any more
                    if (i >= 0) {
                        const int v = ring0 + tc_slot_v(wide, wide ? i >> 1 : i, n), st = v % STAGES;
                        if (!(ok = __all_sync(~0u, tc_wait(sh, &sh.full[st], (v / STAGES) & 1, p, 2) && tc_wait(sh, &sh.p_full[w], ph_p >> w & 1, p, 3)))) break;
                        ph_p ^= 1u << w;
                        tc_fence_after();
                        if (leader) {
                            const uint64_t va = tc_desc(r_addr + st * TILE, TC_BLOCK * 128);
                            const uint32_t o = tmem + O_COL + w * D, pw = tmem + w * 128;
                            const bool add = !F32 && i > 1;
#pragma unroll
                            for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                                for (int k = 0; k < TC_BLOCK / 16; ++k)
                                    tc_mma_ts(o, pw + part * 64 + k * 8, va + (uint64_t)(k * 2048 >> 4), idesc_pv, add || part < PARTS - 1 || k > 0);
                            if (both) tc_commit(&sh.empty[st]);
                            if (F32 || last) tc_commit(&sh.o_full[w]);
                        }
                    }
                    if (!last) {
                        const int kn = ring0 + tc_slot_k(wide, wide ? (i + 2) >> 1 : i + 2), st = kn % STAGES;
                        if (!(ok = __all_sync(~0u, tc_wait(sh, &sh.full[st], (kn / STAGES) & 1, p, 2)))) break;
                        tc_fence_after();
                        if (leader) {
                            const uint64_t qa = tc_desc(q_addr + (wide ? w * TILE : 0), 16), ka = tc_desc(r_addr + st * TILE, 16);
                            const uint32_t d = tmem + w * 128;
                            // (low parts first: a sum is truncated where it is, and theirs are small)
#pragma unroll
                            for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                                for (int k = 0; k < D / 16; ++k) {
                                    const uint32_t off = (k >> 2) * (TC_BLOCK * 128) + (k & 3) * 32;
                                    tc_mma_ss(d, qa + (uint64_t)((part * TILE + off) >> 4), ka + (uint64_t)(off >> 4), idesc_qk, part < PARTS - 1 || k > 0);
                                }
                            tc_commit(&sh.s_full[w]);
                            if (both) tc_commit(&sh.empty[st]);
                        }
                    }
                }
                if (!ok) break;
                ring0 += 2 * n;
            }
            if (leader) {
                tc_commit(&sh.drain);
                (void)mbar_wait_bounded(&sh.drain, 0, TC_DRAIN);
            }
        } else if (warp == 10) {
            // ------------------------------------------------------- units of every sequence, their running sum, the CTA's segments
            TcBatch g(a, sh.info);
            const int seqs = a.B.n;
            auto count = [&](int i) {   // units of sequence i
                if (i >= seqs) return 0;
                TcTile x;
                x.s = g.seq(i);
                int units = 0;
#pragma unroll 1
                for (x.t = 0; x.t * g.step < x.s.rows; ++x.t) {
                    tc_span(g, x);
                    units = min(units + x.units(), TC_MOST);
                }
                return (int)min((long long)units * a.P.kv, (long long)TC_MOST);
            };
            if (seqs <= 32) {   // (a small batch)
                g.open = 0;
                int units = count(lane);
                for (int o = 16; o; o >>= 1) units = min(units + __shfl_xor_sync(~0u, units, o), TC_MOST);
                if (units >= TC_FEW * p.n_ctas) g.open = TC_OPEN;
            }
            int total = 0;
            if (lane == 0) sh.prefix[0] = 0;
#pragma unroll 1
            for (int i0 = 0; i0 < seqs; i0 += 32) {   // a lane a sequence
                const int i = i0 + lane;
                int units = count(i);
                if (seqs > 1)
                    for (int o = 1; o < 32; o <<= 1) {
                        const int y = __shfl_up_sync(~0u, units, o);
                        if (lane >= o) units = min(units + y, TC_MOST);
                    }
                units = min(total + units, TC_MOST);
                if (i < seqs) sh.prefix[i + 1] = units;
                total = __shfl_sync(~0u, units, seqs > 1 ? 31 : 0);
            }
            __syncwarp();
            // (offsets that overlap could claim more rows than there are: such a batch is left alone)
            if (total >= TC_MOST) total = 0;
            const int per = max((int)(((long long)total + p.n_ctas - 1) / p.n_ctas), TC_MIN_UNITS);
            // lane 0 finds where the range begins, lane 1 where it ends
            TcWalk wk;
            {
                const long long u = (long long)(cta + (lane & 1)) * per;
                wk.j0 = tc_cut(g, sh.prefix, total, (int)(u < total ? u : total), wk.x);
                wk.e_seq = __shfl_sync(~0u, wk.x.seq, 1);
                wk.e_t = __shfl_sync(~0u, wk.x.t, 1);
                wk.e_h = __shfl_sync(~0u, wk.x.h, 1);
                wk.e_block = __shfl_sync(~0u, wk.j0, 1);
            }
            if (lane == 0) {
                int cuts = 0;
                bool more = wk.check(g);
#pragma unroll 1
                for (;;) {
                    const int at = n_seg % TC_SEGS;
                    if (!tc_wait(sh, &sh.seg_empty[at], ((n_seg / TC_SEGS) & 1) ^ 1, p, 11)) break;
                    TcSegment &x = sh.seg[at];
                    x.s = wk.x.s;
                    x.h = wk.x.h; x.tok0 = wk.x.tok0; x.ntok = wk.x.ntok;
                    x.first = wk.x.k0 + wk.j0;
                    x.n = more ? wk.j1 - wk.j0 : -1;
                    x.base = wk.x.base; x.nb = wk.x.nb; x.j0 = wk.j0;
                    mbar_arrive(&sh.seg_full[at]);
                    if (!more) break;
                    // the first of a cut tile's pieces says how many follow: the cuts that stay inside the tile
                    if (wk.j0 == 0 && wk.j1 < wk.x.nb) {
                        // (block >= edge and block <= nb - edge, in units)
                        const int edge = tc_edge(g, wk.x), from = wk.x.base + wk.x.opening;
                        const int lo = from + edge * wk.x.per_block, hi = from + (wk.x.nb - edge + 1) * wk.x.per_block - 1;
                        int *mt = p.meta + cta * 8;
                        cuts = hi / per - (lo - 1) / per;
                        mt[1] = wk.x.s.first + wk.x.tok0; mt[2] = wk.x.ntok; mt[3] = wk.x.h; mt[4] = !F32 && wk.x.ntok > tq;
                    }
                    ++n_seg;
                    more = wk.next(g);
                }
                p.meta[cta * 8] = cuts;
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int w = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // TMEM lane base of the warp, in the address's upper half
        const bool flip = a.scale_log2 < 0.f;                // a negative scale turns the queries round
        const float c0 = fmaxf(fabsf(a.scale_log2), 1e-30f); // (a scale of 0: hidden positions still get 2^-inf)
        uint32_t ph_s = 0, ph_b = 0, ph_o = 0, ph_both = 0, ph_half = 0;
        auto wait = [&](uint64_t *bar, uint32_t parity, int site) { return ok = __all_sync(~0u, tc_wait(sh, bar, parity, p, site)); };
        // both groups, or the four warps of one, wait for one another (as bounded as any other wait)
        auto meet = [&](uint64_t *bar, uint32_t &ph, int site) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
            const bool k = wait(bar, ph, site);
            ph ^= 1;
            return k;
        };
        while (wait(&sh.seg_full[n_seg % TC_SEGS], (n_seg / TC_SEGS) & 1, 10)) {
            const TcSegment &x = segment();
            const int n = x.n, k_first = x.first;
            if (n < 0) break;
            const bool wide = !F32 && x.ntok > tq;
            const bool whole = n == x.nb;
            // Up to 32 rows are held four times over and every copy weighs a quarter of a block's positions: four warps then work on
            // what one would.
            const int held = min(x.ntok, tq) * a.group;
            const int each = wide || held > 32 ? 128 : 32, reps = 128 / each;
            const int rr = r & (each - 1), part = reps > 1 ? r >> 5 : -1;   // the thread's row and quarter
            const int tok = x.tok0 + (wide ? w * tq : 0) + rr / a.group;
            TcRow row;
            row.mine = rr < tq * a.group && tok < x.tok0 + x.ntok;
            const int out_row = x.s.first + tok, head = x.h * a.group + rr % a.group;
            row.lo = row.hi = 0;
            if (row.mine) row_span(a, x.s.len, x.s.len - x.s.rows + tok, row.lo, row.hi);
            // pages that are not there: looked for once a segment
            bool odd = false;
            #pragma unroll 1
            for (int c = (k_first * TC_BLOCK >> a.P.shift) + tid; (c << a.P.shift) < min((k_first + n) * TC_BLOCK, x.s.len); c += 256)
                odd |= page_of(a.P, x.s.slot, c << a.P.shift) < 0;

            // ---- queries into shared memory, four loads at a time; the first are on their way before the groups meet
            const int q_rows = wide && w ? (x.ntok - tq) * a.group : held;
            const long long q_tok = x.s.first + x.tok0 + (wide ? w * tq : 0);
            uint8_t *const q_tile = qs + (wide ? w * TILE : 0);
            constexpr int E = F32 ? D / 32 : 8;              // values of a load: a row per warp, or 16 bytes
            const int q_units = n == 0 ? 0 : (F32 ? q_rows : q_rows * (D / 8)), q_step = F32 ? 8 : (wide ? 128 : 256);
            const int q_me = F32 ? warp : (wide ? r : tid);
            uint4 qv[4];
            auto q_load = [&](int i0) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int i = i0 + u * q_step;
                    if (i >= q_units) break;
                    const int rw = F32 ? i : i / (D / 8), d = F32 ? lane * E : (i % (D / 8)) * 8;
                    const long long at = (q_tok + rw / a.group) * a.qs[0] + (long long)(x.h * a.group + rw % a.group) * a.qs[1] + d;
                    if constexpr (!F32) qv[u] = *(const uint4 *)((const uint16_t *)a.q + at);
                    else if constexpr (D == 128) qv[u] = *(const uint4 *)((const float *)a.q + at);
                    else *(uint2 *)&qv[u] = *(const uint2 *)((const float *)a.q + at);
                }
            };
            q_load(q_me);
            if (__any_sync(~0u, odd) && lane == 0) sh.gone[n_seg & 1][warp] = 1;
            if (!meet(&sh.both, ph_both, 12)) break;   // (both groups have left the segment before)
            row.odd = false;
            for (int i = 0; i < 8; ++i) row.odd |= sh.gone[n_seg & 1][i] != 0;
            if (lane == 0) sh.gone[(n_seg & 1) ^ 1][warp] = 0;
            if (n > 0) {
#pragma unroll 1
                for (int i0 = q_me; i0 < q_units; i0 += 4 * q_step) {
                    if (i0 > q_me) q_load(i0);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int i = i0 + u * q_step;
                        if (i >= q_units) break;
                        if constexpr (F32) {
                            const float *v = (const float *)&qv[u];
                            float mx = 0.f;
#pragma unroll
                            for (int e = 0; e < E; ++e) mx = fmaxf(mx, fabsf(v[e]));
                            for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
                            // the row's largest value lands in [2^13, 2^14): what is 2^-27 of it still has 11 bits
                            const int ex = mx < INFINITY ? max((int)(__float_as_uint(mx) >> 23) - 127, -100) : 0;
                            const float by = __uint_as_float((uint32_t)(127 + 13 - ex) << 23) * (flip ? -1.f : 1.f);
                            if (lane == 0) sh.unit[i] = __uint_as_float((uint32_t)max(127 - 13 + ex, 1) << 23);
#pragma unroll
                            for (int e = 0; e < E; e += 2) {
                                const float u0 = v[e] * by, u1 = v[e + 1] * by;
                                const uint32_t hi = pack16<false>(u0, u1);
                                const float2 h = unpack16(hi);
                                const uint32_t lw = pack16<false>(u0 - h.x, u1 - h.y);
                                const int d = lane * E + e;
                                for (int c = 0; c < reps; ++c) {
                                    uint8_t *at = q_tile + (d >> 6) * (TC_BLOCK * 128) + sw128(i + c * each, (d >> 3) & 7) + (d & 7) * 2;
                                    *(uint32_t *)at = hi;
                                    *(uint32_t *)(at + TILE) = lw;
                                }
                            }
                        } else {
                            uint4 v = qv[u];
                            if (flip) { v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u; }
                            const int rw = i / (D / 8), ch = i % (D / 8);
                            for (int c = 0; c < reps; ++c) *(uint4 *)(q_tile + (ch >> 3) * (TC_BLOCK * 128) + sw128(rw + c * each, ch & 7)) = v;
                        }
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.q_full);
            }

            // ---- blocks
            float m = -INFINITY, l = 0.f;   // m: of the scaled scores, what the weights refer to
            const bool warp_mine = __any_sync(~0u, row.mine);
            // What lies behind the sequence in its last page takes part in the product with weight 0: it may not be NaN.
            auto clear_tail = [&](int j, int pos) {
                const int idx = ring0 + tc_slot_v(wide, j, n);
                if (!wait(&sh.full[idx % STAGES], (idx / STAGES) & 1, 6)) return false;
                if (pos + r >= x.s.len) {
                    uint8_t *v = ring + (idx % STAGES) * TILE + r * 128;
#pragma unroll
                    for (int k = 0; k < PANELS * 8; ++k) *(uint4 *)(v + (k >> 3) * (TC_BLOCK * 128) + (k & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
                return true;
            };
            const int slot = 2 * cta + (x.j0 == 0 ? 1 : 0);
            float *const scratch = (float *)qs;   // [128][D], once a segment's queries have done their work: 16-byte chunks swizzled by the row
            // A narrow tile's results go through the scratch: 32 values of the thread's own row, relative to `top` with the weights' sum lt.
            auto put_scratch = [&](int h, const float *f) {
#pragma unroll
                for (int k = 0; k < 32; k += 4) ((float4 *)scratch)[r * (D / 4) + (((h + k) / 4) ^ (rr & (D / 4 - 1)))] = make_float4(f[k], f[k + 1], f[k + 2], f[k + 3]);
            };
            // ... and the 128 threads of a group join the copies and write the rows, or a piece of them.
            auto join_copies = [&](float top_, float lt_) {
                sh.red[r][0] = top_;
                sh.red[r][1] = lt_;
                if (!meet(&sh.half, ph_half, 13)) return;
#pragma unroll 1
                for (int i = r; i < held * (D / 4); i += 128) {
                    const int rw = i / (D / 4), ch = i % (D / 4);
                    float top = -INFINITY, lt = 0.f;
#pragma unroll 1
                    for (int q = 0; q < reps; ++q) top = fmaxf(top, sh.red[q * each + rw][0]);
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                    for (int q = 0; q < reps; ++q) {
                        const float mq = sh.red[q * each + rw][0], b = mq == -INFINITY ? 0.f : ex2(mq - top);
                        const float4 o = ((const float4 *)scratch)[(q * each + rw) * (D / 4) + (ch ^ (rw & (D / 4 - 1)))];
                        lt += sh.red[q * each + rw][1] * b;
                        y.x = fmaf(o.x, b, y.x); y.y = fmaf(o.y, b, y.y); y.z = fmaf(o.z, b, y.z); y.w = fmaf(o.w, b, y.w);
                    }
                    if (whole) {
                        const float inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);
                        y.x *= inv; y.y *= inv; y.z *= inv; y.w *= inv;
                        if (!(fabsf(y.x) + fabsf(y.y) + fabsf(y.z) + fabsf(y.w) < INFINITY)) sh.odd = 1;   // (see attend_join_kernel)
                        put4<TY>(a.out, (long long)(x.s.first + x.tok0 + rw / a.group) * a.os[0] + (long long)(x.h * a.group + rw % a.group) * a.os[1] + ch * 4, y);
                    } else {
                        *(float4 *)(p.part + ((long long)slot * p.ws_rows + rw) * D + ch * 4) = y;
                        if (ch == 0) *(float2 *)(p.ml + ((long long)slot * p.ws_rows + rw) * 2) = make_float2(top, lt);
                    }
                }
            };

            if constexpr (F32) {
                if (!meet(&sh.both, ph_both, 14)) break;   // the rows' powers of two are written
                const float c = c0 * sh.unit[rr];
                if (w == 0) {
                    for (int j = 0; j < n && ok; ++j) {
                        const int b = j & 1, pos = (k_first + j) * TC_BLOCK;
                        if (!wait(&sh.s_full[b], ph_b >> b & 1, 5)) break;
                        // (the sums of the block before last have been taken: its O buffer and its factor are free)
                        if (!wait(&sh.o_free[b], (ph_b >> b & 1) ^ 1, 9)) break;
                        ph_b ^= 1 << b;
                        tc_fence_after();
                        if (warp_mine) sh.by[b][r] = tc_weights32(a, x.s, row, tmem + lanes + b * 128, part, pos, c, m, l);
                        if (pos + TC_BLOCK > x.s.len && !clear_tail(j, pos)) break;
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.p_full[b]);
                    }
                    sh.ml[r][0] = m;
                    sh.ml[r][1] = l;
                    if (!ok || !meet(&sh.both, ph_both, 15)) break;
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
                                tm_ld(tmem + lanes + O_COL + b * D + h, o);
#pragma unroll
                                for (int k = 0; k < 32; ++k) acc[h + k] = fmaf(acc[h + k], by, __uint_as_float(o[k]));
                            }
                        }
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.o_free[b]);
                    }
                    if (!ok || !meet(&sh.both, ph_both, 15)) break;
                    if (row.mine) {
#pragma unroll
                        for (int h = 0; h < D; h += 32) put_scratch(h, acc + h);
                    }
                    join_copies(sh.ml[r][0], sh.ml[r][1]);
                }
            } else {
                const uint32_t ts = tmem + lanes + w * 128, to = tmem + lanes + O_COL + w * D;
                const int cnt = wide ? n : (n - w + 1) >> 1;
                for (int i = 0; i < cnt && ok; ++i) {
                    const int j = wide ? i : 2 * i + w, pos = (k_first + j) * TC_BLOCK;
                    if (!wait(&sh.s_full[w], ph_s, 5)) break;
                    ph_s ^= 1;
                    tc_fence_after();
                    if (warp_mine) tc_weights16<D, BF>(a, x.s, row, ts, to, part, pos, i == 0, c0, m, l);
                    if (pos + TC_BLOCK > x.s.len && !clear_tail(j, pos)) break;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.p_full[w]);
                }
                // ---- the segment's result
                float m1 = -INFINITY, l1 = 0.f;
                const bool two = !wide && n > 1;
                if (!wide) {
                    if (w == 1) { sh.ml[r][0] = m; sh.ml[r][1] = l; }
                    if (!ok || !meet(&sh.both, ph_both, 16)) break;
                    if (w == 0) { m1 = sh.ml[r][0]; l1 = sh.ml[r][1]; }
                }
                if (!ok) break;
                if (n > 0 && (wide || w == 0) && !wait(&sh.o_full[w], ph_o >> w & 1, 7)) break;
                if (two && w == 0 && !wait(&sh.o_full[1], ph_o >> 1, 8)) break;
                ph_o ^= (n > 0 ? 1u : 0u) | ((wide ? n > 0 : n > 1) ? 2u : 0u);
                tc_fence_after();
                if (wide || w == 0) {
                    const float top = fmaxf(m, m1);
                    // (weights that refer to -inf are all 0, and their O holds zeros)
                    const float b0 = m == -INFINITY ? 0.f : ex2(m - top), b1 = m1 == -INFINITY ? 0.f : ex2(m1 - top);
                    const float lt = l * b0 + l1 * b1, inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt), u = wide && whole ? inv : b0;
                    const long long ws_at = (long long)slot * p.ws_rows + w * 128 + r;
                    if (warp_mine) {
#pragma unroll 1
                        for (int h = 0; h < D; h += 32) {
                            uint32_t o[32];
                            float *f = (float *)o;
                            if (n > 0) {
                                tm_ld(to + h, o);
                            } else {
#pragma unroll
                                for (int k = 0; k < 32; ++k) o[k] = 0;
                            }
#pragma unroll
                            for (int k = 0; k < 32; ++k) f[k] *= u;
                            if (two) {
                                uint32_t o1[32];
                                tm_ld(to + D + h, o1);
#pragma unroll
                                for (int k = 0; k < 32; ++k) f[k] = fmaf(__uint_as_float(o1[k]), b1, f[k]);
                            }
                            if (!row.mine) continue;
                            if (!wide) {
                                put_scratch(h, f);
                            } else if (whole) {
                                float size = 0.f;
#pragma unroll
                                for (int k = 0; k < 32; ++k) size += fabsf(f[k]);
                                if (!(size < INFINITY)) sh.odd = 1;   // (see attend_join_kernel)
                                uint16_t *out = (uint16_t *)a.out + out_row * a.os[0] + head * a.os[1] + h;
#pragma unroll
                                for (int k = 0; k < 32; k += 8)
                                    *(uint4 *)(out + k) = make_uint4(pack16<BF>(f[k], f[k + 1]), pack16<BF>(f[k + 2], f[k + 3]), pack16<BF>(f[k + 4], f[k + 5]),
                                                                     pack16<BF>(f[k + 6], f[k + 7]));
                            } else {
                                float *pt = p.part + ws_at * D + h;
#pragma unroll
                                for (int k = 0; k < 32; k += 4) *(float4 *)(pt + k) = make_float4(f[k], f[k + 1], f[k + 2], f[k + 3]);
                            }
                        }
                        if (wide && !whole && row.mine) *(float2 *)(p.ml + ws_at * 2) = make_float2(top, lt);
                    }
                    if (!wide) join_copies(top, lt);
                }
            }
            ring0 += 2 * n;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.seg_empty[n_seg % TC_SEGS]);
            ++n_seg;
            if (!ok) break;
        }
    }

    // ---- close: no copy and no tensor instruction may be in flight when the CTA ends
    __syncthreads();
    if (tid == 0) p.meta[cta * 8 + 6] = sh.odd;
    if (warp == 9) {
        tc_fence_after();
        tm_dealloc(tmem, 512);
    }
}

// Row t's head hd over again, position by position.  The warp that calls it is the last to have stored the row.
template <int D, typename T, typename C>
__device__ __noinline__ void attend_mend(const AttendParams &a, int t, int hd, int lane) {
    const int i = batch_find(a.B, t);
    if (i < 0) return;
    const SeqRows s = batch_seq(a.P, a.B, i);
    __syncwarp();
    attend_row<D, T, C>(a, s, t, hd, lane);
}

// The heads of row t that whole tiles have left not finite.  Rows of cut tiles are being stored by this very grid: who joins
// them mends them.
template <int D, typename T, typename C>
__device__ __noinline__ void attend_mend_whole(const TcParams &p, int t, int warp, int lane) {
    constexpr int E = D / 32;
    const AttendParams &a = p.a;
    for (int hd = warp; hd < a.heads; hd += 8) {
        bool cut = false;
        for (int c = lane; c < p.n_ctas; c += 32) {
            const int4 mt = *(const int4 *)(p.meta + c * 8);
            cut |= mt.x > 0 && t >= mt.y && t < mt.y + mt.z && mt.w == hd / a.group;
        }
        if (__any_sync(~0u, cut)) continue;
        const T *o = (const T *)a.out + t * a.os[0] + hd * a.os[1] + lane * E;
        float size = 0.f;
        for (int e = 0; e < E; ++e) size += fabsf(to_f32(o[e]));
        if (__any_sync(~0u, !(size < INFINITY))) attend_mend<D, T, C>(a, t, hd, lane);
    }
}

// Merges the pieces of a cut tile: block c those of the tile whose first piece CTA c has left.  Piece 0 lies in slot 1 of CTA c,
// the others in slot 0 of the CTAs behind it.  A warp per row, in the order of the pieces.
// An infinity or NaN in V at a position that some rows of a tile do not see has met their weight of 0 in the product.  Such
// rows show it by not being finite; they are done over here, position by position: a row of a cut tile by the warp that has
// joined it, a row of a whole tile, which the kernel in front has stored, by any.
template <int D, int TY>
__global__ void __launch_bounds__(256, 3) attend_join_kernel(const __grid_constant__ TcParams p) {
    constexpr int LANES = D / 4, ROWS = 32 / LANES;   // lanes a row, four values each; rows a warp
    typedef typename Elem<TY>::T T;
    typedef typename Elem<TY == PTY_BF16 ? PTY_BF16 : PTY_F16>::T C;
    const AttendParams &a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pages_let_next();
    pages_wait_front();
    const int4 mt = *(const int4 *)(p.meta + blockIdx.x * 8);
    const int more = mt.x, row0 = mt.y, ntok = mt.z, h = mt.w;
    int odd = 0;
    uint32_t bad = 0;   // rows of the warp that are not finite: bit iteration * ROWS + sub (four iterations at most: 32 rows or fewer a block)
    for (int i = threadIdx.x; i < p.n_ctas; i += 256) odd |= p.meta[i * 8 + 6];
    if (more > 0 && more < p.n_ctas - (int)blockIdx.x) {
        const int tq = 128 / a.group;
        const bool wide = p.meta[blockIdx.x * 8 + 4];
        const int n_rows = wide ? 128 + (ntok - tq) * a.group : ntok * a.group, sub = lane / LANES, ch = lane % LANES;
        const int r_first = (blockIdx.y * 8 + warp) * ROWS, r_step = 8 * ROWS * gridDim.y;
#pragma unroll 1
        for (int r0 = r_first, it = 0; r0 < n_rows; r0 += r_step, it += ROWS) {
            const int r = min(r0 + sub, n_rows - 1), rr = r & 127, tok = (r >= 128 ? tq : 0) + rr / a.group;
            const bool mine = r0 + sub < n_rows && rr < tq * a.group;
            auto at = [&](int piece) { return (2 * ((int)blockIdx.x + piece) + (piece == 0)) * p.ws_rows + r; };
            float top = -INFINITY, l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = ch; i <= more; i += LANES) top = fmaxf(top, p.ml[(long long)at(i) * 2]);
#pragma unroll
            for (int x = LANES / 2; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
#pragma unroll 1
            for (int i0 = 0; i0 <= more; i0 += LANES) {
                float b = 0.f;   // the lane's piece: its weight
                if (i0 + ch <= more) {
                    const float2 ml = *(const float2 *)(p.ml + (long long)at(i0 + ch) * 2);
                    if (ml.x != -INFINITY) b = ex2(ml.x - top);
                    l = fmaf(b, ml.y, l);
                }
                const int n = min(LANES, more + 1 - i0);
                const float *src = p.part + (long long)at(i0) * D + ch * 4;
                const long long step = 2ll * p.ws_rows * D, jump = i0 == 0 ? step - (long long)p.ws_rows * D : step;   // (piece 0 lies in slot 1)
#pragma unroll 1
                for (int i = 0; i < n; i += 8) {   // eight pieces' loads at a time
                    float4 v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (i + k < n) v[k] = *(const float4 *)(src + (i + k == 0 ? 0 : jump + (i + k - 1) * step));
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float bi = __shfl_sync(~0u, b, (sub * LANES) | ((i + k) & (LANES - 1)));
                        if (i + k < n) { o.x = fmaf(bi, v[k].x, o.x); o.y = fmaf(bi, v[k].y, o.y); o.z = fmaf(bi, v[k].z, o.z); o.w = fmaf(bi, v[k].w, o.w); }
                    }
                }
            }
#pragma unroll
            for (int x = LANES / 2; x; x >>= 1) l += __shfl_xor_sync(~0u, l, x);
            const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
            o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
            const int row = row0 + tok, head = h * a.group + rr % a.group;
            if (mine) put4<TY>(a.out, row * a.os[0] + head * a.os[1] + ch * 4, o);
            const uint32_t is = __ballot_sync(~0u, mine && !(fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w) < INFINITY));
#pragma unroll
            for (int i = 0; i < ROWS; ++i) bad |= (is >> (i * LANES) & (~0u >> (32 - LANES)) ? 1u : 0u) << (it + i);
        }
#pragma unroll 1
        for (; bad; bad &= bad - 1) {
            const int i = __ffs(bad) - 1, r = r_first + i / ROWS * r_step + i % ROWS, rr = r & 127;
            attend_mend<D, T, C>(a, row0 + (r >= 128 ? tq : 0) + rr / a.group, h * a.group + rr % a.group, lane);
        }
    }
    if (__syncthreads_or(odd))
        for (int t = blockIdx.y * gridDim.x + blockIdx.x; t < a.B.rows; t += gridDim.x * gridDim.y) attend_mend_whole<D, T, C>(p, t, warp, lane);
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
    const TcBatch g(p, nullptr);
    s.rows = p.B.rows > g.tq ? (g.step > g.tq ? 256 : 128) : p.B.rows * p.group;
    s.meta = ((size_t)n_sm * 8 * 4 + 255) / 256 * 256;
    s.ml = ((size_t)n_sm * 2 * s.rows * 2 * 4 + 255) / 256 * 256;
    s.part = (size_t)n_sm * 2 * s.rows * p.P.dim * 4;
    return s;
}

template <int D>
constexpr int tc_smem() {
    constexpr int n = 1024 + (2 + 512 / D) * TC_BLOCK * D * 2 + (int)sizeof(TcShared) + 4 * PAGES_MAX_BATCH;
    static_assert(n <= 232448, "shared memory of a block");
    return n;
}

template <int D, int TY>
cudaError_t tc_prepare() { return cudaFuncSetAttribute(attend_tc_kernel<D, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize, tc_smem<D>()); }

template <int D, int TY>
cudaError_t launch_tc(const AttendParams &p, int n_sm, void *ws, long long wait_limit, cudaStream_t st, int *launches) {
    constexpr int smem = tc_smem<D>();
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
    cudaError_t e = launch_front(attend_tc_kernel<D, TY>, dim3(n_sm), TC_THREADS, smem, st, q, km, vm);
    if (e != cudaSuccess) return e;
    e = launch_front(attend_join_kernel<D, TY>, dim3(n_sm, (z.rows + 31) / 32), 256, 0, st, q);
    if (e != cudaSuccess) return e;
    *launches += 2;
    return cudaGetLastError();
}

}  // namespace

cudaError_t prepare_attend() {
    for (cudaError_t e : {tc_prepare<64, PTY_F32>(), tc_prepare<64, PTY_F16>(), tc_prepare<64, PTY_BF16>(), tc_prepare<128, PTY_F32>(),
                          tc_prepare<128, PTY_F16>(), tc_prepare<128, PTY_BF16>()})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}

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
