// Attention of new rows over a paged KV cache.
#include "pages.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

// o = sum_j p_j v_j / sum_j p_j, p_j = 2^(scale_log2 q.k_j - m), m the running maximum: one pass over the positions.
// One warp per (row, head), the head's dimensions over the lanes.  A position that is not visible is not read at all,
// so nothing that it holds (infinities, NaN, what an earlier sequence left) reaches a result.
template <int D, typename T, typename C>
__device__ void attend_row(const AttendParams &p, const SeqRows &s, int t, int h, int lane) {
    constexpr int E = D / 32;
    const int kvh = h / p.group;
    const int pos = s.len - s.rows + (t - s.first);
    const int hi = p.causal ? min(pos + 1, s.len) : s.len;
    const int lo = p.window ? max(0, pos - p.window + 1) : 0;
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

template <int D, int TY, bool BF>
__global__ void __launch_bounds__(256) attend_rows_kernel(const __grid_constant__ AttendParams p) {
    typedef typename Elem<TY>::T T;
    typedef typename Elem<BF ? PTY_BF16 : PTY_F16>::T C;
    const long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int t = (int)(u / p.heads), h = (int)(u % p.heads);
    if (t >= p.B.rows) return;
    const int i = batch_find(p.B, t);
    if (i < 0) return;
    attend_row<D, T, C>(p, batch_seq(p.P, p.B, i), t, h, threadIdx.x & 31);
}

template <int D>
void launch_rows(const AttendParams &p, unsigned grid, cudaStream_t st) {
    if (p.ty == PTY_F32) attend_rows_kernel<D, PTY_F32, false><<<grid, 256, 0, st>>>(p);
    else if (p.ty == PTY_F16) attend_rows_kernel<D, PTY_F16, false><<<grid, 256, 0, st>>>(p);
    else attend_rows_kernel<D, PTY_BF16, true><<<grid, 256, 0, st>>>(p);
}

}  // namespace

cudaError_t launch_attend(const AttendParams &p, int, cudaStream_t st, int *launches) {
    const unsigned grid = (unsigned)(((long long)p.B.rows * p.heads + 7) / 8);
    if (p.P.dim == 128) launch_rows<128>(p, grid, st);
    else launch_rows<64>(p, grid, st);
    *launches += 1;
    return cudaGetLastError();
}

}  // namespace apk
