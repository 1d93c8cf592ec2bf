// The paged KV cache on the device: what its kernels share, and their launchers (pages.cu, pages_attn.cu).
//
// A pool holds n_pages pages of `page` positions for every layer; a sequence is a row of `table` (the pages of its
// positions, in order) and a length.  refs[p] counts the sequences that hold page p; 0 = free.
// Everything that the kernels read out of these arrays is checked before it becomes an address: a page number outside
// the pool is a page that is not there, a length beyond the table's row is cut to the row.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace apk {

enum { PTY_F32 = 0, PTY_F16 = 1, PTY_BF16 = 30 };  // GGML type ids

constexpr int PAGES_MAX_LIST = 1024;   // sequences that one reserve, fork or release names
constexpr int PAGES_MAX_BATCH = 4096;  // sequences of one batch of rows

// work[]: what the kernels of one pool hand on to one another
constexpr int PW_SHORT = 0;    // reserve: pages that were missing (0: done, -1: a row of the table is too short, PW_UNTRIED)
constexpr int PW_ERR = 1;      // a wait inside a kernel ran out (stays until it has been reported)
constexpr int PW_COPIES = 2;   // entries of the copy list
constexpr int PW_LIST = 64;    // n_seqs x {source page, destination page, positions, 0}, then the page lists
constexpr int PW_UNTRIED = -2; // in work[PW_SHORT]: reserve has changed nothing, because an expired wait is to be reported

struct PagesDev {
    uint16_t *k, *v;            // 16-bit elements
    long long ks[4], vs[4];     // elements between layers, pages, positions, kv heads
    int *table;
    long long table_stride;
    int *lens, *refs, *work;
    int n_seqs, width, n_layers, n_pages, page, shift, kv, dim, bf16;
};

// The packed rows of a batch: rows cu[i] .. cu[i+1] belong to sequence seqs[i] (null: i), and are its last positions.
struct BatchDev {
    const int *cu, *seqs;
    int n, rows;
};

struct SeqRows { int slot, first, rows, len; };

__host__ __device__ __forceinline__ int pages_len(const PagesDev &P, int slot) {
    const long long cap = (long long)P.width << P.shift;
    const int len = P.lens[slot];
    return len < 0 ? 0 : ((long long)len > cap ? (int)cap : len);
}

// Sequence i of the batch, with everything clamped to what exists; a slot outside the table has no positions.
__host__ __device__ __forceinline__ SeqRows batch_seq(const PagesDev &P, const BatchDev &B, int i) {
    SeqRows s;
    const int a = min(max(B.cu[i], 0), B.rows), b = min(max(B.cu[i + 1], a), B.rows);
    s.first = a;
    s.rows = b - a;
    s.slot = B.seqs ? B.seqs[i] : i;
    if (s.slot < 0 || s.slot >= P.n_seqs) {
        s.slot = 0;
        s.len = 0;
    } else {
        s.len = pages_len(P, s.slot);
    }
    return s;
}

// The sequence that row t belongs to; -1: none.
__host__ __device__ __forceinline__ int batch_find(const BatchDev &B, int t) {
    int lo = 0, hi = B.n;  // the last i with cu[i] <= t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (B.cu[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    --lo;
    return lo >= 0 && t < B.cu[lo + 1] ? lo : -1;
}

// Page that holds position j of a slot; -1: none.
__host__ __device__ __forceinline__ int page_of(const PagesDev &P, int slot, int j) {
    const int p = P.table[(long long)slot * P.table_stride + (j >> P.shift)];
    return (unsigned)p < (unsigned)P.n_pages ? p : -1;
}

struct AttendParams {
    PagesDev P;
    BatchDev B;
    int layer;
    const void *q;
    void *out;
    int ty;                      // of q and out
    long long qs[2], os[2];      // elements between rows, heads
    int heads, group;
    float scale_log2;            // scale * log2(e): the softmax runs in powers of two
    int causal, window;
};

struct RopeParams {
    PagesDev P;
    BatchDev B;
    int layer;
    const void *q, *k, *v;
    void *out;
    int ty, out_ty;
    long long qs[2], ks[2], vs[2], os[2];  // elements between rows, heads
    int heads;
    const int *positions;        // per row, or null: the row's own position in its sequence
    const float *q_norm, *k_norm;
    float eps;
    int rot, pairs;              // dimensions rotated; 1: neighbouring pairs, 0: halves
    float mag;                   // factor on sine and cosine
    double turn[128];            // turns a position, per pair
};

// Programmatic dependent launch: the kernel may be placed while the one in front of it in the stream is still ending.  Every
// kernel that is launched so calls pages_wait_front() before it reads or writes anything that another one touches.
template <typename... Args>
cudaError_t launch_front(void (*kernel)(Args...), dim3 grid, int block, size_t smem, cudaStream_t st, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
__device__ __forceinline__ void pages_wait_front() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pages_let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct SlotList {
    int n;
    int a[PAGES_MAX_LIST], b[PAGES_MAX_LIST];
};

cudaError_t launch_rope_append(const RopeParams &p, int n_sm, cudaStream_t st, int *launches);
cudaError_t prepare_attend();   // once per context, on its device
size_t attend_ws_bytes(const AttendParams &p, int n_sm);
cudaError_t launch_attend(const AttendParams &p, int n_sm, void *ws, long long wait_limit, cudaStream_t st, int *launches);
cudaError_t launch_pages_fork(const PagesDev &P, const SlotList &l, cudaStream_t st, int *launches);
cudaError_t launch_pages_release(const PagesDev &P, const SlotList &l, cudaStream_t st, int *launches);
cudaError_t launch_pages_reserve(const PagesDev &P, const SlotList &l, int heed, int n_sm, cudaStream_t st, int *launches);
cudaError_t launch_pages_compact(const PagesDev &P, int *page_map, int n_sm, cudaStream_t st, int *launches);

}  // namespace apk
