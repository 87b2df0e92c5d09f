// paged.cu -- page copies (forks) and the compaction of accepted drafts in a paged KV cache
// (the cache of src/kv_cache.rs:34-41 cut into pages; include/pyxis_serve.h).  Both only move
// bytes: 16 bytes per thread and access, several accesses in flight.
//
// Measured (28 layers, pages of 16 positions, 8 kv heads of 128): 96 bf16 pages copied in 57 us, 6.2 TB/s
// of reads and writes (a floor of 54.5 us at the rate of a plain copy); 2 f32 pages 4.1 us, of which a
// launch is most.  Compaction of 64 trees of 16 nodes, bf16, 14 us for 47 MB, one tree of 64 nodes, f32,
// 8 us: not the bytes (7 and 2 us) but the chain mask - table - rows bounds it.
#include <algorithm>

#include "common.cuh"
#include "serve.h"

namespace pyxis {
namespace {

constexpr int kThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kMoveUnroll = 8;  // moves of one column in flight

struct PageGeom {
    char *k, *v;
    long long layer_stride, page_stride, slot_stride, head_stride;  // bytes
    int n_layers, num_pages, page_size, n_kv;
    int row_vecs;  // 16-byte vectors of one head's row
};

PageGeom geom(const pyxis_kv_pages &kv) {
    const long long es = kv.dtype == PYXIS_DTYPE_F32 ? 4 : 2;
    return PageGeom{(char *)kv.k,          (char *)kv.v,          kv.layer_stride * es, kv.page_stride * es,
                    kv.slot_stride * es,   kv.head_stride * es,   kv.n_layers,          kv.num_pages,
                    kv.page_size,          kv.n_kv_heads,         (int)(kv.head_dim * es / 16)};
}

// grid (chunks of a page, pairs, 2 * layers).  `flat`: a page is one contiguous run of bytes.
__global__ void __launch_bounds__(kThreads) kv_copy_pages_kernel(const PageGeom g, const int32_t *__restrict__ src,
                                                                const int32_t *__restrict__ dst, int flat) {
    pdl_wait();
    pdl_trigger();
    const int s = src[blockIdx.y], d = dst[blockIdx.y];
    if (s < 0 || d < 0 || s >= g.num_pages || d >= g.num_pages || s == d) return;
    char *base = ((blockIdx.z & 1) ? g.v : g.k) + (long long)(blockIdx.z >> 1) * g.layer_stride;
    const char *from = base + s * g.page_stride;
    char *to = base + d * g.page_stride;
    const int vecs = g.page_size * g.n_kv * g.row_vecs;
    const int first = blockIdx.x * (kThreads * kCopyUnroll) + threadIdx.x;
    uint4 x[kCopyUnroll];
    long long at[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u) {
        const int i = first + u * kThreads;
        if (flat) {
            at[u] = (long long)i * 16;
        } else {
            const int row = i / g.row_vecs, slot = row / g.n_kv;
            at[u] = slot * g.slot_stride + (row - slot * g.n_kv) * g.head_stride + (i - row * g.row_vecs) * 16;
        }
        if (i < vecs) x[u] = *reinterpret_cast<const uint4 *>(from + at[u]);
    }
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
        if (first + u * kThreads < vecs) *reinterpret_cast<uint4 *>(to + at[u]) = x[u];
}

// grid (parts, sequences): the 16-byte columns of a sequence's rows, over all layers' keys and values,
// are dealt to the threads of its parts.  A thread moves its column through all of the sequence's
// moves in order.  A move's place is never a later move's source: node j of rank r goes to r <= j,
// and later sources lie beyond j.  So a batch of loads may run ahead of its stores, and one thread's
// order of accesses to its column is all the ordering needed.  Latency bounds it (the mask, the
// table, then the rows): a CTA forms the moves once for several columns per thread.
__global__ void __launch_bounds__(kThreads)
    kv_compact_kernel(const PageGeom g, const int32_t *__restrict__ table, long long table_stride, int table_width,
                      const int32_t *__restrict__ context_len, const unsigned long long *__restrict__ accepted,
                      int32_t *__restrict__ new_len) {
    __shared__ long long from[64], to[64];
    pdl_wait();
    pdl_trigger();
    const int seq = blockIdx.y;
    const unsigned long long acc = accepted[seq];
    const int ctx = max(context_len[seq], 0);
    const int n = __popcll(acc);
    const int lead = acc == ~0ull ? 64 : __ffsll(~acc) - 1;  // accepted nodes already in their place
    if (blockIdx.x == 0 && threadIdx.x == 0) new_len[seq] = ctx + n;
    const int moves = n - lead;
    if (moves <= 0) return;
    if (threadIdx.x < 64 && ((acc >> threadIdx.x) & 1)) {
        const int rank = __popcll(acc & ((1ull << threadIdx.x) - 1));
        if (rank >= lead) {
            long long o[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const long long pos = (long long)ctx + (e ? rank : (int)threadIdx.x), b = pos / g.page_size;
                const int page = b < table_width ? table[seq * table_stride + b] : -1;
                o[e] = page >= 0 && page < g.num_pages ? page * g.page_stride + (pos - b * g.page_size) * g.slot_stride : -1;
            }
            from[rank - lead] = o[1] < 0 ? -1 : o[0];
            to[rank - lead] = o[1];
        }
    }
    __syncthreads();
    const int cols = g.n_kv * g.row_vecs, total = 2 * g.n_layers * cols;
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < total; i += gridDim.x * kThreads) {
        const int plane = i / cols, c = i - plane * cols, head = c / g.row_vecs;
        char *col = ((plane & 1) ? g.v : g.k) + (plane >> 1) * g.layer_stride + head * g.head_stride + (c - head * g.row_vecs) * 16;
        for (int m0 = 0; m0 < moves; m0 += kMoveUnroll) {
            uint4 x[kMoveUnroll];
#pragma unroll
            for (int u = 0; u < kMoveUnroll; ++u)
                if (m0 + u < moves && from[m0 + u] >= 0) x[u] = *reinterpret_cast<const uint4 *>(col + from[m0 + u]);
#pragma unroll
            for (int u = 0; u < kMoveUnroll; ++u)
                if (m0 + u < moves && from[m0 + u] >= 0) *reinterpret_cast<uint4 *>(col + to[m0 + u]) = x[u];
        }
    }
}

}  // namespace

cudaError_t launch_kv_copy_pages(const pyxis_kv_pages &kv, const int32_t *src, const int32_t *dst, size_t n, int num_sms,
                                 cudaStream_t st) {
    (void)num_sms;
    const PageGeom g = geom(kv);
    const long long row = kv.head_dim;
    const int flat = (kv.head_stride == row && kv.slot_stride == row * kv.n_kv_heads) ||
                     (kv.slot_stride == row && kv.head_stride == row * kv.page_size);
    const int vecs = kv.page_size * kv.n_kv_heads * g.row_vecs, per = kThreads * kCopyUnroll;
    for (size_t i = 0; i < n; i += 65535) {  // grid.y
        const unsigned m = (unsigned)(n - i < 65535 ? n - i : 65535);
        const cudaError_t e = launch_kernel(kv_copy_pages_kernel, dim3((vecs + per - 1) / per, m, 2 * kv.n_layers),
                                            dim3(kThreads), 0, st, g, src + i, dst + i, flat);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_kv_compact(const pyxis_kv_pages &kv, const int32_t *block_table, size_t table_stride,
                              size_t table_width, const int32_t *context_len, const uint64_t *accepted, size_t n_seq,
                              int32_t *new_len, int num_sms, cudaStream_t st) {
    const PageGeom g = geom(kv);
    // about four CTAs an SM, and no more than one column per thread
    const size_t total = (size_t)2 * kv.n_layers * kv.n_kv_heads * g.row_vecs;
    const size_t parts = std::max<size_t>(1, std::min((total + kThreads - 1) / kThreads, (size_t)num_sms * 4 / n_seq));
    return launch_kernel(kv_compact_kernel, dim3((unsigned)parts, (unsigned)n_seq), dim3(kThreads), 0, st, g, block_table, (long long)table_stride, (int)table_width, context_len,
                         (const unsigned long long *)accepted, new_len);
}

}  // namespace pyxis
