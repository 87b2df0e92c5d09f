// tree_attn.cuh -- what the tree-attention kernels (tree_attn.cu on the CUDA cores, tree_attn_tc.cu
// on the tensor cores) share: their parameters and a sequence's shape.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "serve.h"

namespace pyxis {

constexpr float kLog2e = 1.4426950408889634f;

struct TreeParams {
    const char *q, *k, *v;
    char *out;
    long long q_row, q_head, out_row, out_head;              // bytes
    long long page_stride, slot_stride, head_stride;         // bytes
    const int32_t *q_start, *context_len, *block_table;
    const unsigned long long *tree_mask;
    long long table_stride, capacity;                        // capacity: positions that a table row names
    int n_rows, n_q, n_kv, group, page_size, num_pages, max_tree, splits, row_tiles;
    float scale2;                                            // scale * log2 e
    float *part_o, *part_ml;                                 // [row][head][split][HD], [..][2] (splits > 1)
    int *err;
};

// A sequence's rows and keys, from device memory and clamped to what the buffers hold.
struct SeqShape {
    int row0, nodes;
    long long ctx, total;
};
PYXIS_DEVINL SeqShape seq_shape(const TreeParams &p, int seq) {
    SeqShape s;
    s.row0 = min(max(p.q_start[seq], 0), p.n_rows);
    const int end = min(max(p.q_start[seq + 1], s.row0), p.n_rows);
    s.nodes = min(end - s.row0, p.max_tree);
    s.ctx = min((long long)max(p.context_len[seq], 0), p.capacity);
    s.total = min(s.ctx + s.nodes, p.capacity);
    return s;
}

PYXIS_DEVINL void store(float *p, float x) { *p = x; }
PYXIS_DEVINL void store(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// Sums of values that are not finite (infinite or NaN; 0 if there are none).  Products in several terms need them
// for the columns of their outputs that are not finite: a weight's second term may be zero or negative, and an
// infinite value has none.  Nothing else calls them, so they stay out of the kernels' registers.
//
// In C columns per lane of a kv head (the first one's address in page 0), over the positions a .. b - 1 of a
// sequence with these pages: one pass of the whole warp for all of its columns, as the others wait meanwhile.
template <typename T, int C>
__device__ __noinline__ float4 odd_columns(const char *columns, const int32_t *pages, int num_pages, int page_size,
                                           long long page_stride, long long slot_stride, long long a, long long b) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const T *mine = reinterpret_cast<const T *>(columns) + (threadIdx.x & 31) * C;
#pragma unroll 4
    for (; a < b; ++a) {
        const long long i = a / page_size;
        const int page = min(max(__ldg(pages + i), 0), num_pages - 1);
        const T *v = reinterpret_cast<const T *>(reinterpret_cast<const char *>(mine) + page * page_stride +
                                                 (a - i * page_size) * slot_stride);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float x = (float)v[c];
            if (!isfinite(x)) sum[c] += x;
        }
    }
    return make_float4(sum[0], sum[1], sum[2], sum[3]);
}
template <typename T, int C>
PYXIS_DEVINL float4 odd_columns(const TreeParams &p, const SeqShape &sh, int seq, int kvh, int d, long long a, long long b) {
    return odd_columns<T, C>(p.v + kvh * p.head_stride + d * (int)sizeof(T), p.block_table + seq * p.table_stride, p.num_pages,
                             p.page_size, p.page_stride, p.slot_stride, a, min(b, sh.ctx));
}
// In one column, over those of the drafts at positions a .. b - 1 that a row with this mask sees.
template <typename T>
__device__ __noinline__ float odd_drafts(const char *column, const int32_t *pages, int num_pages, int page_size,
                                         long long page_stride, long long slot_stride, long long ctx, unsigned long long mask,
                                         long long a, long long b) {
    float sum = 0.f;
    for (; a < b; ++a) {
        if (!((mask >> (a - ctx)) & 1)) continue;
        const long long i = a / page_size;
        const int page = min(max(pages[i], 0), num_pages - 1);
        const float x = (float)*reinterpret_cast<const T *>(column + page * page_stride + (a - i * page_size) * slot_stride);
        if (!isfinite(x)) sum += x;
    }
    return sum;
}
template <typename T>
PYXIS_DEVINL float odd_drafts(const TreeParams &p, const SeqShape &sh, int seq, int kvh, int d, unsigned long long mask, long long a,
                              long long b) {
    return odd_drafts<T>(p.v + kvh * p.head_stride + d * (int)sizeof(T), p.block_table + seq * p.table_stride, p.num_pages,
                         p.page_size, p.page_stride, p.slot_stride, sh.ctx, mask, max(a, sh.ctx), min(b, sh.total));
}
// 0, or NaN if one of the values is not finite.
template <int N>
PYXIS_DEVINL float odd_mark(const float (&x)[N]) {
    float z[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) z[i & 1] = fmaf(x[i], 0.f, z[i & 1]);
    return z[0] + z[1];
}

// q . k of the key at a position of an f32 cache (its head's address in page 0), in f32: for keys that
// products in several terms cannot take.
template <int HD>
__device__ __noinline__ float key_score(const float *q, const char *head, const int32_t *pages, int num_pages, int page_size,
                                        long long page_stride, long long slot_stride, long long pos) {
    const long long i = pos / page_size;
    const float *k = reinterpret_cast<const float *>(head + min(max(pages[i], 0), num_pages - 1) * page_stride +
                                                     (pos - i * page_size) * slot_stride);
    float x = 0.f;
#pragma unroll 4
    for (int d = 0; d < HD; ++d) x = fmaf(q[d], k[d], x);
    return x;
}
template <int HD>
PYXIS_DEVINL float key_score(const TreeParams &p, const float *q, int seq, int kvh, long long pos) {
    return key_score<HD>(q, p.k + kvh * p.head_stride, p.block_table + seq * p.table_stride, p.num_pages, p.page_size,
                         p.page_stride, p.slot_stride, pos);
}

// The tensor-core forms, bf16 and f32 pages of sizes that tile their blocks of keys: whether one takes
// the call, its workspace, its launch.
bool tree_attention_tc_supported(const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv);
size_t tree_attention_tc_workspace(const pyxis_kv_pages &kv, int num_sms);
cudaError_t launch_tree_attention_tc(const TreeParams &p, const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv,
                                     void *workspace, int num_sms, cudaStream_t st);
bool tree_attention_tc32_supported(const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv);
size_t tree_attention_tc32_workspace(const pyxis_kv_pages &kv, int num_sms);
cudaError_t launch_tree_attention_tc32(const TreeParams &p, const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv,
                                       void *workspace, int num_sms, cudaStream_t st);

}  // namespace pyxis
