// serve.h -- internal launcher interface between the entry points of include/pyxis_serve.h
// (serve_api.cu) and their kernels.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/pyxis_serve.h"

namespace pyxis {

cudaError_t launch_qk_norm_rope(const pyxis_qk_norm_rope_args &a, const pyxis_kv_pages &kv, int num_sms,
                                cudaStream_t st);

// How a call's keys are split over the GPU, from sizes the host knows.
struct TreePlan {
    bool tensor;    // on the tensor cores, which split rows and keys on the device
    int row_tile;   // query rows (nodes x heads of one kv head) of a CTA
    int row_tiles;  // CTAs over the rows of one (sequence, kv head)
    int splits;     // CTAs over the keys
    int per_sm;     // CTAs that share an SM
};
TreePlan plan_tree_attention(const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv, int num_sms);
size_t tree_attention_workspace(const TreePlan &p, const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv,
                                int num_sms);
cudaError_t launch_tree_attention(const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv, const TreePlan &p,
                                  void *workspace, int *err, int num_sms, cudaStream_t st);

cudaError_t launch_kv_copy_pages(const pyxis_kv_pages &kv, const int32_t *src, const int32_t *dst, size_t n, int num_sms,
                                 cudaStream_t st);
cudaError_t launch_kv_compact(const pyxis_kv_pages &kv, const int32_t *block_table, size_t table_stride,
                              size_t table_width, const int32_t *context_len, const uint64_t *accepted, size_t n_seq,
                              int32_t *new_len, int num_sms, cudaStream_t st);

cudaError_t launch_sample(const void *logits, int dtype, size_t M, size_t n, size_t ld, const float *uniforms,
                          const pyxis_sample_params &p, int32_t *idx, float *prob, int num_sms, cudaStream_t st);

}  // namespace pyxis
