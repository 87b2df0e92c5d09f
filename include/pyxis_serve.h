/*
 * pyxis_serve.h -- operators of a decoding step that verifies drafted tokens over a paged KV cache.
 *
 * One step of a serving loop takes the q|k|v rows of pyxis_cuda_matmul_dev, normalises and rotates
 * their heads and puts keys and values into the cache's pages (pyxis_cuda_qk_norm_rope_dev),
 * attends with a tree of drafted tokens per sequence (pyxis_cuda_tree_attention_dev; a tree of one
 * node is a plain decode step, a chain a prompt's chunk), draws a token for every node from its
 * logits (pyxis_cuda_sample_dev), moves the accepted branch's cache entries to the front of their
 * drafts (pyxis_cuda_kv_compact_dev) and forks sequences by copying pages
 * (pyxis_cuda_kv_copy_pages_dev).
 *
 * The operators extend the reference's parts of the same names: QK-norm and RoPE
 * (src/attention.rs:81-93, :144-162), the KV cache (src/kv_cache.rs), causal attention
 * (src/attention.rs:107-135) and Sampler::sample (src/sampler.rs:23-110).
 *
 * Conventions are those of pyxis_cuda.h: status codes and pyxis_cuda_last_error(); every pointer
 * named below is device memory of the context's device unless it says host; calls are asynchronous
 * on `stream` (NULL: the context's) and may be captured into a CUDA graph.  dtype is
 * PYXIS_DTYPE_F32 or PYXIS_DTYPE_BF16; sums, maxima and norms are f32 or wider for both.  Indexes
 * read from device memory (pages, slots, lengths) are bounds-checked by the kernels: a page or slot
 * outside the cache is never read or written, and what a sequence naming one gets is unspecified.
 * Kernels that wait for copies or tensor-core products give up after a limit, with their outputs partly
 * unwritten: pyxis_cuda_check_device_error reports it.
 */
#ifndef PYXIS_SERVE_H
#define PYXIS_SERVE_H

#include <stddef.h>
#include <stdint.h>

#include "pyxis_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A paged KV cache.  Element d of head h in slot s of page p of layer l is at
 * base + l * layer_stride + p * page_stride + s * slot_stride + h * head_stride + d (strides in
 * elements, the same for k and v; any order of the axes).  k and v are 16-byte aligned and every
 * stride is a multiple of 16 bytes; head_dim is 64 or 128.  num_pages * page_size < 2^31.
 * A sequence's position j lives in slot j % page_size of page block_table[j / page_size]. */
typedef struct {
    void *k, *v;
    int dtype;
    int n_layers, num_pages, page_size, n_kv_heads, head_dim;
    int64_t layer_stride, page_stride, slot_stride, head_stride;
} pyxis_kv_pages;

/* Rotary frequencies, computed on the host in 64 bits: freq[i] for i < rotary_dim / 2 (host memory),
 * and *scale, the factor of cos and sin (1 but for YARN).
 *   PLAIN   theta^(-2i / rotary_dim)
 *   LINEAR  those / factor                           (positions divided by factor)
 *   NTK     theta * factor^(rotary_dim / (rotary_dim - 2)) in theta's place
 *   YARN    plain / factor where the frequency turns less than beta_slow times over
 *           original_context positions, plain where it turns more than beta_fast times, a mixture
 *           between them: with r = clamp((i - low) / (high - low), 0, 1),
 *             freq[i] = plain (1 - r) + plain / factor r,
 *             low = max(0, floor(at(beta_fast))), high = min(rotary_dim - 1, ceil(at(beta_slow))),
 *             at(b) = rotary_dim ln(original_context / (2 pi b)) / (2 ln theta), the index of the
 *             frequency that turns b times (which may lie past the last one)
 *           (high <= low: plain up to low, plain / factor after it); *scale = 0.1 ln(factor) + 1
 * rotary_dim is even and positive, theta > 0, factor >= 1, and for YARN original_context > 0 and
 * beta_fast > beta_slow > 0 (others ignore those). */
enum { PYXIS_ROPE_PLAIN = 0, PYXIS_ROPE_LINEAR = 1, PYXIS_ROPE_NTK = 2, PYXIS_ROPE_YARN = 3 };
int pyxis_rope_frequencies(int kind, double theta, int rotary_dim, double factor, double original_context,
                           double beta_fast, double beta_slow, double *freq, double *scale);

/* RMSNorm of every query and key head (skipped for a NULL weight), then the rotation of each head's
 * first rotary_dim elements by positions[t] * inv_freq[i], in one pass over the q|k|v rows:
 *   qkv  [n_tokens][ld_qkv]: n_q_heads query heads, then n_kv_heads key heads, then value heads
 *   q    [n_tokens][ld_q]: the query heads; may be qkv itself (same stride)
 *   kv   one layer's pages (n_layers is ignored): key and value heads of token t go to slot
 *        slots[t] (page slots[t] / page_size); a slot outside [0, num_pages * page_size), such as
 *        -1 of a padded row, is left out.  Slots of one call are distinct.
 * Pairs are elements (i, i + rotary_dim / 2) or, with interleaved != 0, (2i, 2i + 1).  The angle is
 * formed and reduced in 64 bits, so far positions keep f32 accuracy; cos and sin are multiplied by
 * rope_scale.  rotary_dim is a multiple of 16 up to head_dim, or 0 for none; q_norm, k_norm
 * [head_dim] f32; inv_freq [rotary_dim / 2] f64 (pyxis_rope_frequencies, copied to the device).
 * qkv and q have the cache's dtype, rows of 16-byte multiples and 16-byte aligned bases. */
typedef struct {
    const void *qkv;
    void *q;
    size_t n_tokens, ld_qkv, ld_q; /* strides in elements */
    const int32_t *positions, *slots;
    const double *inv_freq;
    const float *q_norm, *k_norm;
    int n_q_heads, rotary_dim, interleaved;
    float eps, rope_scale;
} pyxis_qk_norm_rope_args;
int pyxis_cuda_qk_norm_rope_dev(pyxis_cuda_ctx *ctx, const pyxis_qk_norm_rope_args *a, const pyxis_kv_pages *kv,
                                void *stream);

/* Attention of drafted tokens over a paged cache, grouped query heads.  Sequence s owns the query
 * rows q_start[s] .. q_start[s+1] - 1; its node j (row q_start[s] + j) attends to the cache's
 * positions 0 .. context_len[s] - 1 and to every node i of the sequence with bit i of
 * tree_mask[row] set, whose keys and values are at position context_len[s] + i.  A NULL tree_mask
 * is a chain: node j attends to nodes 0 .. j.
 *   q, out  [rows][n_q_heads][head_dim], strides q_row / q_head and out_row / out_head in elements
 *   n_seq sequences, at most max_tree nodes each (1 .. 64; further nodes get no output);
 *   max_tree * n_q_heads <= 65535
 *   block_table [n_seq][table_stride] pages, table_width of them valid
 *   max_context  a bound of context_len that only plans the split of the keys over the GPU
 * out = softmax(scale * q . k) v; a row that attends to nothing is zero, rows outside
 * [q_start[0], q_start[n_seq]) are left as they are.  Non-finite keys or values at positions that
 * a row does not attend to do not reach it; an infinite value that it attends to is infinite in its
 * column of the output, a key whose score is -inf has no weight.
 * Scores, weights and sums are f32.  bf16 pages: products are exact, weights enter P V in f32 or as two
 * bf16 terms (off by 2^-16 at most), and the output is rounded to bf16 once.  f32 pages: up to 8 rows
 * (nodes x query heads of a kv head) products are f32, above that two terms per operand leave 2^-21 of a
 * product, and from 17 rows on an element below 2^-12 of the largest of its group (a query row, a kv
 * head's 64 context positions) keeps 2^-34 of that largest instead.  How work is split, and with it the
 * last bits, depends on the batch; the same call gives the same bits.  kv is one layer's pages, dtype that of q and out.
 * The split's partial sums need `workspace` of pyxis_cuda_tree_attention_workspace_size() bytes,
 * 256-byte aligned; NULL uses the context's, under the rules of pyxis_cuda_matmul_dev's. */
typedef struct {
    const void *q;
    void *out;
    int64_t q_row, q_head, out_row, out_head;
    size_t n_rows, n_seq;
    const int32_t *q_start, *context_len, *block_table;
    const uint64_t *tree_mask;
    size_t table_stride, table_width;
    int n_q_heads, max_tree;
    int64_t max_context;
    float scale;
} pyxis_tree_attention_args;
int pyxis_cuda_tree_attention_dev(pyxis_cuda_ctx *ctx, const pyxis_tree_attention_args *a, const pyxis_kv_pages *kv,
                                  void *workspace, size_t workspace_bytes, void *stream);
size_t pyxis_cuda_tree_attention_workspace_size(pyxis_cuda_ctx *ctx, const pyxis_tree_attention_args *a,
                                                const pyxis_kv_pages *kv);

/* Pages src[i] -> dst[i] for i < n, keys and values of every layer (a fork's partly filled page).
 * No page of dst may be in dst twice or in src. */
int pyxis_cuda_kv_copy_pages_dev(pyxis_cuda_ctx *ctx, const pyxis_kv_pages *kv, const int32_t *src, const int32_t *dst,
                                 size_t n, void *stream);

/* Keeps the accepted nodes of each sequence's tree: the cache entries at positions
 * context_len[s] + j of the set bits j of accepted[s] move, in order, to context_len[s],
 * context_len[s] + 1, ... in every layer, and new_len[s] = context_len[s] + their number.
 * new_len is not context_len (a captured graph may replay the call).  No page may be in the tables
 * of two sequences at the positions moved. */
int pyxis_cuda_kv_compact_dev(pyxis_cuda_ctx *ctx, const pyxis_kv_pages *kv, const int32_t *block_table,
                              size_t table_stride, size_t table_width, const int32_t *context_len,
                              const uint64_t *accepted, size_t n_seq, int32_t *new_len, void *stream);

/* Draws one token per row of logits [M][n] (row stride ld elements) from a given uniform number:
 *   weights  w_i = exp((x_i - max x) / temperature); a temperature of 0 (or below, or NaN) is the
 *            greedy choice, the first maximum
 *   order    from the largest logit down, equal ones by index
 *   top_k    the first top_k tokens (0 or less: all)
 *   top_p    of those, the tokens before which less than top_p of their total weight lies (1 or
 *            more: all; the first token always stays)
 *   min_p    of those, the tokens with w_i >= min_p (w of the most likely token is 1)
 *   draw     the first token, in that order, at which the running sum of the kept weights exceeds
 *            uniform * their total; uniform in [0, 1), values outside are clamped
 * idx[r] is the token, prob[r] (may be NULL) its share of the kept weights (1 for greedy rows).
 * NaN logits count as -inf; with +inf logits only those have weight; a row without any number above
 * -inf gives idx -1, prob 0.  Parameters come per row from the arrays, or where an array is NULL
 * from the value next to it.  Weights are summed as 64-bit fixed-point numbers, so the choice does
 * not depend on the order of the sums.  n <= 2^31 - 1, M <= 65535. */
typedef struct {
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p;
    double temperature_all;
    int32_t top_k_all;
    double top_p_all, min_p_all;
} pyxis_sample_params;
int pyxis_cuda_sample_dev(pyxis_cuda_ctx *ctx, const void *logits, int dtype, size_t M, size_t n, size_t ld,
                          const float *uniforms, const pyxis_sample_params *params, int32_t *idx, float *prob,
                          void *stream);

#ifdef __cplusplus
}
#endif
#endif
