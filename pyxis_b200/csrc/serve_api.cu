// serve_api.cu -- the extern "C" boundary of include/pyxis_serve.h: argument checks and dispatch.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "common.cuh"
#include "ctx.h"
#include "kernels.h"
#include "serve.h"

using namespace pyxis;

namespace {

int fail(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return record_error(code, buf);
}

int cuda_status(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return PYXIS_OK;
    return fail(PYXIS_ECUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

// Makes ctx's device current for the call and restores the caller's device afterwards.
struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) cudaSetDevice(dev);
    }
    ~DeviceGuard() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

cudaStream_t pick_stream(pyxis_cuda_ctx *ctx, void *stream) { return stream ? (cudaStream_t)stream : ctx->stream; }

bool is_dtype(int t) { return t == PYXIS_DTYPE_F32 || t == PYXIS_DTYPE_BF16; }
size_t elem(int dtype) { return dtype == PYXIS_DTYPE_F32 ? 4 : 2; }
bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// [a, a + an) and [b, b + bn) share bytes.
bool overlap(const void *a, size_t an, const void *b, size_t bn) {
    const char *x = (const char *)a, *y = (const char *)b;
    return x < y + bn && y < x + an;
}

// `layers`: whether the call uses the layer axis.
int check_pages(const pyxis_kv_pages *kv, bool layers) {
    if (!kv || !kv->k || !kv->v) return fail(PYXIS_EINVAL, "null cache pages");
    if (!is_dtype(kv->dtype)) return fail(PYXIS_EINVAL, "cache dtype %d is neither f32 nor bf16", kv->dtype);
    if (kv->head_dim != 64 && kv->head_dim != 128) return fail(PYXIS_EINVAL, "head_dim %d is not 64 or 128", kv->head_dim);
    if (kv->num_pages <= 0 || kv->page_size <= 0 || kv->n_kv_heads <= 0 || (layers && kv->n_layers <= 0))
        return fail(PYXIS_EINVAL, "cache of %d layers, %d pages of %d slots, %d heads", kv->n_layers, kv->num_pages,
                    kv->page_size, kv->n_kv_heads);
    if ((long long)kv->num_pages * kv->page_size >= (1ll << 31))
        return fail(PYXIS_EINVAL, "num_pages * page_size must be below 2^31");
    if ((long long)kv->page_size * kv->n_kv_heads * kv->head_dim >= (1ll << 31))
        return fail(PYXIS_EINVAL, "a page of 2^31 elements or more");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return fail(PYXIS_EINVAL, "cache bases must be 16-byte aligned");
    const int64_t v = 16 / (int64_t)elem(kv->dtype);
    const struct {
        const char *name;
        int64_t stride;
        bool used;
    } s[4] = {{"layer", kv->layer_stride, layers && kv->n_layers > 1},
              {"page", kv->page_stride, kv->num_pages > 1},
              {"slot", kv->slot_stride, kv->page_size > 1},
              {"head", kv->head_stride, kv->n_kv_heads > 1}};
    for (const auto &x : s)
        if (x.used && (x.stride < kv->head_dim || x.stride % v != 0))
            return fail(PYXIS_EINVAL, "cache %s stride %lld: a multiple of 16 bytes of at least head_dim is needed", x.name,
                        (long long)x.stride);
    return PYXIS_OK;
}

int check_tree(const pyxis_tree_attention_args *a, const pyxis_kv_pages *kv) {
    if (!a) return fail(PYXIS_EINVAL, "null arguments");
    if (const int rc = check_pages(kv, false)) return rc;
    if (a->n_q_heads <= 0 || a->n_q_heads % kv->n_kv_heads)
        return fail(PYXIS_EINVAL, "%d query heads over %d kv heads", a->n_q_heads, kv->n_kv_heads);
    if (a->max_tree < 1 || a->max_tree > 64) return fail(PYXIS_EINVAL, "max_tree %d outside 1 .. 64", a->max_tree);
    if (a->n_rows > (size_t)INT32_MAX || a->n_seq > (size_t)INT32_MAX) return fail(PYXIS_EINVAL, "too many rows or sequences");
    if (a->max_context < 0) return fail(PYXIS_EINVAL, "negative max_context");
    if (a->n_seq > 1 && a->table_stride < a->table_width)
        return fail(PYXIS_EINVAL, "block table rows of %zu with stride %zu", a->table_width, a->table_stride);
    if (a->table_width > (size_t)INT32_MAX) return fail(PYXIS_EINVAL, "block table too wide");
    if ((long long)a->max_tree * a->n_q_heads > 65535) return fail(PYXIS_EINVAL, "too many query heads");
    return PYXIS_OK;
}

}  // namespace

extern "C" {

int pyxis_rope_frequencies(int kind, double theta, int rotary_dim, double factor, double original_context,
                           double beta_fast, double beta_slow, double *freq, double *scale) {
    if (!freq || !scale) return fail(PYXIS_EINVAL, "null freq or scale");
    if (rotary_dim <= 0 || rotary_dim % 2) return fail(PYXIS_EINVAL, "rotary_dim %d is not even and positive", rotary_dim);
    if (kind < PYXIS_ROPE_PLAIN || kind > PYXIS_ROPE_YARN) return fail(PYXIS_EINVAL, "unknown frequency scaling %d", kind);
    if (!(theta > 0.0) || !std::isfinite(theta) || !(factor >= 1.0) || !std::isfinite(factor))
        return fail(PYXIS_EINVAL, "theta %g must be positive and factor %g at least 1", theta, factor);
    if (kind == PYXIS_ROPE_YARN && (!(theta > 1.0) || !(original_context > 0.0) || !(beta_slow > 0.0) || !(beta_fast > beta_slow) ||
                                    !std::isfinite(original_context) || !std::isfinite(beta_fast)))
        return fail(PYXIS_EINVAL, "yarn needs theta > 1, original_context > 0 and beta_fast > beta_slow > 0");
    if (kind == PYXIS_ROPE_NTK) {
        if (rotary_dim <= 2) return fail(PYXIS_EINVAL, "ntk scaling needs rotary_dim > 2");
        theta *= std::pow(factor, (double)rotary_dim / (rotary_dim - 2));
    }
    const int n = rotary_dim / 2;
    *scale = kind == PYXIS_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
    double low = 0, high = 0;
    if (kind == PYXIS_ROPE_YARN) {
        // index of the frequency that turns `beta` times over the original context
        const auto index = [&](double beta) {
            return rotary_dim * std::log(original_context / (beta * 6.283185307179586477)) / (2.0 * std::log(theta));
        };
        low = std::max(0.0, std::floor(index(beta_fast)));
        high = std::max(low, std::min(rotary_dim - 1.0, std::ceil(index(beta_slow))));  // (past the last index, n - 1, too)
    }
    for (int i = 0; i < n; ++i) {
        const double f = std::pow(theta, -2.0 * i / rotary_dim);
        if (kind == PYXIS_ROPE_LINEAR) {
            freq[i] = f / factor;
        } else if (kind == PYXIS_ROPE_YARN) {
            const double ramp = high > low ? std::min(1.0, std::max(0.0, (i - low) / (high - low))) : (i > low ? 1.0 : 0.0);
            freq[i] = f * (1.0 - ramp) + f / factor * ramp;
        } else {
            freq[i] = f;
        }
    }
    return PYXIS_OK;
}

int pyxis_cuda_qk_norm_rope_dev(pyxis_cuda_ctx *ctx, const pyxis_qk_norm_rope_args *a, const pyxis_kv_pages *kv,
                                void *stream) {
    if (!a) return fail(PYXIS_EINVAL, "null arguments");
    if (const int rc = check_pages(kv, false)) return rc;
    if (a->n_tokens == 0) return PYXIS_OK;
    if (a->n_tokens > (size_t)INT32_MAX) return fail(PYXIS_EINVAL, "too many tokens");
    if (!a->qkv || !a->q || !a->slots) return fail(PYXIS_EINVAL, "null qkv, q or slots");
    if (a->n_q_heads <= 0 || (long long)a->n_q_heads + 2ll * kv->n_kv_heads > (1 << 20))
        return fail(PYXIS_EINVAL, "%d query heads", a->n_q_heads);
    if (a->rotary_dim < 0 || a->rotary_dim > kv->head_dim || a->rotary_dim % 16)
        return fail(PYXIS_EINVAL, "rotary_dim %d is not a multiple of 16 up to head_dim %d", a->rotary_dim, kv->head_dim);
    if (a->rotary_dim && (!a->positions || !a->inv_freq)) return fail(PYXIS_EINVAL, "null positions or inv_freq");
    const size_t es = elem(kv->dtype), v = 16 / es;
    const size_t row = ((size_t)a->n_q_heads + 2 * kv->n_kv_heads) * kv->head_dim, qrow = (size_t)a->n_q_heads * kv->head_dim;
    if ((a->n_tokens > 1 && (a->ld_qkv < row || a->ld_q < qrow)) || a->ld_qkv % v || a->ld_q % v)
        return fail(PYXIS_EINVAL, "rows of qkv (stride %zu) and q (%zu) must hold their heads and be multiples of 16 bytes",
                    a->ld_qkv, a->ld_q);
    if (!aligned(a->qkv, 16) || !aligned(a->q, 16)) return fail(PYXIS_EINVAL, "qkv and q must be 16-byte aligned");
    const size_t n = a->n_tokens - 1;
    if (overlap(a->qkv, (n * a->ld_qkv + row) * es, a->q, (n * a->ld_q + qrow) * es) &&
        !(a->qkv == a->q && (n == 0 || a->ld_qkv == a->ld_q)))
        return fail(PYXIS_EINVAL, "q overlaps qkv without being qkv itself");
    if (!ctx) return fail(PYXIS_EINVAL, "null context");
    DeviceGuard g(ctx->device);
    return cuda_status(launch_qk_norm_rope(*a, *kv, ctx->num_sms, pick_stream(ctx, stream)), "qk_norm_rope launch");
}

size_t pyxis_cuda_tree_attention_workspace_size(pyxis_cuda_ctx *ctx, const pyxis_tree_attention_args *a,
                                                const pyxis_kv_pages *kv) {
    if (!ctx || check_tree(a, kv) != PYXIS_OK || a->n_seq == 0 || a->n_rows == 0) return 0;
    return tree_attention_workspace(plan_tree_attention(*a, *kv, ctx->num_sms), *a, *kv, ctx->num_sms);
}

int pyxis_cuda_tree_attention_dev(pyxis_cuda_ctx *ctx, const pyxis_tree_attention_args *a, const pyxis_kv_pages *kv,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    if (const int rc = check_tree(a, kv)) return rc;
    if (a->n_seq == 0 || a->n_rows == 0) return PYXIS_OK;
    if (!a->q || !a->out || !a->q_start || !a->context_len || (!a->block_table && a->table_width))
        return fail(PYXIS_EINVAL, "null q, out, q_start, context_len or block_table");
    const size_t es = elem(kv->dtype);
    if (!aligned(a->q, es) || !aligned(a->out, es)) return fail(PYXIS_EINVAL, "q and out must be aligned to their type");
    const int64_t hd = kv->head_dim, rows = (int64_t)a->n_rows - 1, heads = a->n_q_heads - 1;
    if (a->q_row < 0 || a->q_head < 0 || (heads && a->out_head < hd) || (rows && a->out_row < hd) || (heads && a->q_head < hd) ||
        (rows && a->q_row < hd))
        return fail(PYXIS_EINVAL, "strides of q and out must be at least head_dim");
    if (overlap(a->q, (size_t)(rows * a->q_row + heads * a->q_head + hd) * es, a->out,
                (size_t)(rows * a->out_row + heads * a->out_head + hd) * es))
        return fail(PYXIS_EINVAL, "out overlaps q");
    if (!ctx) return fail(PYXIS_EINVAL, "null context");
    DeviceGuard g(ctx->device);
    cudaStream_t st = pick_stream(ctx, stream);
    const TreePlan plan = plan_tree_attention(*a, *kv, ctx->num_sms);
    const size_t need = tree_attention_workspace(plan, *a, *kv, ctx->num_sms);
    if (need && workspace) {
        if (workspace_bytes < need || !aligned(workspace, 256))
            return fail(PYXIS_EINVAL, "tree attention workspace: %zu bytes, 256-byte aligned, are needed", need);
    } else if (need) {
        if (const int rc = context_workspace(ctx, need, st)) return rc;
        workspace = ctx->ws;
    }
    return cuda_status(launch_tree_attention(*a, *kv, plan, workspace, ctx->d_err, ctx->num_sms, st),
                       "tree attention launch");
}

int pyxis_cuda_kv_copy_pages_dev(pyxis_cuda_ctx *ctx, const pyxis_kv_pages *kv, const int32_t *src, const int32_t *dst,
                                 size_t n, void *stream) {
    if (const int rc = check_pages(kv, true)) return rc;
    if (n == 0) return PYXIS_OK;
    if (!src || !dst) return fail(PYXIS_EINVAL, "null src or dst");
    if (kv->n_layers > 32767) return fail(PYXIS_EINVAL, "more than 32767 layers");
    if (!ctx) return fail(PYXIS_EINVAL, "null context");
    DeviceGuard g(ctx->device);
    return cuda_status(launch_kv_copy_pages(*kv, src, dst, n, ctx->num_sms, pick_stream(ctx, stream)), "kv_copy_pages launch");
}

int pyxis_cuda_kv_compact_dev(pyxis_cuda_ctx *ctx, const pyxis_kv_pages *kv, const int32_t *block_table,
                              size_t table_stride, size_t table_width, const int32_t *context_len,
                              const uint64_t *accepted, size_t n_seq, int32_t *new_len, void *stream) {
    if (const int rc = check_pages(kv, true)) return rc;
    if (n_seq == 0) return PYXIS_OK;
    if (!block_table || !context_len || !accepted || !new_len)
        return fail(PYXIS_EINVAL, "null block_table, context_len, accepted or new_len");
    if ((long long)kv->n_layers * kv->n_kv_heads * kv->head_dim >= (1ll << 30)) return fail(PYXIS_EINVAL, "cache rows too long");
    if (n_seq > 65535 || table_width > (size_t)INT32_MAX) return fail(PYXIS_EINVAL, "more than 65535 sequences, or too wide a table");
    if (n_seq > 1 && table_stride < table_width)
        return fail(PYXIS_EINVAL, "block table rows of %zu with stride %zu", table_width, table_stride);
    if (overlap(context_len, n_seq * 4, new_len, n_seq * 4)) return fail(PYXIS_EINVAL, "new_len overlaps context_len");
    if (!ctx) return fail(PYXIS_EINVAL, "null context");
    DeviceGuard g(ctx->device);
    return cuda_status(launch_kv_compact(*kv, block_table, table_stride, table_width, context_len, accepted, n_seq, new_len,
                                         ctx->num_sms, pick_stream(ctx, stream)),
                       "kv_compact launch");
}

int pyxis_cuda_sample_dev(pyxis_cuda_ctx *ctx, const void *logits, int dtype, size_t M, size_t n, size_t ld,
                          const float *uniforms, const pyxis_sample_params *params, int32_t *idx, float *prob,
                          void *stream) {
    if (!params) return fail(PYXIS_EINVAL, "null params");
    if (!is_dtype(dtype)) return fail(PYXIS_EINVAL, "logits dtype %d is neither f32 nor bf16", dtype);
    if (M == 0) return PYXIS_OK;
    if (n == 0) return fail(PYXIS_EINVAL, "sample from an empty row");
    if (n > (size_t)INT32_MAX) return fail(PYXIS_EINVAL, "row too long to sample from (%zu)", n);
    if (M > 65535) return fail(PYXIS_EINVAL, "sample: %zu rows > 65535 per call", M);
    if (M > 1 && ld < n) return fail(PYXIS_EINVAL, "row stride smaller than the row");
    if (!logits || !uniforms || !idx) return fail(PYXIS_EINVAL, "null logits, uniforms or idx");
    if (!aligned(logits, elem(dtype))) return fail(PYXIS_EINVAL, "logits are not aligned to their type");
    if (!ctx) return fail(PYXIS_EINVAL, "null context");
    DeviceGuard g(ctx->device);
    return cuda_status(launch_sample(logits, dtype, M, n, ld, uniforms, *params, idx, prob, ctx->num_sms,
                                     pick_stream(ctx, stream)),
                       "sample launch");
}

}  // extern "C"
