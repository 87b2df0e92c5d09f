// qk_rope.cu -- per-head RMSNorm of queries and keys, rotary positions and the append to a paged
// cache in one pass over the q|k|v rows (src/attention.rs:81-100 for many tokens at once, with the
// pair orders, partial rotation and scaled frequencies that the reference's :144-162 lacks).
//
//   x' = x * (w / sqrt(mean x^2 + eps));  (x_i, x_j)' = (x_i c - x_j s, x_j c + x_i s),
//   c, s = m cos a, m sin a,  a = position * inv_freq_i
//
// Bytes bound it: every element is read once and written once.  A head lies across HD / V lanes
// with V = 16 bytes of elements each, so the norm is a shuffle sum and the rotation's partner a
// shuffle away (halves) or in the same register vector (interleaved pairs).  The angles of a
// token are the same for all its heads: the CTA forms them once, in 64 bits (position * frequency
// has far more than 24 significant bits at far positions; reduced by multiples of pi/2 to
// [-pi/4, pi/4] before it is rounded to f32), while the heads' loads are in flight.
#include <cuda_bf16.h>

#include "common.cuh"
#include "serve.h"

namespace pyxis {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;      // heads in flight per lane group
constexpr int kMaxTokens = 4;   // tokens per CTA

// 16 bytes of T as f32.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int N = 4;
    static PYXIS_DEVINL void load(const uint4 &u, float (&v)[4]) {
        v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
    }
    static PYXIS_DEVINL uint4 store(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static PYXIS_DEVINL void load(const uint4 &u, float (&v)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static PYXIS_DEVINL uint4 store(const float (&v)[8]) {  // the one rounding of the bf16 form
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// cos and sin of pos * f, each rounded to f32 from an argument reduced in 64 bits.
PYXIS_DEVINL float2 cos_sin(int pos, double f) {
    const double a = (double)pos * f;
    const double n = rint(a * 0.63661977236758134308);  // 2 / pi
    // pi / 2 as the sum of two doubles
    double r = fma(-n, 1.57079632679489655800, a);
    r = fma(-n, 6.12323399573676603587e-17, r);
    float s, c;
    sincosf((float)r, &s, &c);
    const int q = (int)((long long)n & 3);
    const float cc = (q & 1) ? s : c, ss = (q & 1) ? c : s;
    return make_float2((q == 1 || q == 2) ? -cc : cc, (q & 2) ? -ss : ss);
}

struct RopeParams {
    const char *qkv;
    char *q, *k, *v;
    long long ld_qkv, ld_q;                           // bytes
    long long page_stride, slot_stride, head_stride;  // bytes
    int n_tokens, n_q, n_kv, page_size, num_slots, rot, interleaved, tokens_per_cta;
    const int32_t *positions, *slots;
    const double *inv_freq;
    const float *q_norm, *k_norm;
    float eps, scale;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const RopeParams p) {
    constexpr int V = Vec<T>::N, L = HD / V;  // lanes of a head
    constexpr int kGroups = kThreads / L;
    __shared__ float2 cs[kMaxTokens][HD / 2];
    pdl_wait();
    pdl_trigger();
    const int t0 = blockIdx.x * p.tokens_per_cta;
    const int nt = min(p.tokens_per_cta, p.n_tokens - t0);
    const int heads = p.n_q + 2 * p.n_kv, items = nt * heads;
    const int group = threadIdx.x / L, li = threadIdx.x % L;
    const int half = p.rot / 2;
    const int off = half / V;  // lanes between the partners of the halves form
    bool have_angles = false;

    // item = token-major (token, head); the trip count is the same for every group of the CTA
    for (int base = 0; base < items; base += kGroups * kUnroll) {
        uint4 raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int it = base + u * kGroups + group;
            if (it < items)
                raw[u] = *reinterpret_cast<const uint4 *>(p.qkv + (t0 + it / heads) * p.ld_qkv +
                                                          (size_t)(it % heads) * HD * sizeof(T) + li * 16);
            else
                raw[u] = make_uint4(0, 0, 0, 0);
        }
        if (!have_angles) {
            for (int i = threadIdx.x; i < nt * half; i += kThreads) {
                const int t = i / half, f = i - t * half;
                float2 c = cos_sin(p.positions[t0 + t], p.inv_freq[f]);
                cs[t][f] = make_float2(c.x * p.scale, c.y * p.scale);
            }
            __syncthreads();
            have_angles = true;
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int it = base + u * kGroups + group;
            const int t = it < items ? it / heads : 0, h = it < items ? it - t * heads : 0;
            const bool is_q = h < p.n_q, is_v = h >= p.n_q + p.n_kv;
            float x[V];
            Vec<T>::load(raw[u], x);
            const float *w = is_v ? nullptr : is_q ? p.q_norm : p.k_norm;
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (w) {
                const float f = rms_factor(ss, HD, p.eps);
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = rms_scale(x[e], f, __ldg(w + li * V + e));
            }
            if (p.interleaved) {
                if (!is_v && li * V < p.rot) {
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float2 c = cs[t][(li * V + e) / 2];
                        const float a = x[e], b = x[e + 1];
                        x[e] = rope_rot(a, b, c.x, c.y, true);
                        x[e + 1] = rope_rot(b, a, c.x, c.y, false);
                    }
                }
            } else {
                const bool first = li < off, turns = li < 2 * off;
                const int src = first ? li + off : turns ? li - off : li;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float other = __shfl_sync(0xffffffffu, x[e], src, L);
                    if (!is_v && turns) {
                        const float2 c = cs[t][(first ? li : li - off) * V + e];
                        x[e] = rope_rot(x[e], other, c.x, c.y, first);
                    }
                }
            }
            if (it >= items) continue;
            const uint4 out = is_v ? raw[u] : Vec<T>::store(x);
            if (is_q) {
                *reinterpret_cast<uint4 *>(p.q + (t0 + t) * p.ld_q + (size_t)h * HD * sizeof(T) + li * 16) = out;
            } else {
                const int slot = __ldg(p.slots + t0 + t);
                if (slot >= 0 && slot < p.num_slots) {
                    const int page = slot / p.page_size, kh = is_v ? h - p.n_q - p.n_kv : h - p.n_q;
                    char *dst = (is_v ? p.v : p.k) + page * p.page_stride + (slot - page * p.page_size) * p.slot_stride +
                                kh * p.head_stride;
                    *reinterpret_cast<uint4 *>(dst + li * 16) = out;
                }
            }
        }
    }
}

}  // namespace

cudaError_t launch_qk_norm_rope(const pyxis_qk_norm_rope_args &a, const pyxis_kv_pages &kv, int num_sms,
                                cudaStream_t st) {
    const long long es = kv.dtype == PYXIS_DTYPE_F32 ? 4 : 2;
    RopeParams p;
    p.qkv = (const char *)a.qkv;
    p.q = (char *)a.q;
    p.k = (char *)kv.k;
    p.v = (char *)kv.v;
    p.ld_qkv = (long long)a.ld_qkv * es;
    p.ld_q = (long long)a.ld_q * es;
    p.page_stride = kv.page_stride * es;
    p.slot_stride = kv.slot_stride * es;
    p.head_stride = kv.head_stride * es;
    p.n_tokens = (int)a.n_tokens;
    p.n_q = a.n_q_heads;
    p.n_kv = kv.n_kv_heads;
    p.page_size = kv.page_size;
    p.num_slots = kv.num_pages * kv.page_size;
    p.rot = a.rotary_dim;
    p.interleaved = a.interleaved;
    // one token per CTA until the tokens cover the GPU a few times over
    p.tokens_per_cta = a.n_tokens <= (size_t)num_sms * 8 ? 1 : kMaxTokens;
    p.positions = a.positions;
    p.slots = a.slots;
    p.inv_freq = a.inv_freq;
    p.q_norm = a.q_norm;
    p.k_norm = a.k_norm;
    p.eps = a.eps;
    p.scale = a.rope_scale;
    const dim3 grid((unsigned)((a.n_tokens + p.tokens_per_cta - 1) / p.tokens_per_cta));
    if (kv.dtype == PYXIS_DTYPE_F32)
        return kv.head_dim == 128 ? launch_kernel(qk_norm_rope_kernel<float, 128>, grid, dim3(kThreads), 0, st, p)
                                  : launch_kernel(qk_norm_rope_kernel<float, 64>, grid, dim3(kThreads), 0, st, p);
    return kv.head_dim == 128 ? launch_kernel(qk_norm_rope_kernel<__nv_bfloat16, 128>, grid, dim3(kThreads), 0, st, p)
                              : launch_kernel(qk_norm_rope_kernel<__nv_bfloat16, 64>, grid, dim3(kThreads), 0, st, p);
}

}  // namespace pyxis
