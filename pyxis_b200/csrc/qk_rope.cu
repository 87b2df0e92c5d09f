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
// token are the same for all its heads: a warp takes a token (or a part of its heads), forms the
// angles once, in 64 bits (position * frequency has far more than 24 significant bits at far
// positions; reduced by multiples of pi/2 to [-pi/4, pi/4] before it is rounded to f32), while the
// first heads' loads are in flight, and keeps its factors in registers.  Warps share nothing, so
// one's angles overlap the others' traffic.
//
// Measured (16 query and 8 kv heads of 128): 16384 bf16 tokens with norms and 64 of 128 dimensions turned
// 49.5 us, 5.4 TB/s of reads and writes (84 % of a plain copy's rate; the rest is the 64-bit angles and the
// paged stores' order); one f32 token 5.5 us, a launch and three dependent accesses.
#include <cuda_bf16.h>

#include "common.cuh"
#include "serve.h"

namespace pyxis {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // accesses in flight per warp and kind

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
    int n_tokens, n_q, n_kv, page_size, num_slots, rot, interleaved, parts;
    const int32_t *positions, *slots;
    const double *inv_freq;
    const float *q_norm, *k_norm;
    float eps, scale;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const RopeParams p) {
    constexpr int V = Vec<T>::N, L = HD / V;  // lanes of a head
    constexpr int kHeads = 32 / L, kHead = HD * (int)sizeof(T);  // heads of a warp's access
    __shared__ float2 cs[kThreads / 32][HD / 2];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int job = blockIdx.x * (kThreads / 32) + warp, t = job / p.parts, part = job - t * p.parts;
    if (t >= p.n_tokens) return;
    const int li = lane % L, sub = lane / L;
    const int half = p.rot / 2;
    const int off = half / V;  // lanes between the partners of the halves form
    const bool first = li < off, turns = p.interleaved ? li * V < p.rot : li < 2 * off;
    const int partner = first ? li + off : turns ? li - off : li;
    const int step = p.parts * kHeads, h0 = part * kHeads + sub;  // this lane group's heads: h0, h0 + step, ...
    const char *src = p.qkv + t * p.ld_qkv + li * 16;
    const char *ksrc = src + p.n_q * kHead, *vsrc = ksrc + p.n_kv * kHead;

    auto load = [&](const char *base, int h, int heads, uint4 (&raw)[kUnroll]) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            raw[u] = make_uint4(0, 0, 0, 0);
            if (h + u * step < heads) raw[u] = *reinterpret_cast<const uint4 *>(base + (h + u * step) * kHead);
        }
    };
    uint4 raw[kUnroll];
    load(src, h0, p.n_q, raw);  // on its way while the angles are formed
    const int slot = p.slots[t];
    // this lane's rotation factors: its pairs' (c, s), or with halves each of its elements' c and the
    // partner's signed s
    float2 f[V];
    if (p.rot) {
        const int pos = p.positions[t];
        for (int i = lane; i < half; i += 32) {
            const float2 c = cos_sin(pos, p.inv_freq[i]);
            cs[warp][i] = make_float2(c.x * p.scale, c.y * p.scale);
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < V; ++e) {
            f[e] = f2(1.f, 0.f);
            if (p.interleaved) {
                if (turns && e < V / 2) f[e] = cs[warp][li * (V / 2) + e];
            } else if (turns) {
                f[e] = cs[warp][(first ? li : li - off) * V + e];
                f[e].y = first ? -f[e].y : f[e].y;
            }
        }
    }
    auto weights = [&](const float *w, float (&out)[V]) {
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = w ? __ldg(w + li * V + e) : 1.f;
    };
    // a head's norm and rotation
    auto turn = [&](uint4 in, const float (&w)[V], bool norm) -> uint4 {
        float x[V];
        Vec<T>::load(in, x);
        if (norm) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = rsqrtf(fmaf(ss, 1.0f / HD, p.eps));
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] *= r * w[e];
        }
        if (p.rot) {
            if (p.interleaved) {
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const float a = x[e], b = x[e + 1];
                    x[e] = fmaf(a, f[e / 2].x, -(b * f[e / 2].y));
                    x[e + 1] = fmaf(b, f[e / 2].x, a * f[e / 2].y);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    x[e] = fmaf(x[e], f[e].x, __shfl_sync(0xffffffffu, x[e], partner, L) * f[e].y);
            }
        }
        return Vec<T>::store(x);
    };

    // queries, keys, values; the trip counts are the whole warp's
    float w[V];
    weights(p.q_norm, w);
    for (int h = h0, base = part * kHeads; base < p.n_q; h += step * kUnroll, base += step * kUnroll) {
        if (h != h0) load(src, h, p.n_q, raw);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (base + u * step >= p.n_q) break;  // of the whole warp
            const uint4 x = turn(raw[u], w, p.q_norm != nullptr);
            if (h + u * step < p.n_q)
                *reinterpret_cast<uint4 *>(p.q + t * p.ld_q + (h + u * step) * kHead + li * 16) = x;
        }
    }
    if (slot < 0 || slot >= p.num_slots) return;
    const int page = slot / p.page_size;
    const long long at = page * p.page_stride + (slot - page * p.page_size) * p.slot_stride + li * 16;
    weights(p.k_norm, w);
    for (int h = h0, base = part * kHeads; base < p.n_kv; h += step * kUnroll, base += step * kUnroll) {
        uint4 v[kUnroll];
        load(ksrc, h, p.n_kv, raw);
        load(vsrc, h, p.n_kv, v);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (base + u * step >= p.n_kv) break;
            const uint4 x = turn(raw[u], w, p.k_norm != nullptr);
            if (h + u * step < p.n_kv) {
                const long long to = at + (h + u * step) * p.head_stride;
                *reinterpret_cast<uint4 *>(p.k + to) = x;
                *reinterpret_cast<uint4 *>(p.v + to) = v[u];
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
    // a token's heads are dealt to up to 8 warps while the tokens alone do not fill the GPU
    p.parts = 1;
    while (p.parts < 8 && a.n_tokens * p.parts * 2 <= (size_t)num_sms * 32) p.parts *= 2;
    p.positions = a.positions;
    p.slots = a.slots;
    p.inv_freq = a.inv_freq;
    p.q_norm = a.q_norm;
    p.k_norm = a.k_norm;
    p.eps = a.eps;
    p.scale = a.rope_scale;
    const dim3 grid((unsigned)((a.n_tokens * p.parts + kThreads / 32 - 1) / (kThreads / 32)));
    if (kv.dtype == PYXIS_DTYPE_F32)
        return kv.head_dim == 128 ? launch_kernel(qk_norm_rope_kernel<float, 128>, grid, dim3(kThreads), 0, st, p)
                                  : launch_kernel(qk_norm_rope_kernel<float, 64>, grid, dim3(kThreads), 0, st, p);
    return kv.head_dim == 128 ? launch_kernel(qk_norm_rope_kernel<__nv_bfloat16, 128>, grid, dim3(kThreads), 0, st, p)
                              : launch_kernel(qk_norm_rope_kernel<__nv_bfloat16, 64>, grid, dim3(kThreads), 0, st, p);
}

}  // namespace pyxis
