// tree_attn.cu -- attention of a tree of drafted tokens over a paged KV cache
// (src/attention.rs:107-135 with pages, grouped heads and a per-node mask; definition in
// include/pyxis_serve.h), f32 or bf16, on the CUDA cores in f32.
//
//   s_rj = scale q_r . k_j;  m = max_j s_rj;  o_r = sum_j 2^(s_rj - m) v_j / sum_j 2^(s_rj - m)
//
// (scores in log2 units).  The rows of one (sequence, kv head) are its nodes times the G query
// heads that share the kv head, so a key is read once for all of them.  A CTA takes a tile of RT
// rows and a range of the keys (the host's split); its warps work through the range's 32-key blocks
// on their own, each with its own shared-memory buffers, running maximum, sum and output, so no
// barrier stands between the loads of one warp and the arithmetic of another.  The warps' results
// are joined in shared memory, the splits' by a second kernel.
//
// Within a block a lane first is a key: its key row lies in shared memory (rows padded by 16 bytes,
// so 16-byte reads of 32 rows do not collide), the query rows are broadcast reads.  For P V a lane
// is HD / 32 columns of the output and the probabilities are broadcast.  Rows arrive by one bulk
// copy each (an mbarrier per buffer): the next block's keys are under way during P V, its values
// during Q K.
//
// Measured (16 query and 8 kv heads of 128, f32, pages of 16): 64 sequences of 2303 positions, one node
// each, 194 us, 5.6 TB/s (a floor of 167 us at the rate of a plain copy): HBM bounds it up to 4 rows, its
// arithmetic from 8; one sequence of 152 positions 8.2 us, latency.  From 9 rows the products of f32 pages
// go to mma.sync in two tf32 terms (below; 16 rows over 16 x 2303 positions 90 us, a floor of 41: 12 warps
// per SM, which is what their buffers leave room for, and chains of dependent MMAs), more rows and bf16
// pages to tcgen05 (tree_attn_tc32.cu, tree_attn_tc.cu).
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "serve.h"
#include "tc_ptx.cuh"
#include "tree_attn.cuh"

namespace pyxis {
namespace {

constexpr int kBlock = 32;  // keys of a warp's block: one per lane
constexpr uint64_t kTimeoutNs = 2000000000ull;
enum { kErrLoad = 0x701, kErrDrain = 0x702 };

PYXIS_DEVINL float redux_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// Four consecutive elements of a row in shared memory as f32.
PYXIS_DEVINL float4 ld4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
PYXIS_DEVINL float4 ld4(const __nv_bfloat16 *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xFFFF0000u));
}
PYXIS_DEVINL float2 ld2(const float *p) { return *reinterpret_cast<const float2 *>(p); }
PYXIS_DEVINL float2 ld2(const __nv_bfloat16 *p) {
    const uint32_t u = *reinterpret_cast<const uint32_t *>(p);
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
// 16 bytes of T hold no infinity and no NaN.
template <typename T>
PYXIS_DEVINL bool all_finite(uint4 x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    bool ok = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ok = ok && (w[i] & 0x7F800000u) != 0x7F800000u;
        if (sizeof(T) == 2) ok = ok && (w[i] & 0x7F80u) != 0x7F80u;
    }
    return ok;
}
PYXIS_DEVINL float to_f32(float x) { return x; }
PYXIS_DEVINL float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
// Byte offset in the cache of the key at a position of the sequence; -1 past its last.
PYXIS_DEVINL long long key_offset(const TreeParams &p, const SeqShape &sh, int seq, int kvh, long long pos) {
    if (pos >= sh.total) return -1;
    // (a 32-bit division where the tables reach no further)
    const long long page_i = p.capacity >> 31 ? pos / p.page_size : (long long)((unsigned)pos / (unsigned)p.page_size);
    const int page = min(max(__ldg(p.block_table + seq * p.table_stride + page_i), 0), p.num_pages - 1);
    return page * p.page_stride + (pos - page_i * p.page_size) * p.slot_stride + kvh * p.head_stride;
}

// A block's rows into a warp's buffer: every lane with an offset copies its own.
template <uint32_t BYTES, int PITCH>
PYXIS_DEVINL void load_rows(const char *base, void *dst, uint64_t *bar, long long off, int lane) {
    const unsigned valid = __ballot_sync(0xffffffffu, off >= 0);
    if (lane == 0) tc::mbar_arrive_expect_tx(bar, __popc(valid) * BYTES);
    __syncwarp();
    if (off >= 0) tc::bulk_load(reinterpret_cast<char *>(dst) + lane * PITCH, base + off, BYTES, bar);
}

// Joins the warps' outputs (f32 [RT][HD] at the start of each warp's part of shared memory) by their
// maxima and sums, and writes the tile or its split's partial sums.
template <typename T, int HD, int RT, int WARPS>
PYXIS_DEVINL void join_warps(const TreeParams &p, const SeqShape &sh, const unsigned char *parts, int part_bytes,
                             const float *sml, int rows, int r0, int kvh, int split) {
    const int n_out = min(rows, RT) * HD;
    for (int i = threadIdx.x; i < n_out; i += WARPS * 32) {
        const int r = i / HD, d = i % HD;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sml[(w * RT + r) * 2]);
        const float base = m == -INFINITY ? 0.f : m;
        float o = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = exp2f(sml[(w * RT + r) * 2] - base);
            o = fmaf(f, reinterpret_cast<const float *>(parts + w * part_bytes)[r * HD + d], o);
            l = fmaf(f, sml[(w * RT + r) * 2 + 1], l);
        }
        const int t = (r0 + r) / p.group, head = kvh * p.group + (r0 + r) % p.group;
        const long long row = sh.row0 + t;
        if (p.splits == 1) {
            store(reinterpret_cast<T *>(p.out + row * p.out_row + head * p.out_head) + d, l == 0.f ? 0.f : o / l);
        } else {
            const long long at = (row * p.n_q + head) * p.splits + split;
            p.part_o[at * HD + d] = o;
            if (d == 0) p.part_ml[at * 2] = m, p.part_ml[at * 2 + 1] = l;
        }
    }
}

// PER: CTAs that share an SM.
template <typename T, int HD, int RT, int PER>
struct TreeCfg {
    static constexpr int kPitch = HD * (int)sizeof(T) + 16;          // bytes of a K or V row in shared memory
    static constexpr int kHalf = kBlock * kPitch;                    // a warp's K buffer (V follows)
    static constexpr int kPPitch = kBlock + 4;                       // floats of a row of probabilities
    static constexpr int kWarpBytes = 2 * kHalf + RT * kPPitch * 4;
    static constexpr int kQBytes = RT * HD * 4 + RT * 8 + 16;        // q, masks, abort flag
    static constexpr int kPerWarp = kWarpBytes + RT * 8 + 16;        // and its m and l, mbarriers
    static constexpr int kMost = PER == 1 ? 232448 : 115712;         // of 228 KB with 1 KB more per CTA
    static constexpr int kFit = (kMost - kQBytes) / kPerWarp;
    static constexpr int kWarps = kFit < 12 ? kFit : 12;
    static constexpr int kBytes = kQBytes + kWarps * kPerWarp;
    static_assert(RT * HD * 4 <= 2 * kHalf, "a warp's output fits its buffers");
    static_assert(kBytes <= kMost, "shared memory of an SM");
};

template <typename T, int HD, int RT, int PER>
__global__ void __launch_bounds__(TreeCfg<T, HD, RT, PER>::kWarps * 32) tree_attention_kernel(const TreeParams p) {
    using C = TreeCfg<T, HD, RT, PER>;
    constexpr int kWarps = C::kWarps, kCols = HD / 32;
    extern __shared__ __align__(128) unsigned char smem[];
    float *sq = reinterpret_cast<float *>(smem + kWarps * C::kWarpBytes);  // [RT][HD], times scale2
    unsigned long long *smask = reinterpret_cast<unsigned long long *>(sq + RT * HD);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smask + RT);  // [kWarps][2]: K, V
    float *sml = reinterpret_cast<float *>(bars + 2 * kWarps);  // [kWarps][RT][2]: maximum and sum
    volatile int *abort_flag = reinterpret_cast<volatile int *>(sml + kWarps * RT * 2);

    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x, kvh = blockIdx.y / p.row_tiles, r0 = (blockIdx.y % p.row_tiles) * RT, seq = blockIdx.z;
    const SeqShape sh = seq_shape(p, seq);
    const int rows = sh.nodes * p.group - r0;  // of this tile and later ones
    if (rows <= 0) return;
    const long long blocks = (sh.total + kBlock - 1) / kBlock;
    const long long b0 = blocks * split / p.splits, b1 = blocks * (split + 1) / p.splits;

    unsigned char *mine = smem + warp * C::kWarpBytes;
    T *sk = reinterpret_cast<T *>(mine), *sv = reinterpret_cast<T *>(mine + C::kHalf);
    float *sp = reinterpret_cast<float *>(mine + 2 * C::kHalf);
    uint64_t *kbar = bars + 2 * warp, *vbar = kbar + 1;
    if (lane == 0) {
        tc::mbar_init(kbar, 1);
        tc::mbar_init(vbar, 1);
        tc::fence_mbar_init();
    }
    if (threadIdx.x == 0) *abort_flag = 0;
    for (int i = threadIdx.x; i < RT * HD; i += kWarps * 32) {
        const int r = i / HD, d = i % HD;
        float x = 0.f;
        if (r < rows) {
            const int t = (r0 + r) / p.group, g = (r0 + r) % p.group;
            x = p.scale2 * to_f32(*reinterpret_cast<const T *>(p.q + (sh.row0 + t) * p.q_row +
                                                               (kvh * p.group + g) * p.q_head + d * sizeof(T)));
        }
        sq[i] = x;
    }
    if (threadIdx.x < RT) {
        unsigned long long m = 0;
        if ((int)threadIdx.x < rows) {
            const int t = (r0 + threadIdx.x) / p.group;
            m = p.tree_mask ? p.tree_mask[sh.row0 + t] : (2ull << t) - 1;
        }
        smask[threadIdx.x] = m;
    }
    __syncthreads();

    auto row_offset = [&](long long b) -> long long { return key_offset(p, sh, seq, kvh, b * kBlock + lane); };
    auto load = [&](const char *base, T *dst, uint64_t *bar, long long off) {
        load_rows<HD * sizeof(T), C::kPitch>(base, dst, bar, off, lane);
    };

    float2 acc[RT][kCols / 2];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < kCols / 2; ++c) acc[r][c] = make_float2(0.f, 0.f);
    float m_run = -INFINITY, l_run = 0.f;  // of row `lane` (lane < RT)

    bool ok = true;
    uint32_t phase = 0;
    long long b = b0 + warp;
    long long off = b < b1 ? row_offset(b) : -1;
    if (b < b1) {
        load(p.k, sk, kbar, off);
        load(p.v, sv, vbar, off);
    }
    for (; b < b1 && ok; b += kWarps, phase ^= 1) {
        const long long next_off = b + kWarps < b1 ? row_offset(b + kWarps) : -1;
        const long long pos = b * kBlock + lane;
        ok = __all_sync(0xffffffffu, tc::mbar_wait_bounded(kbar, phase, abort_flag, p.err, kErrLoad, kTimeoutNs));
        if (!ok) break;
        // ---- scores: this lane's key against every row
        float s[RT];
        {
            float2 s2[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) s2[r] = make_float2(0.f, 0.f);
            const T *krow = reinterpret_cast<const T *>(reinterpret_cast<const char *>(sk) + lane * C::kPitch);
#pragma unroll 4
            for (int d = 0; d < HD; d += 4) {
                const float4 kv = ld4(krow + d);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const float4 qv = ld4(sq + r * HD + d);
                    s2[r] = ffma2(f2(qv.x, qv.y), f2(kv.x, kv.y), s2[r]);
                    s2[r] = ffma2(f2(qv.z, qv.w), f2(kv.z, kv.w), s2[r]);
                }
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) s[r] = s2[r].x + s2[r].y;
        }
        __syncwarp();
        if (b + kWarps < b1) load(p.k, sk, kbar, next_off);
        const bool tail = (b + 1) * kBlock > sh.ctx;  // holds drafts or ends inside
        if (tail) {
            const long long draft = pos - sh.ctx;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const bool seen = draft < 0 ? true : pos < sh.total && ((smask[r] >> draft) & 1);
                if (!seen) s[r] = -INFINITY;
            }
        }
        // ---- running maximum, probabilities
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const float m_old = __shfl_sync(0xffffffffu, m_run, r);
            const float m_new = fmaxf(m_old, redux_max(s[r]));
            const float base = m_new == -INFINITY ? 0.f : m_new;  // nothing seen yet: p = 2^-inf = 0
            if (m_new > m_old) {
                const float alpha = exp2f(m_old - base);
#pragma unroll
                for (int c = 0; c < kCols / 2; ++c) acc[r][c].x *= alpha, acc[r][c].y *= alpha;
                if (lane == r) l_run *= alpha, m_run = m_new;
            }
            sp[r * C::kPPitch + lane] = exp2f(s[r] - base);
        }
        __syncwarp();
        if (lane < RT) {
            const float *row = sp + lane * C::kPPitch;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < kBlock; j += 4) {
                const float4 x = ld4(row + j);
                sum += (x.x + x.y) + (x.z + x.w);
            }
            l_run += sum;
        }
        ok = __all_sync(0xffffffffu, tc::mbar_wait_bounded(vbar, phase, abort_flag, p.err, kErrLoad, kTimeoutNs));
        if (!ok) break;
        // ---- O += P V: this lane's columns
        const int nk = tail ? (int)min((long long)kBlock, sh.total - b * kBlock) : kBlock;
        // Whether every value is fit to be multiplied by a weight of zero.  Few rows go key by key
        // without looking: the look at 32 rows of values costs more (one token over 152 f32 positions: 12 us
        // with it, 8 without).
        bool plain = !tail;
        if (RT > 4 && tail) {
            char *row = reinterpret_cast<char *>(sv) + lane * C::kPitch;
            bool finite = true;
#pragma unroll 8
            for (int i = 0; i < HD * (int)sizeof(T) / 16; ++i) {
                uint4 *x = reinterpret_cast<uint4 *>(row) + i;
                if (lane >= nk)
                    *x = make_uint4(0, 0, 0, 0);  // never loaded
                else
                    finite = finite && all_finite<T>(*x);
            }
            plain = __all_sync(0xffffffffu, finite);
            tc::fence_proxy_async_smem();  // the buffer's next copy comes after these stores
            __syncwarp();
        }
        if (plain) {
#pragma unroll 2
            for (int j = 0; j < kBlock; j += 4) {
                float2 v[4][kCols / 2];
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const T *vrow = reinterpret_cast<const T *>(reinterpret_cast<const char *>(sv) + (j + jj) * C::kPitch) +
                                    lane * kCols;
                    if constexpr (kCols == 4) {
                        const float4 x = ld4(vrow);
                        v[jj][0] = f2(x.x, x.y), v[jj][1] = f2(x.z, x.w);
                    } else {
                        v[jj][0] = ld2(vrow);
                    }
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const float4 pr = ld4(sp + r * C::kPPitch + j);
#pragma unroll
                    for (int c = 0; c < kCols / 2; ++c) {
                        acc[r][c] = ffma2(f2(pr.x, pr.x), v[0][c], acc[r][c]);
                        acc[r][c] = ffma2(f2(pr.y, pr.y), v[1][c], acc[r][c]);
                        acc[r][c] = ffma2(f2(pr.z, pr.z), v[2][c], acc[r][c]);
                        acc[r][c] = ffma2(f2(pr.w, pr.w), v[3][c], acc[r][c]);
                    }
                }
            }
        } else {
            // a value that is not finite reaches the rows that see it, and no others: key by key, a weight
            // of zero leaves the value out (the other rows' sums are those of the loop above, bit for bit)
            for (int j = 0; j < nk; ++j) {
                const T *vrow = reinterpret_cast<const T *>(reinterpret_cast<const char *>(sv) + j * C::kPitch) + lane * kCols;
                float2 v[kCols / 2];
#pragma unroll
                for (int c = 0; c < kCols / 2; ++c) v[c] = ld2(vrow + 2 * c);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const float pr = sp[r * C::kPPitch + j];
                    if (pr != 0.f) {
#pragma unroll
                        for (int c = 0; c < kCols / 2; ++c) acc[r][c] = ffma2(f2(pr, pr), v[c], acc[r][c]);
                    }
                }
            }
        }
        __syncwarp();
        if (b + kWarps < b1) load(p.v, sv, vbar, next_off);
    }
    if (!ok) {  // a copy did not land in time: give those in flight a last chance before the buffers go
        volatile int never = 0;
        tc::mbar_wait_bounded(kbar, phase, &never, p.err, kErrDrain, 100000000ull);
        tc::mbar_wait_bounded(vbar, phase, &never, p.err, kErrDrain, 100000000ull);
    }

    // ---- join the warps: their outputs go where their K and V were
    __syncwarp();
    float *so = reinterpret_cast<float *>(mine);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < kCols / 2; ++c)
            *reinterpret_cast<float2 *>(so + r * HD + lane * kCols + 2 * c) = acc[r][c];
    if (lane < RT) sml[(warp * RT + lane) * 2] = m_run, sml[(warp * RT + lane) * 2 + 1] = l_run;
    __syncthreads();
    join_warps<T, HD, RT, kWarps>(p, sh, smem, C::kWarpBytes, sml, rows, r0, kvh, split);
}

// The same with the products on the tensor cores (mma.sync m16n8k8, tf32), for more rows than the
// CUDA cores' FMAs keep up with: a warp's 16-key block against MT tiles of 16 rows.  f32 operands are
// split into two tf32 terms and multiplied as lo.hi + hi.lo + hi.hi, which leaves 2^-22 of a product;
// bf16 operands are tf32 numbers already, only the probabilities are split.
// A fragment's k index may name the dims (keys) in any order that both operands share: lane c of a
// quad takes dims 4c .. 4c + 3 of 16 with one 16-byte read, keys 2c and 2c + 1 of 8 (the columns of S
// that it holds), and an output tile's columns are every fourth dim, so V is read 16 bytes at a time
// and P never leaves its registers.
struct Split {
    uint32_t hi, lo;
};
template <bool TWO>
PYXIS_DEVINL Split split(float x) {
    if constexpr (!TWO) return Split{__float_as_uint(x), 0u};
    // tf32 is the upper 19 bits, and the multiplier drops the rest: hi is x cut off (no overflow), lo
    // the remainder rounded (half a step added before its cut), off by 2^-23 of x
    const uint32_t h = __float_as_uint(x) & 0xffffe000u;
    return Split{h, __float_as_uint(x - __uint_as_float(h)) + 0x1000u};
}
PYXIS_DEVINL void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// q . k in f32, q as its two terms.
template <int HD>
__device__ __noinline__ float shared_score(const float *hi, const float *lo, const float *k) {
    float x = 0.f;
#pragma unroll 4
    for (int d = 0; d < HD; ++d) x = fmaf(hi[d] + lo[d], k[d], x);
    return x;
}

constexpr int kMmaKeys = 16;  // keys of a warp's block here: small buffers, so that more warps fit an SM

template <typename T, int HD, int MT, int PER>
struct MmaCfg {
    static constexpr bool kTwo = sizeof(T) == 4;                     // operands of two tf32 terms
    static constexpr int kRows = 16 * MT, kQPitch = HD + 4;          // floats of a query row in shared memory
    static constexpr int kPitch = HD * (int)sizeof(T) + 16, kHalf = kMmaKeys * kPitch;
    static constexpr int kQBytes = (kTwo ? 2 : 1) * kRows * kQPitch * 4 + kRows * 8 + 16;
    static constexpr int kWarpBytes = 2 * kHalf > kRows * HD * 4 ? 2 * kHalf : kRows * HD * 4;  // K, V; then the output
    static constexpr int kPerWarp = kWarpBytes + kRows * 8 + 16;
    static constexpr int kFit = ((PER == 1 ? 232448 : 115712) - kQBytes) / kPerWarp;
    static constexpr int kMost = (MT == 1 ? 12 : 8) / PER;  // 168 or 255 registers a thread
    static constexpr int kWarps = kFit < kMost ? kFit : kMost;
    static constexpr int kBytes = kQBytes + kWarps * kPerWarp;
};

template <typename T, int HD, int MT, int PER>
__global__ void __launch_bounds__(MmaCfg<T, HD, MT, PER>::kWarps * 32, PER) tree_attention_mma_kernel(const TreeParams p) {
    using C = MmaCfg<T, HD, MT, PER>;
    constexpr int kWarps = C::kWarps, RT = C::kRows;
    constexpr bool kTwo = C::kTwo;
    constexpr int kTiles = kMmaKeys / 8;
    extern __shared__ __align__(128) unsigned char smem[];
    float *sq = reinterpret_cast<float *>(smem + kWarps * C::kWarpBytes);  // [hi, lo][RT][kQPitch], times scale2
    unsigned long long *smask = reinterpret_cast<unsigned long long *>(sq + (kTwo ? 2 : 1) * RT * C::kQPitch);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smask + RT);
    float *sml = reinterpret_cast<float *>(bars + 2 * kWarps);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(sml + kWarps * RT * 2);

    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int split_i = blockIdx.x, kvh = blockIdx.y / p.row_tiles, r0 = (blockIdx.y % p.row_tiles) * RT, seq = blockIdx.z;
    const SeqShape sh = seq_shape(p, seq);
    const int rows = sh.nodes * p.group - r0;
    if (rows <= 0) return;
    const long long blocks = (sh.total + kMmaKeys - 1) / kMmaKeys;
    const long long b0 = blocks * split_i / p.splits, b1 = blocks * (split_i + 1) / p.splits;

    unsigned char *mine = smem + warp * C::kWarpBytes;
    T *sk = reinterpret_cast<T *>(mine), *sv = reinterpret_cast<T *>(mine + C::kHalf);
    uint64_t *kbar = bars + 2 * warp, *vbar = kbar + 1;
    if (lane == 0) {
        tc::mbar_init(kbar, 1);
        tc::mbar_init(vbar, 1);
        tc::fence_mbar_init();
    }
    if (threadIdx.x == 0) *abort_flag = 0;
    for (int i = threadIdx.x; i < RT * HD; i += kWarps * 32) {
        const int r = i / HD, d = i % HD;
        float x = 0.f;
        if (r < rows) {
            const int t = (r0 + r) / p.group, gg = (r0 + r) % p.group;
            x = to_f32(*reinterpret_cast<const T *>(p.q + (sh.row0 + t) * p.q_row + (kvh * p.group + gg) * p.q_head + d * sizeof(T)));
        }
        // f32: times the scale, in two terms; bf16: as it is (the scale follows in f32)
        const Split s = split<kTwo>(kTwo ? x * p.scale2 : x);
        sq[r * C::kQPitch + d] = __uint_as_float(s.hi);
        if (kTwo) sq[(RT + r) * C::kQPitch + d] = __uint_as_float(s.lo);
    }
    if (threadIdx.x < RT) {
        unsigned long long m = 0;
        if ((int)threadIdx.x < rows) {
            const int t = (r0 + threadIdx.x) / p.group;
            m = p.tree_mask ? p.tree_mask[sh.row0 + t] : (2ull << t) - 1;
        }
        smask[threadIdx.x] = m;
    }
    __syncthreads();

    auto row_offset = [&](long long b) -> long long { return lane < kMmaKeys ? key_offset(p, sh, seq, kvh, b * kMmaKeys + lane) : -1; };
    auto load = [&](const char *base, T *dst, uint64_t *bar, long long off) {
        load_rows<HD * sizeof(T), C::kPitch>(base, dst, bar, off, lane);
    };
    float acc[MT][HD / 8][4];  // tile 4 j + e, column n: dim 32 j + 4 n + e
    float m_run[MT][2], l_run[MT][2];  // rows g and g + 8 of each tile; l: this lane's keys only
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[mt][i][k] = 0.f;
        m_run[mt][0] = m_run[mt][1] = -INFINITY;
        l_run[mt][0] = l_run[mt][1] = 0.f;
    }
    bool ok = true;
    uint32_t phase = 0;
    long long b = b0 + warp;
    long long off = b < b1 ? row_offset(b) : -1;
    if (b < b1) {
        load(p.k, sk, kbar, off);
        load(p.v, sv, vbar, off);
    }
    for (; b < b1 && ok; b += kWarps, phase ^= 1) {
        const long long next_off = b + kWarps < b1 ? row_offset(b + kWarps) : -1;
        ok = __all_sync(0xffffffffu, tc::mbar_wait_bounded(kbar, phase, abort_flag, p.err, kErrLoad, kTimeoutNs));
        if (!ok) break;
        // ---- S: columns nt * 8 + 2 c, + 1 of rows g, g + 8
        float s[MT][kTiles][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[mt][nt][k] = 0.f;
#pragma unroll 2
        for (int d = 4 * c; d < HD; d += 16) {
            Split kf[kTiles][4];
#pragma unroll
            for (int nt = 0; nt < kTiles; ++nt) {
                const float4 x = ld4(reinterpret_cast<const T *>(reinterpret_cast<const char *>(sk) + (nt * 8 + g) * C::kPitch) + d);
                kf[nt][0] = split<kTwo>(x.x), kf[nt][1] = split<kTwo>(x.y), kf[nt][2] = split<kTwo>(x.z), kf[nt][3] = split<kTwo>(x.w);
            }
            // products of one kind for all tiles before the next kind: no MMA waits for the one before
            uint4 h0[MT], h1[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float *q0 = sq + (mt * 16 + g) * C::kQPitch + d;
                h0[mt] = *reinterpret_cast<const uint4 *>(q0);
                h1[mt] = *reinterpret_cast<const uint4 *>(q0 + 8 * C::kQPitch);
            }
            if constexpr (kTwo) {
                uint4 l0[MT], l1[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const float *q0 = sq + (RT + mt * 16 + g) * C::kQPitch + d;
                    l0[mt] = *reinterpret_cast<const uint4 *>(q0);
                    l1[mt] = *reinterpret_cast<const uint4 *>(q0 + 8 * C::kQPitch);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < kTiles; ++nt)
                        mma_tf32(s[mt][nt], l0[mt].x, l1[mt].x, l0[mt].y, l1[mt].y, kf[nt][0].hi, kf[nt][1].hi);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < kTiles; ++nt)
                        mma_tf32(s[mt][nt], l0[mt].z, l1[mt].z, l0[mt].w, l1[mt].w, kf[nt][2].hi, kf[nt][3].hi);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < kTiles; ++nt)
                        mma_tf32(s[mt][nt], h0[mt].x, h1[mt].x, h0[mt].y, h1[mt].y, kf[nt][0].lo, kf[nt][1].lo);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < kTiles; ++nt)
                        mma_tf32(s[mt][nt], h0[mt].z, h1[mt].z, h0[mt].w, h1[mt].w, kf[nt][2].lo, kf[nt][3].lo);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < kTiles; ++nt)
                    mma_tf32(s[mt][nt], h0[mt].x, h1[mt].x, h0[mt].y, h1[mt].y, kf[nt][0].hi, kf[nt][1].hi);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < kTiles; ++nt)
                    mma_tf32(s[mt][nt], h0[mt].z, h1[mt].z, h0[mt].w, h1[mt].w, kf[nt][2].hi, kf[nt][3].hi);
        }
        if constexpr (kTwo) {
            // A key with an infinity has no second term, and a query's may be zero: scores that are not finite
            // are taken again in f32.
            float z = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) z = fmaf(s[mt][nt][k], 0.f, z);
            if (__any_sync(0xffffffffu, isnan(z))) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (!isfinite(s[mt][nt][k])) {
                                const float *q = sq + (mt * 16 + g + 8 * (k >> 1)) * C::kQPitch;
                                s[mt][nt][k] = shared_score<HD>(q, q + RT * C::kQPitch, reinterpret_cast<const float *>(reinterpret_cast<const char *>(sk) + (nt * 8 + 2 * c + (k & 1)) * C::kPitch));
                            }
            }
        }
        __syncwarp();
        if (b + kWarps < b1) load(p.k, sk, kbar, next_off);
        const bool tail = (b + 1) * kMmaKeys > sh.ctx;  // holds drafts or ends inside
        if (!kTwo) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[mt][nt][k] *= p.scale2;
        }
        if (tail) {
            const long long d0 = b * kMmaKeys - sh.ctx;  // draft of column 0
            const int avail = (int)(sh.total - sh.ctx);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const unsigned long long m = smask[mt * 16 + g + 8 * h];
#pragma unroll
                    for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const long long d = d0 + nt * 8 + 2 * c + i;
                            if (d >= 0 && (d >= avail || !((m >> d) & 1))) s[mt][nt][2 * h + i] = -INFINITY;
                        }
                }
        }
        // ---- running maximum, probabilities
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float top = fmaxf(s[mt][0][2 * h], s[mt][0][2 * h + 1]);
#pragma unroll
                for (int nt = 1; nt < kTiles; ++nt) top = fmaxf(top, fmaxf(s[mt][nt][2 * h], s[mt][nt][2 * h + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // the reference is raised only by more than 2^8: the weights stay below that, and their
                // f32 precision is the same
                const bool raise = top > m_run[mt][h] + 8.f || (m_run[mt][h] == -INFINITY && top > m_run[mt][h]);
                if (__any_sync(0xffffffffu, raise)) {
                    const float alpha = raise ? exp2f(m_run[mt][h] - top) : 1.f;
                    if (raise) m_run[mt][h] = top;
                    l_run[mt][h] *= alpha;
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i) acc[mt][i][2 * h] *= alpha, acc[mt][i][2 * h + 1] *= alpha;
                }
                const float base = m_run[mt][h] == -INFINITY ? 0.f : m_run[mt][h];
#pragma unroll
                for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float x = exp2f(s[mt][nt][2 * h + i] - base);
                        s[mt][nt][2 * h + i] = x;
                        l_run[mt][h] += x;
                    }
            }
        ok = __all_sync(0xffffffffu, tc::mbar_wait_bounded(vbar, phase, abort_flag, p.err, kErrLoad, kTimeoutNs));
        if (!ok) break;
        // ---- O += P V
        if (tail) {
            // every value has to be fit to be multiplied by a weight of zero
            const int nk = (int)min((long long)kMmaKeys, sh.total - b * kMmaKeys);
            char *row = reinterpret_cast<char *>(sv) + lane * C::kPitch;
            bool finite = true;
#pragma unroll 8
            for (int i = 0; i < (lane < kMmaKeys ? HD * (int)sizeof(T) / 16 : 0); ++i) {
                uint4 *x = reinterpret_cast<uint4 *>(row) + i;
                if (lane >= nk)
                    *x = make_uint4(0, 0, 0, 0);  // never loaded
                else
                    finite = finite && all_finite<T>(*x);
            }
            tc::fence_proxy_async_smem();  // the buffer's next copy comes after these stores
            __syncwarp();
            unsigned odd = __ballot_sync(0xffffffffu, !finite);
            if (odd) {
                // a value that is not finite reaches the rows that see it, and no others: those get it
                // here, then it becomes zero
                for (unsigned rest = odd; rest; rest &= rest - 1) {
                    const int k = __ffs(rest) - 1;
                    const T *vrow = reinterpret_cast<const T *>(reinterpret_cast<const char *>(sv) + k * C::kPitch);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            // key k's weight: by masks, as an index would move s out of the registers
                            uint32_t bits = 0;
#pragma unroll
                            for (int i = 0; i < 2 * kTiles; ++i)
                                bits |= __float_as_uint(s[mt][i >> 1][2 * h + (i & 1)]) &
                                        (((k >> 3) * 2 + (k & 1)) == i ? 0xffffffffu : 0u);
                            const float w = __uint_as_float(__shfl_sync(0xffffffffu, bits, (lane & ~3) | ((k >> 1) & 3)));
#pragma unroll
                            for (int i = 0; i < HD / 8; ++i)
#pragma unroll
                                for (int n = 0; n < 2; ++n) {
                                    const float x = to_f32(vrow[32 * (i >> 2) + 4 * (2 * c + n) + (i & 3)]);
                                    if (w != 0.f && !isfinite(x)) acc[mt][i][2 * h + n] += x;
                                }
                        }
                }
                __syncwarp();
                if (!finite)
                    for (int i = 0; i < HD; ++i)
                        if (!isfinite(to_f32(reinterpret_cast<const T *>(row)[i]))) store(reinterpret_cast<T *>(row) + i, 0.f);
                tc::fence_proxy_async_smem();
                __syncwarp();
            }
        }
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt) {
            Split a[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                a[mt][0] = split<true>(s[mt][nt][0]), a[mt][1] = split<true>(s[mt][nt][2]);
                a[mt][2] = split<true>(s[mt][nt][1]), a[mt][3] = split<true>(s[mt][nt][3]);
            }
            const char *v0 = reinterpret_cast<const char *>(sv) + (nt * 8 + 2 * c) * C::kPitch;
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                const float4 x = ld4(reinterpret_cast<const T *>(v0) + 32 * j + 4 * g);
                const float4 y = ld4(reinterpret_cast<const T *>(v0 + C::kPitch) + 32 * j + 4 * g);
                const float xe[4] = {x.x, x.y, x.z, x.w}, ye[4] = {y.x, y.y, y.z, y.w};
                Split u[4], v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] = split<kTwo>(xe[e]), v[e] = split<kTwo>(ye[e]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        mma_tf32(acc[mt][4 * j + e], a[mt][0].lo, a[mt][1].lo, a[mt][2].lo, a[mt][3].lo, u[e].hi, v[e].hi);
                if constexpr (kTwo) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            mma_tf32(acc[mt][4 * j + e], a[mt][0].hi, a[mt][1].hi, a[mt][2].hi, a[mt][3].hi, u[e].lo, v[e].lo);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        mma_tf32(acc[mt][4 * j + e], a[mt][0].hi, a[mt][1].hi, a[mt][2].hi, a[mt][3].hi, u[e].hi, v[e].hi);
            }
        }
        __syncwarp();
        if (b + kWarps < b1) load(p.v, sv, vbar, next_off);
    }
    if (!ok) {  // a copy did not land in time: give those in flight a last chance before the buffers go
        volatile int never = 0;
        tc::mbar_wait_bounded(kbar, phase, &never, p.err, kErrDrain, 100000000ull);
        tc::mbar_wait_bounded(vbar, phase, &never, p.err, kErrDrain, 100000000ull);
    }

    // ---- join the warps: their outputs go where their K and V were
    __syncwarp();
    float *so = reinterpret_cast<float *>(mine), odd = 0.f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = mt * 16 + g + 8 * h;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    so[r * HD + 32 * (i >> 2) + 4 * (2 * c + n) + (i & 3)] = acc[mt][i][2 * h + n];
                    odd = fmaf(acc[mt][i][2 * h + n], 0.f, odd);
                }
            float l = l_run[mt][h];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (c == 0) sml[(warp * RT + r) * 2] = m_run[mt][h], sml[(warp * RT + r) * 2 + 1] = l;
        }
    if (__any_sync(0xffffffffu, isnan(odd))) {
        // A weight's second term may be zero, and an infinite value has none: a sum over values that are not
        // finite is taken from the values of this warp's blocks, a row per lane (one whose weights are NaN is NaN).
        __syncwarp();
        constexpr int kC = HD / 32;  // columns per lane
        float4 bad = make_float4(0.f, 0.f, 0.f, 0.f);
        for (b = b0 + warp; b < b1; b += kWarps) {
            const float4 x = odd_columns<T, kC>(p, sh, seq, kvh, 0, b * kMmaKeys, (b + 1) * kMmaKeys);
            bad.x += x.x, bad.y += x.y, bad.z += x.z, bad.w += x.w;
        }
        const bool mine = lane < min(rows, RT) && isfinite(sml[(warp * RT + lane) * 2 + 1]);
#pragma unroll 1
        for (int d = 0; d < HD; ++d) {
            const int e = d % kC;
            float x = __shfl_sync(0xffffffffu, e == 0 ? bad.x : e == 1 ? bad.y : e == 2 ? bad.z : bad.w, d / kC);
            if (!mine || isfinite(so[lane * HD + d])) continue;
            for (b = b0 + warp; b < b1; b += kWarps)
                x += odd_drafts<T>(p, sh, seq, kvh, d, smask[lane], b * kMmaKeys, (b + 1) * kMmaKeys);
            if (x != 0.f) so[lane * HD + d] = x;
        }
    }
    __syncthreads();
    join_warps<T, HD, RT, kWarps>(p, sh, smem, C::kWarpBytes, sml, rows, r0, kvh, split_i);
}

// Joins the splits: a warp per (node, query head).
template <typename T, int HD>
__global__ void __launch_bounds__(256) tree_join_kernel(const TreeParams p) {
    constexpr int kCols = HD / 32;
    pdl_wait();
    pdl_trigger();
    const int item = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, seq = blockIdx.y;
    const SeqShape sh = seq_shape(p, seq);
    const int t = item / p.n_q, head = item % p.n_q;
    if (t >= sh.nodes) return;
    const long long row = sh.row0 + t, at = (row * p.n_q + head) * p.splits;
    // a batch of the splits' sums in flight at a time: one latency each, not one per split (one tree of 8
    // nodes over 26000 f32 positions, 102 splits: 43 us with four, 35 with sixteen)
    constexpr int kBatch = 16;
    float o[kCols] = {}, l = 0.f, m = -INFINITY;
    for (int s0 = 0; s0 < p.splits; s0 += kBatch) {
        float2 ml[kBatch], x[kBatch][kCols / 2];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const bool there = s0 + k < p.splits;
            ml[k] = there ? reinterpret_cast<const float2 *>(p.part_ml)[at + s0 + k] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int c = 0; c < kCols / 2; ++c)
                x[k][c] = there ? reinterpret_cast<const float2 *>(p.part_o + (at + s0 + k) * HD + lane * kCols)[c]
                                : make_float2(0.f, 0.f);
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) top = fmaxf(top, ml[k].x);
        const float base = top == -INFINITY ? 0.f : top, old = exp2f(m - base);
        m = top;
        l *= old;
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[c] *= old;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float f = exp2f(ml[k].x - base);
            l = fmaf(f, ml[k].y, l);
#pragma unroll
            for (int c = 0; c < kCols / 2; ++c) {
                o[2 * c] = fmaf(f, x[k][c].x, o[2 * c]);
                o[2 * c + 1] = fmaf(f, x[k][c].y, o[2 * c + 1]);
            }
        }
    }
    T *dst = reinterpret_cast<T *>(p.out + row * p.out_row + head * p.out_head) + lane * kCols;
#pragma unroll
    for (int c = 0; c < kCols; ++c) store(dst + c, l == 0.f ? 0.f : o[c] / l);
}

template <typename T, int HD>
cudaError_t run_kernel(void (*kern)(TreeParams), int threads, int smem, std::atomic<uint64_t> &done, const TreeParams &p,
                       size_t n_seq, cudaStream_t st) {
    cudaError_t e =
        once_per_device(done, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (e != cudaSuccess) return e;
    PdlScope pdl;
    for (size_t s = 0; s < n_seq; s += 65535) {  // grid.z
        TreeParams q = p;
        q.q_start += s, q.context_len += s, q.block_table += s * p.table_stride;
        const unsigned m = (unsigned)std::min<size_t>(n_seq - s, 65535);
        e = launch_kernel(kern, dim3(p.splits, p.n_kv * p.row_tiles, m), dim3(threads), smem, st, q);
        if (e == cudaSuccess && p.splits > 1)
            e = launch_kernel(tree_join_kernel<T, HD>, dim3((p.max_tree * p.n_q + 7) / 8, m), dim3(256), 0, st, q);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}
template <typename T, int HD, int RT, int PER>
cudaError_t run_fma(const TreeParams &p, size_t n_seq, cudaStream_t st) {
    using C = TreeCfg<T, HD, RT, PER>;
    static std::atomic<uint64_t> done{0};
    return run_kernel<T, HD>(tree_attention_kernel<T, HD, RT, PER>, C::kWarps * 32, C::kBytes, done, p, n_seq, st);
}
template <typename T, int HD, int MT, int PER>
cudaError_t run_mma(const TreeParams &p, size_t n_seq, cudaStream_t st) {
    using C = MmaCfg<T, HD, MT, PER>;
    static std::atomic<uint64_t> done{0};
    return run_kernel<T, HD>(tree_attention_mma_kernel<T, HD, MT, PER>, C::kWarps * 32, C::kBytes, done, p, n_seq, st);
}

template <typename T, int HD>
cudaError_t run_tree(const TreeParams &p, const TreePlan &t, size_t n_seq, cudaStream_t st) {
    switch (t.row_tile) {
    case 2: return t.per_sm == 1 ? run_fma<T, HD, 2, 1>(p, n_seq, st) : run_fma<T, HD, 2, 2>(p, n_seq, st);
    case 4: return t.per_sm == 1 ? run_fma<T, HD, 4, 1>(p, n_seq, st) : run_fma<T, HD, 4, 2>(p, n_seq, st);
    case 8: return t.per_sm == 1 ? run_fma<T, HD, 8, 1>(p, n_seq, st) : run_fma<T, HD, 8, 2>(p, n_seq, st);
    case 16: return t.per_sm == 1 ? run_mma<T, HD, 1, 1>(p, n_seq, st) : run_mma<T, HD, 1, 2>(p, n_seq, st);
    default: return t.per_sm == 1 ? run_mma<T, HD, 2, 1>(p, n_seq, st) : run_mma<T, HD, 2, 2>(p, n_seq, st);
    }
}

}  // namespace

TreePlan plan_tree_attention(const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv, int num_sms) {
    TreePlan t{false, 0, 1, 1, 1};
    const long long rows = (long long)a.max_tree * (a.n_q_heads / kv.n_kv_heads);
    const long long keys = std::max<long long>(1, std::min<long long>(std::min<long long>(a.max_context, 1ll << 40) + a.max_tree,
                                                                     (long long)a.table_width * kv.page_size));
    // bf16: few rows over few keys are done on the CUDA cores before the tensor-core kernel has started
    // its pipeline.  Measured (16 query heads, 8 kv heads of 128): 2 rows, one sequence of 152 positions 7 us
    // against 14, 16 of 600 12 against 21, of 2303 40 against 38, 64 of 600 43 against 49, of 1200 72 against
    // 67; 4 rows, 16 of 600 15 against 22, of 1200 30 against 28; 8 rows, 4 of 600 18 against 17, 16 of 600 26
    // against 21, of 300 17 against 19.
    // f32: the tcgen05 kernel pays the same for 1 row as for 128 (three products of 128 rows and the
    // conversion of every key), the mma.sync kernel for each tile of 16.  16 sequences of 2303 positions:
    // 16 rows 88 us against the tcgen05 kernel's 104, 32 rows 160 against 103, 64 rows 270 against 105;
    // one sequence of 152: 16 rows 15 against 23, 128 rows 29 against 27.  Trees over next to no context are
    // done before its pipeline has started: 4 sequences of 86 keys and 48 rows 21 against 23, 16 of 17 keys
    // and 128 rows of one kv head 20 against 33; 4 of 224 keys 28 against 25, and 512 CTAs' worth, 16 of 65
    // keys and 128 rows, 58 against 36.
    const bool f32 = kv.dtype == PYXIS_DTYPE_F32;
    const bool brief = keys <= 128 && (long long)a.n_seq * kv.n_kv_heads * ((rows + 31) / 32) <= num_sms;
    t.tensor = f32 ? tree_attention_tc32_supported(a, kv) && rows > 16 && !brief
                   : tree_attention_tc_supported(a, kv) &&
                         (rows > 4 || (double)a.n_seq * kv.n_kv_heads * keys * rows > 640e3);
    if (t.tensor) return t;
    t.row_tile = 2;
    while (t.row_tile < 32 && t.row_tile < rows) t.row_tile *= 2;
    t.row_tiles = (int)((rows + t.row_tile - 1) / t.row_tile);
    // Much work: two CTAs of half the warps to an SM, so that one's start and end overlap the other's loads.
    // Measured (8 kv heads, f32, one node): 64 sequences of 2303 positions 195 us against 197, with heads of
    // 64 104 against 125, 20 sequences of 800 39 against 47, 4 of 40000 199 against 209; the other way round
    // one sequence of 152 12 against 9, of 9000 30 against 27, 16 of 2303 and 2 nodes 68 against 66.
    // With mma.sync (8 nodes) 64 sequences of 1200 182 against 211, 20 of 800 67 against 82, but 4 of 40000
    // 325 against 282.
    const long long units = (long long)a.n_seq * kv.n_kv_heads * t.row_tiles;
    t.per_sm = units >= num_sms || (t.row_tile <= 8 && (double)units * keys >= 4096.0 * num_sms) ? 2 : 1;
    // the split that wastes least of the last wave, a split costing about 32 KB of f32 keys of start-up (20
    // sequences of 800 43 -> 39 us with that instead of 64 KB for two CTAs per SM), 64 or 128 bf16 ones
    const long long slots = (long long)num_sms * t.per_sm;
    // (partial sums are kept by query row: not more of them than 256 MB, however long the buffer of rows is)
    const double split_bytes = std::max(1.0, (double)a.n_rows * a.n_q_heads * (kv.head_dim + 2) * 4);
    const long long most = std::min({256ll, (keys + 255) / 256, std::max(1ll, (long long)(268435456.0 / split_bytes))});
    const double start = f32 ? 64.0 * 128 / kv.head_dim : 64.0 * t.per_sm;
    double best = 0;
    t.splits = 1;
    for (long long s = 1; s <= most; ++s) {
        const double waves = (double)((units * s + slots - 1) / slots);
        const double cost = waves * ((double)keys / s + start) + (s > 1 ? 128.0 : 0.0);
        if (s == 1 || cost < best * 0.98) best = cost, t.splits = (int)s;
    }
    return t;
}

size_t tree_attention_workspace(const TreePlan &t, const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv,
                                int num_sms) {
    if (t.tensor)
        return kv.dtype == PYXIS_DTYPE_F32 ? tree_attention_tc32_workspace(kv, num_sms) : tree_attention_tc_workspace(kv, num_sms);
    return t.splits == 1 ? 0 : a.n_rows * a.n_q_heads * t.splits * (size_t)(kv.head_dim + 2) * 4;
}

cudaError_t launch_tree_attention(const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv, const TreePlan &t,
                                  void *workspace, int *err, int num_sms, cudaStream_t st) {
    const long long es = kv.dtype == PYXIS_DTYPE_F32 ? 4 : 2;
    TreeParams p;
    p.q = (const char *)a.q;
    p.k = (const char *)kv.k;
    p.v = (const char *)kv.v;
    p.out = (char *)a.out;
    p.q_row = a.q_row * es;
    p.q_head = a.q_head * es;
    p.out_row = a.out_row * es;
    p.out_head = a.out_head * es;
    p.page_stride = kv.page_stride * es;
    p.slot_stride = kv.slot_stride * es;
    p.head_stride = kv.head_stride * es;
    p.q_start = a.q_start;
    p.context_len = a.context_len;
    p.block_table = a.block_table;
    p.tree_mask = (const unsigned long long *)a.tree_mask;
    p.table_stride = (long long)a.table_stride;
    p.capacity = (long long)a.table_width * kv.page_size;
    p.n_rows = (int)a.n_rows;
    p.n_q = a.n_q_heads;
    p.n_kv = kv.n_kv_heads;
    p.group = a.n_q_heads / kv.n_kv_heads;
    p.page_size = kv.page_size;
    p.num_pages = kv.num_pages;
    p.max_tree = a.max_tree;
    p.splits = t.splits;
    p.row_tiles = t.row_tiles;
    p.scale2 = a.scale * kLog2e;
    p.err = err;
    if (t.tensor)
        return kv.dtype == PYXIS_DTYPE_F32 ? launch_tree_attention_tc32(p, a, kv, workspace, num_sms, st)
                                           : launch_tree_attention_tc(p, a, kv, workspace, num_sms, st);
    p.part_ml = (float *)workspace;
    p.part_o = p.part_ml ? p.part_ml + a.n_rows * a.n_q_heads * t.splits * 2 : nullptr;
    if (kv.dtype == PYXIS_DTYPE_F32)
        return kv.head_dim == 128 ? run_tree<float, 128>(p, t, a.n_seq, st)
                                  : run_tree<float, 64>(p, t, a.n_seq, st);
    return kv.head_dim == 128 ? run_tree<__nv_bfloat16, 128>(p, t, a.n_seq, st)
                              : run_tree<__nv_bfloat16, 64>(p, t, a.n_seq, st);
}

}  // namespace pyxis
