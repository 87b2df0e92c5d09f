// tree_attn_tc.cuh -- what the tensor-core tree-attention kernels (tree_attn_tc.cu for bf16 pages,
// tree_attn_tc32.cu for f32 ones) share: how the tiles of all units are dealt to the CTAs, and the
// join of the units that several CTAs worked on.
#pragma once

#include "tc_ptx.cuh"
#include "tmap.cuh"
#include "tree_attn.cuh"

namespace pyxis {
namespace {

constexpr int kTcRows = 128;     // rows of a unit: the TMEM lanes
constexpr int kTcMinTiles = 2;   // tiles per CTA before the next CTA gets any

struct TcParams {
    TreeParams t;
    int n_seq;
    int box_rows;       // rows of a TMA box: a page, or a tile of a larger page
    int tile_pages;     // boxes per tile
    int page_tiles;     // tiles per page (1 for pages of up to 128 slots)
    int head_units;     // bf16: 64-column panels from a kv head to the next; 0 if that is no whole number
    int vec_q, vec_out; // 16-byte accesses to q's and out's rows
    uint32_t q_sign;    // flips q's signs for a negative scale (bf16 pairs)
    float *part_o, *part_ml;  // [CTA][2][HD][128], [CTA][2][128][2]
    struct Shared *shared;    // [CTA]
};

// A unit that begins in a CTA and goes on in the next ones, up to CTA `last` (-1: the CTA has none).
// Its sums are in slot 1 of the first CTA and slot 0 of the others.
struct Shared {
    int last, row0, kvh, r0, rows;
};

PYXIS_DEVINL void tma_load_5d(void *dst, const void *tmap, int x, int y, int z, int w, int v, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
            tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(tc::smem_u32(bar))
        : "memory");
}
PYXIS_DEVINL void tma_load_4d(void *dst, const void *tmap, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(tc::smem_u32(bar))
        : "memory");
}

// Operand in the 128-byte swizzle: 64-element panels `panel` bytes apart (which a K-major one does not
// look at), 8-row groups `group` bytes apart.
PYXIS_DEVINL uint64_t desc_rows_sw128(uint32_t smem_addr, uint32_t panel, uint32_t group) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(panel >> 4) << 16;
    d |= (uint64_t)(group >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
PYXIS_DEVINL void named_bar(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// True in one lane of the (converged) warp.
PYXIS_DEVINL bool elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}

// 2^x, denormal results as zero (a weight below 2^-126 of the largest).
PYXIS_DEVINL float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 16 consecutive 32-bit columns of this warp's 32 TMEM lanes (complete after tmem_wait_st).
PYXIS_DEVINL void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// One column of this warp's 32 TMEM lanes (the store complete after tmem_wait_st).
PYXIS_DEVINL float tmem_ld1(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;" : "=r"(r) : "r"(taddr) : "memory");
    return __uint_as_float(r);
}
PYXIS_DEVINL void tmem_st1(uint32_t taddr, float x) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(__float_as_uint(x)) : "memory");
}

PYXIS_DEVINL uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&x);
}
// 4 N bytes of an output row of ELEM-byte elements.
template <int N, int ELEM = 2>
PYXIS_DEVINL void write_row(char *dst, const uint32_t (&u)[N], int vec) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < N; i += 4) reinterpret_cast<uint4 *>(dst)[i / 4] = make_uint4(u[i], u[i + 1], u[i + 2], u[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (ELEM == 4) {
                reinterpret_cast<uint32_t *>(dst)[i] = u[i];
            } else {
                reinterpret_cast<uint16_t *>(dst)[2 * i] = (uint16_t)u[i];
                reinterpret_cast<uint16_t *>(dst)[2 * i + 1] = (uint16_t)(u[i] >> 16);
            }
        }
    }
}

// Units of a sequence: (kv head, 128-row tile); key tiles of each.
struct SeqWork {
    SeqShape sh;
    int row_tiles, units;
    int tiles;
    PYXIS_DEVINL long long work() const { return (long long)units * tiles; }
};
template <int TILE>
PYXIS_DEVINL SeqWork seq_work(const TreeParams &p, int seq) {
    SeqWork w;
    w.sh = seq_shape(p, seq);
    w.row_tiles = (w.sh.nodes * p.group + kTcRows - 1) / kTcRows;
    w.units = w.row_tiles * p.n_kv;
    w.tiles = (int)((w.sh.total + TILE - 1) / TILE);
    if (w.tiles < 1) w.tiles = 1;  // rows without keys still get their zeros
    return w;
}

// CTAs that share `total` tiles, and the first tile of CTA c.
PYXIS_DEVINL int shares(long long total, int grid) {
    const long long most = (total + kTcMinTiles - 1) / kTcMinTiles;
    return (int)(most < grid ? most : grid);
}
PYXIS_DEVINL long long quotient(long long a, int b) {  // a 32-bit division where it will do
    return a >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}
PYXIS_DEVINL long long first_tile(long long total, int c, int g) {  // total c / g, g at most an SM's number
    const long long q = quotient(total, g);
    return q * c + (unsigned)((int)(total - q * g) * c) / (unsigned)g;
}

// The segments (a unit's tiles, or part of them) of a CTA's range, one after another.
template <int TILE>
struct Walk {
    SeqWork w;
    int seq, unit;
    long long left;        // tiles left to this CTA
    int tile;              // next tile of the unit
    int tb, te;            // the segment
    bool from_before;      // its unit began in an earlier CTA
    bool first;
    PYXIS_DEVINL void begin(const TreeParams &p, int seq0, long long offset, long long count) {
        seq = seq0;
        w = seq_work<TILE>(p, seq);
        unit = (int)quotient(offset, w.tiles);
        tile = (int)(offset - (long long)unit * w.tiles);
        left = count;
        first = true;
    }
    PYXIS_DEVINL bool next(const TreeParams &p, int n_seq) {
        if (left <= 0) return false;
        if (!first && tile >= w.tiles) {
            tile = 0;
            if (++unit >= w.units) {
                unit = 0;
                do {
                    if (++seq >= n_seq) return false;
                    w = seq_work<TILE>(p, seq);
                } while (w.units == 0);
            }
        }
        from_before = tile > 0;  // only the CTA's first segment can start inside a unit
        first = false;
        tb = tile;
        te = w.tiles - tile < left ? w.tiles : tile + (int)left;
        left -= te - tb;
        tile = te;
        return true;
    }
    PYXIS_DEVINL int kvh() const { return unit / w.row_tiles; }
    PYXIS_DEVINL int row0() const { return (unit % w.row_tiles) * kTcRows; }
    PYXIS_DEVINL bool whole() const { return tb == 0 && te == w.tiles; }
};

// Inclusive sum over the block's threads; *all is the sum of all of them.
PYXIS_DEVINL long long block_scan(long long x, long long *warp_sum, long long *all) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    *all = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
        if (w < warp) x += warp_sum[w];
        *all += warp_sum[w];
    }
    return x;
}

// The tiles of this CTA: [lo, lo + count) of `total`, dealt to `ctas` of the grid's CTAs.  All threads;
// warp_sum, start_seq and start_off are in shared memory.
struct Range {
    long long total, lo, count;
    int ctas;
};
template <int TILE>
PYXIS_DEVINL Range begin_walk(const TcParams &a, Walk<TILE> &w, long long *warp_sum, int &start_seq, long long &start_off) {
    const TreeParams &p = a.t;
    const int threads = blockDim.x;
    long long mine = 0, incl = 0, sum;
    Range r{0, 0, 0, 0};
    for (int s0 = 0; s0 < a.n_seq; s0 += threads) {
        const int s = s0 + threadIdx.x;
        mine = s < a.n_seq ? seq_work<TILE>(p, s).work() : 0;
        incl = block_scan(mine, warp_sum, &sum);
        r.total += sum;
    }
    const int c = blockIdx.x;
    r.ctas = shares(r.total, gridDim.x);
    if (c < r.ctas) {
        r.lo = first_tile(r.total, c, r.ctas);
        r.count = first_tile(r.total, c + 1, r.ctas) - r.lo;
    }
    if (threadIdx.x == 0) a.shared[c].last = -1;
    if (r.count <= 0) return r;
    long long before = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += threads) {
        const int s = s0 + threadIdx.x;
        if (a.n_seq > threads) {  // else they are still at hand
            mine = s < a.n_seq ? seq_work<TILE>(p, s).work() : 0;
            incl = block_scan(mine, warp_sum, &sum);
        }
        const long long first = before + incl - mine;
        if (mine > 0 && r.lo >= first && r.lo < first + mine) start_seq = s, start_off = r.lo - first;
        before += sum;
    }
    tc::fence_proxy_async_smem();  // warp_sum may lie where a copy lands next
    __syncthreads();
    w.begin(p, start_seq, start_off, r.count);
    return r;
}

// Joins the unit that CTA blockIdx.x of the first kernel left unfinished, kJoinCols columns: a row per
// thread.  Many small blocks and several CTAs' sums in flight per thread: a unit shared by all the
// SMs' CTAs is read at L2 speed, not one latency per CTA.
constexpr int kJoinCols = 8, kJoinUnroll = 4;
template <typename T, int HD>
__global__ void __launch_bounds__(kTcRows) tree_join_tc_kernel(const TcParams a) {
    const TreeParams &p = a.t;
    pdl_wait();
    pdl_trigger();
    const int c0 = blockIdx.x, row = threadIdx.x, col = blockIdx.y * kJoinCols;
    const Shared u = a.shared[c0];
    if (u.last < 0 || row >= u.rows) return;
    const auto slot = [&](int c) -> long long { return c == c0 ? c * 2 + 1 : c * 2; };
    const auto ml_of = [&](int c) { return reinterpret_cast<const float2 *>(a.part_ml)[slot(c) * kTcRows + row]; };
    float o[kJoinCols] = {}, l = 0.f, m = -INFINITY;
    for (int c = c0; c <= u.last; c += kJoinUnroll) {
        float2 ml[kJoinUnroll];
        float x[kJoinUnroll][kJoinCols];
#pragma unroll
        for (int k = 0; k < kJoinUnroll; ++k) {
            ml[k] = c + k <= u.last ? ml_of(c + k) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < kJoinCols; ++i)
                x[k][i] = c + k <= u.last ? a.part_o[(slot(c + k) * HD + col + i) * kTcRows + row] : 0.f;
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kJoinUnroll; ++k) top = fmaxf(top, ml[k].x);
        const float base = top == -INFINITY ? 0.f : top, old = ex2(m - base);
        m = top;
        l *= old;
#pragma unroll
        for (int i = 0; i < kJoinCols; ++i) o[i] *= old;
#pragma unroll
        for (int k = 0; k < kJoinUnroll; ++k) {
            const float f = ex2(ml[k].x - base);
            l = fmaf(f, ml[k].y, l);
#pragma unroll
            for (int i = 0; i < kJoinCols; ++i) o[i] = fmaf(f, x[k][i], o[i]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int t = (u.r0 + row) / p.group, head = u.kvh * p.group + (u.r0 + row) % p.group;
    char *dst = p.out + (u.row0 + t) * p.out_row + head * p.out_head + col * (int)sizeof(T);
    if constexpr (sizeof(T) == 2) {
        uint32_t w[kJoinCols / 2];
#pragma unroll
        for (int i = 0; i < kJoinCols / 2; ++i) w[i] = pack_bf16(o[2 * i] * inv, o[2 * i + 1] * inv);
        write_row(dst, w, a.vec_out);
    } else {
        uint32_t w[kJoinCols];
#pragma unroll
        for (int i = 0; i < kJoinCols; ++i) w[i] = __float_as_uint(o[i] * inv);
        write_row<kJoinCols, 4>(dst, w, a.vec_out);
    }
}

// Launches the join after a kernel of `grid` CTAs.
template <typename T, int HD>
cudaError_t launch_tree_join(const TcParams &a, int grid, cudaStream_t st) {
    return launch_kernel(tree_join_tc_kernel<T, HD>, dim3(grid, HD / kJoinCols), dim3(kTcRows), 0, st, a);
}

inline size_t tree_tc_workspace(int head_dim, int num_sms) {
    return (size_t)num_sms * (2 * kTcRows * (head_dim + 2) * 4 + sizeof(Shared));
}
// The workspace's parts.
inline void set_tc_workspace(TcParams &a, void *workspace, int head_dim, int num_sms) {
    a.part_o = (float *)workspace;
    a.part_ml = a.part_o + (size_t)num_sms * 2 * kTcRows * head_dim;
    a.shared = reinterpret_cast<Shared *>(a.part_ml + (size_t)num_sms * 2 * kTcRows * 2);
}

}  // namespace
}  // namespace pyxis
