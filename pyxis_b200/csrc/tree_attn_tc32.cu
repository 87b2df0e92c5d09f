// tree_attn_tc32.cu -- tree attention over f32 pages on the tensor cores, with f32-level error
// (include/pyxis_serve.h; tree_attn_tc.cu is the bf16 form).
//
// Every f32 operand is split into two fp16 terms after a scaling by a power of two (hi = fp16(x 2^e),
// lo = fp16(x 2^e - hi), 22 significant bits of the values within 2^-12 of the largest of their group: a
// query row, a tile of K, a tile of V; a key in a tile with drafts), and a product is taken as
// lo.hi + hi.lo + hi.hi with f32 accumulation.  Weights are taken in units of their row's largest in the
// tile, which becomes 2^15: fp16 leaves 2^-40 of that, so that light keys keep their bits however heavy a
// key of another tile is (in units of the running maximum the weights below 2^-25 of it would be lost:
// 40000 of them behind a key 17 nats above, a part in 800 of the sum).  The tensor core's accumulation rounds toward zero, so
// each chain is one tile's products, the small ones first, and the sum over tiles is taken in registers
// with the tiles' scales.
//
// 64 keys of K and V are 64 KB that take 2800 cycles to arrive at an SM; their products are 36 MMAs
// (about 2000 cycles) for up to 128 rows, and Q lies in TMEM, so that they read no more of shared memory
// than K's and V's terms.  The converters bound it: 64 KB read, split and written again per tile by six
// warps.  The scale of a tile is taken from the tile before (with room of a factor of four), which spares
// them a pass over it for its largest magnitude (137 -> 115 us for 16 sequences of 2303 positions and 16
// nodes, 8 kv heads of 128), six warps instead of four 115 -> 106, loops that are not unrolled, for the
// instruction cache's sake, 106 -> 100: a floor of 41 us at the memory's rate.  Tiles with drafts, which
// some rows see and others do not, must not let one draft cost another one bits: a scale for each of
// their keys, and values out of the scale's range added in f32 (100 -> 103 us).  58 sequences of 1731
// positions and 64 nodes 301 us (121).  The softmax warps keep a row's scores and its half of O in 160 registers:
// for heads of 128 they spill 264 bytes.
//
// Infinities: an infinite element has no second term (x - hi is NaN).  The converters mark a tile whose keys hold
// one, and its scores that come out NaN are taken again in f32; a column of O that is not finite is summed again
// from the values themselves.
//
// One CTA per SM takes an equal share of all units' tiles (tree_attn_tc.cuh).  Warps:
//   0       producer: a tile's pages by TMA (one box per page) into a ring of f32 tiles, in the order
//           S_0, S_1, O_0, S_2, O_1, ... of the MMAs
//   1       MMA issuer (and TMEM owner)
//   2-7     converters: a tile from the ring into its two fp16 terms, in the 128-byte swizzle, twice
//           buffered; the tile's largest magnitude is found on the way and sets the next one's scale
//   8-15    softmax: a row per thread, half of a tile's keys and of O's columns per warp.  They split
//           their rows of Q into TMEM at a segment's start.
#include <algorithm>
#include <atomic>

#include "attn_tc.h"
#include "tree_attn_tc.cuh"

namespace pyxis {
namespace {

constexpr int kRows = kTcRows, kTile = 64;
constexpr int kProdWarp = 0, kMmaWarp = 1, kConvWarp0 = 2, kConvWarps = 6, kSmWarp0 = 8, kSmWarps = 8;
constexpr int kThreads = (kSmWarp0 + kSmWarps) * 32;
// Registers per thread of the four warpgroups (producer and MMA, converters, softmax twice): their sum
// stays below what the block is launched with, 4 x 128.
constexpr int kRegsLaunch = 128, kRegsFew = 88, kRegsSoft = 160;
static_assert(2 * kRegsFew + 2 * kRegsSoft <= 4 * kRegsLaunch - 16, "register split");
constexpr uint32_t kTmemCols = 512, kOCol = 2 * kTile, kQCol = kOCol + 2 * 128;  // S twice, O twice, Q hi and lo
constexpr uint64_t kTimeoutNs = 2000000000ull;
constexpr float kTop = 15.0f;  // a tile's largest weight is 2^15, in fp16's range
enum { kErrProd = 0x721, kErrMma = 0x722, kErrConv = 0x723, kErrSoft = 0x724, kErrDrain = 0x725, kErrAlign = 0x726 };

template <int HD>
struct Smem {
    static constexpr int kDB = HD / 64;                 // 64-column panels of a row of fp16
    static constexpr uint32_t kPanel = kTile * 128, kTerm = kDB * kPanel;      // of a tile of K or V: hi; lo follows
    static constexpr uint32_t kEntry = kTile * HD * 4;  // a tile of the ring, f32
    static constexpr int kRing = HD == 128 ? 3 : 9;
    static constexpr uint32_t k = 0;                    // two tiles of two terms each
    static constexpr uint32_t v = k + 4 * kTerm;
    static constexpr uint32_t ring = v + 4 * kTerm;
    static constexpr uint32_t bar = ring + kRing * kEntry;
    static constexpr int kBars = 2 * kRing + 1 + 4 + 4 + 1 + 1 + 2 + 3 * 2;
    static constexpr uint32_t misc = bar + (kBars * 8 + 15) / 16 * 16;
    static constexpr uint32_t wmax = misc + 64;          // [2][kConvWarps] magnitudes
    static constexpr uint32_t scale = wmax + 64;         // [2][4]: 2^-e of K and of V of the latest tiles
    static constexpr uint32_t kodd = scale + 32;         // [4] 1 + the latest tiles' numbers where their keys hold an infinity
    static constexpr uint32_t aside = kodd + 16;         // [4] a segment's drafts that are not in their tiles
    static constexpr uint32_t vexp = aside + 32;         // [2][64] exponents of the values of a tile's drafts
    static constexpr uint32_t kexp = vexp + 2 * kTile;   // [4][64] 127 - e of a tile's keys, where each has its own
    static constexpr uint32_t red = kexp + 4 * kTile;    // [2][2 halves][128 rows]
    static constexpr uint32_t bytes = red + 2 * 2 * kRows * 4;
};
static_assert(Smem<128>::bytes <= 232448 && Smem<64>::bytes <= 232448, "227 KB of shared memory per CTA");
static_assert(kQCol + 128 <= kTmemCols, "TMEM columns");

__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Four values times a power of two as fp16 hi and lo: hi is the value rounded to 11 bits by integer
// arithmetic (so that it need not be read back from fp16), lo the exact remainder, rounded.
PYXIS_DEVINL float to11(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xFFFFE000u); }
PYXIS_DEVINL void split4(float4 x, float sc, uint2 &hi, uint2 &lo) {
    x.x *= sc, x.y *= sc, x.z *= sc, x.w *= sc;
    const float4 h = make_float4(to11(x.x), to11(x.y), to11(x.z), to11(x.w));
    const __half2 ha = __floats2half2_rn(h.x, h.y), hb = __floats2half2_rn(h.z, h.w);
    const __half2 la = __floats2half2_rn(x.x - h.x, x.y - h.y), lb = __floats2half2_rn(x.z - h.z, x.w - h.w);
    hi = make_uint2(*reinterpret_cast<const uint32_t *>(&ha), *reinterpret_cast<const uint32_t *>(&hb));
    lo = make_uint2(*reinterpret_cast<const uint32_t *>(&la), *reinterpret_cast<const uint32_t *>(&lb));
}
// The exponent e that takes a finite magnitude (its bits) to [2^14, 2^15); 2^e and 2^-e are normal.
PYXIS_DEVINL int scale_exp(uint32_t m) { return m ? min(141 - (int)(m >> 23), 100) : 0; }
// The largest finite magnitude of four values, as its bits.
PYXIS_DEVINL uint32_t magnitude(float4 x) {
    const auto bits = [](float v) {
        const uint32_t u = __float_as_uint(v) & 0x7FFFFFFFu;
        return u < 0x7F800000u ? u : 0u;
    };
    return max(max(bits(x.x), bits(x.y)), max(bits(x.z), bits(x.w)));
}
// Byte offset of dims 4 i .. 4 i + 3 of a row in an operand's term (panels of `panel` bytes).
PYXIS_DEVINL uint32_t swizzled(int row, int i, uint32_t panel) {
    return (uint32_t)(i >> 4) * panel + (uint32_t)row * 128 + ((((uint32_t)i >> 1) & 7) ^ ((uint32_t)row & 7)) * 16 +
           (uint32_t)(i & 1) * 8;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attention_tc32_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                               const TcParams a) {
    using L = Smem<HD>;
    constexpr int kDB = L::kDB, kRing = L::kRing, kOH = HD / 2;  // columns of O per softmax warp
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::bar);
    uint64_t *full = bars, *empty = bars + kRing, *cmax = empty + kRing, *cfull = cmax + 1, *cempty = cfull + 4;  // [K, V][2]
    uint64_t *qfull = cempty + 4, *drain = qfull + 1, *ofree = drain + 1;
    // per score buffer: sfull (S_j landed), pfull (P_j written), odone (P_j V_j done)
    uint64_t *sfull = ofree + 2, *pfull = sfull + 2, *odone = pfull + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::misc);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::misc + 4);
    // (the converters are at most two segments ahead of the softmax warps)
    unsigned long long *aside = reinterpret_cast<unsigned long long *>(smem + L::aside);
    uint8_t *kexp = smem + L::kexp;
    volatile int *kodd = reinterpret_cast<volatile int *>(smem + L::kodd);
    volatile uint8_t *vexp = smem + L::vexp;
    long long &start_off = *reinterpret_cast<long long *>(smem + L::misc + 16);
    int &start_seq = *reinterpret_cast<int *>(smem + L::misc + 24);
    volatile uint32_t *wmax = reinterpret_cast<volatile uint32_t *>(smem + L::wmax);
    volatile float *scale = reinterpret_cast<volatile float *>(smem + L::scale);
    float *red = reinterpret_cast<float *>(smem + L::red);
    long long *warp_sum = reinterpret_cast<long long *>(smem + L::ring);  // before the ring is used
    const TreeParams &p = a.t;
    if (tc::smem_u32(smem) & 1023) {  // the swizzled tiles' alignment; there is no static shared memory before them
        if (threadIdx.x == 0) atomicCAS(p.err, 0, kErrAlign);
        return;
    }

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kRing; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], kConvWarps);
        }
        tc::mbar_init(cmax, kConvWarps);
        for (int b = 0; b < 4; ++b) {
            tc::mbar_init(&cfull[b], kConvWarps);
            tc::mbar_init(&cempty[b], 1);
        }
        tc::mbar_init(qfull, kSmWarps);
        tc::mbar_init(drain, 1);
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&ofree[b], kSmWarps);
            tc::mbar_init(&sfull[b], 1);
            tc::mbar_init(&pfull[b], kSmWarps);
            tc::mbar_init(&odone[b], 1);
        }
        *abort_flag = 0;
        for (int i = 0; i < 4; ++i) kodd[i] = 0;
        tc::fence_mbar_init();
        tc::prefetch_tmap(&tm_k);
        tc::prefetch_tmap(&tm_v);
    }
    if (warp == kMmaWarp) tc::tmem_alloc(tmem_slot, kTmemCols);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    pdl_trigger();

    // ---- this CTA's tiles
    Walk<kTile> w;
    const Range r = begin_walk(a, w, warp_sum, start_seq, start_off);
    const long long total = r.total, lo = r.lo, count = r.count;
    const int g = r.ctas, c = blockIdx.x;
    if (count > 0) {
        // (all warps of a warpgroup, and of the CTA, come here or none: count is the CTA's)
        if (warp < kSmWarp0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
        if (warp < kConvWarp0) {
            if (warp == kProdWarp) {
                // ---------------------------------------------------------------- producer
                int e = 0;
                bool ok = true;
                while (ok && w.next(p, a.n_seq)) {
                    const int T = w.te - w.tb, kvh = w.kvh();
                    const int32_t *table = p.block_table + w.seq * p.table_stride;
                    // how many of the pages of tile tb + j exist, and this lane's
                    auto page_count = [&](int j) -> int {
                        if (j >= T) return 0;
                        const long long rest = w.w.sh.total - (long long)(w.tb + j) * kTile;
                        if (rest >= kTile) return a.tile_pages;
                        return rest <= 0 ? 0 : ((int)rest + a.box_rows - 1) / a.box_rows;
                    };
                    auto page_of = [&](int j) -> int {
                        if (lane >= page_count(j)) return 0;
                        const int t = w.tb + j;
                        const int id = __ldg(table + (a.page_tiles == 1 ? t * a.tile_pages + lane : t / a.page_tiles));
                        return min(max(id, 0), p.num_pages - 1);
                    };
                    auto issue = [&](bool is_k, int j, int page) -> bool {
                        const int slot = e % kRing;
                        if (!__all_sync(0xffffffffu, tc::mbar_wait_bounded(&empty[slot], (uint32_t)((e / kRing - 1) & 1), abort_flag,
                                                                           p.err, kErrProd, kTimeoutNs)))
                            return false;
                        const int n = page_count(j);
                        if (lane == 0) tc::mbar_arrive_expect_tx(&full[slot], (uint32_t)(n * a.box_rows * HD * 4));
                        __syncwarp();
                        if (lane < n)
                            tma_load_4d(smem + L::ring + slot * L::kEntry + lane * a.box_rows * HD * 4, is_k ? &tm_k : &tm_v, 0, kvh,
                                        a.page_tiles == 1 ? 0 : (w.tb + j) % a.page_tiles * kTile, page, &full[slot]);
                        ++e;
                        return true;
                    };
                    int prev = 0, cur = page_of(0), next = page_of(1);
                    ok = issue(true, 0, cur);
                    for (int j = 1; ok && j < T; ++j) {
                        prev = cur, cur = next, next = page_of(j + 1);
                        ok = issue(true, j, cur) && issue(false, j - 1, prev);
                    }
                    ok = ok && issue(false, T - 1, cur);
                }
                if (*abort_flag && lane == 0) {  // let the copies already issued land before the CTA exits
                    volatile int no_abort = 0;
                    for (int x = max(0, e - kRing); x < e; ++x)
                        tc::mbar_wait_bounded(&full[x % kRing], (uint32_t)((x / kRing) & 1), &no_abort, p.err, kErrDrain, 100000000ull);
                }
            } else if (warp == kMmaWarp) {
                // ---------------------------------------------------------------- MMA issuer
                if (elect_one()) {
                    constexpr uint32_t idesc_s = idesc_f16(kRows, kTile, false), idesc_o = idesc_f16(kRows, HD, true);
                    const uint64_t k_d = tc::desc_sw128(tc::smem_u32(smem + L::k));
                    const uint64_t v_d = desc_rows_sw128(tc::smem_u32(smem + L::v), L::kPanel, 1024);
                    int kuse = 0, vuse = 0;  // K and V tiles multiplied
                    auto wait = [&](uint64_t *bar, int phase) -> bool {
                        return tc::mbar_wait_bounded(bar, (uint32_t)(phase & 1), abort_flag, p.err, kErrMma, kTimeoutNs);
                    };
                    bool ok = true;
                    auto score = [&]() -> bool {
                        const int b = kuse & 1;
                        // the buffer's earlier probabilities have been multiplied, and K is there
                        if (!wait(&odone[b], kuse / 2 - 1) || !wait(&cfull[b], kuse / 2)) return false;
                        tc::tc_fence_after();
                        const uint32_t tS = tmem_base + (uint32_t)(b * kTile);
                        const uint64_t kd = k_d + (uint64_t)(b * (2 * L::kTerm >> 4));
#pragma unroll 1
                        for (int term = 0; term < 3; ++term) {  // lo.hi, hi.lo, hi.hi
                            const uint32_t qt = tmem_base + kQCol + (uint32_t)(term == 0 ? HD / 2 : 0);
                            const uint64_t kt = kd + (uint64_t)(term == 1 ? L::kTerm >> 4 : 0);
#pragma unroll
                            for (int x = 0; x < kDB; ++x)
#pragma unroll
                                for (int kk = 0; kk < 4; ++kk)  // 16 dims: 8 columns of Q
                                    tc::mma_f16_ts(tS, qt + (uint32_t)(x * 32 + kk * 8),
                                                   kt + (uint64_t)(x * (L::kPanel >> 4) + kk * 2), idesc_s, (uint32_t)(term | x | kk));
                        }
                        tc::mma_commit(&cempty[b]);
                        tc::mma_commit(&sfull[b]);
                        ++kuse;
                        return true;
                    };
                    auto output = [&]() -> bool {
                        const int b = vuse & 1;
                        if (!wait(&cfull[2 + b], vuse / 2) || !wait(&pfull[b], vuse / 2) || !wait(&ofree[b], vuse / 2 - 1)) return false;
                        tc::tc_fence_after();
                        const uint32_t tP = tmem_base + (uint32_t)(b * kTile), tO = tmem_base + kOCol + (uint32_t)(b * HD);
                        const uint64_t vd = v_d + (uint64_t)(b * (2 * L::kTerm >> 4));
#pragma unroll 1
                        for (int term = 0; term < 3; ++term) {
                            const uint32_t pt = tP + (term == 0 ? kTile / 2 : 0);  // lo terms follow the hi ones
                            const uint64_t vt = vd + (uint64_t)(term == 1 ? L::kTerm >> 4 : 0);
#pragma unroll
                            for (int kk = 0; kk < kTile / 16; ++kk)  // 16 keys: 8 columns of P, 16 rows of V
                                tc::mma_f16_ts(tO, pt + (uint32_t)(kk * 8), vt + (uint64_t)(kk * (2048 >> 4)), idesc_o,
                                               (uint32_t)(term | kk));
                        }
                        tc::mma_commit(&cempty[2 + b]);
                        tc::mma_commit(&odone[b]);
                        ++vuse;
                        return true;
                    };
                    for (int seg = 0; ok && w.next(p, a.n_seq); ++seg) {
                        const int T = w.te - w.tb;
                        ok = wait(qfull, seg) && score();
                        for (int j = 1; ok && j < T; ++j) ok = score() && output();
                        ok = ok && output();
                    }
                    // every MMA this thread issued must complete before TMEM is released
                    tc::mma_commit(drain);
                    volatile int no_abort = 0;
                    tc::mbar_wait_bounded(drain, 0, &no_abort, p.err, kErrDrain, kTimeoutNs);
                }
            }
        } else if (warp < kSmWarp0) {
            // ---------------------------------------------------------------- converters
            const int cw = warp - kConvWarp0;
            constexpr int kLanes = HD / 4, kPer = 32 / kLanes, kSteps = kTile / kPer;  // lanes of a row, rows and steps of a warp
            const int li = lane % kLanes, sub = lane / kLanes;
            auto wait = [&](uint64_t *bar, int phase) -> bool {
                return __all_sync(0xffffffffu, tc::mbar_wait_bounded(bar, (uint32_t)(phase & 1), abort_flag, p.err, kErrConv,
                                                                     kTimeoutNs));
            };
            int e = 0, use[2] = {0, 0}, looks = 0;  // looks: exchanges of the largest magnitude
            int ex[2] = {13, 13};                   // scale exponents of K and V
            bool ok = true;
            int seg = 0;
            for (; ok && w.next(p, a.n_seq); ++seg) {
                const int T = w.te - w.tb;
                const SeqShape &sh = w.w.sh;
                if (cw == 0 && lane == 0) aside[seg & 3] = 0;  // (before the exchange that precedes any set bit)
                auto convert = [&](int is_v, int j) -> bool {
                    const int slot = e % kRing;
                    if (!wait(&full[slot], e / kRing)) return false;
                    const long long k0 = (long long)(w.tb + j) * kTile;
                    const int valid = (int)min((long long)kTile, max(sh.total - k0, 0ll));
                    const int drafts = (int)min((long long)kTile, max(sh.ctx - k0, 0ll));  // first draft's row
                    // this lane's four dims of row i * kPer + sub; zero past the last key (never loaded, or
                    // not a key)
                    const float4 *src = reinterpret_cast<const float4 *>(smem + L::ring + slot * L::kEntry) + lane;
                    auto edge = [&](int i) { return i * kPer + sub < valid ? src[i * 32] : make_float4(0.f, 0.f, 0.f, 0.f); };
                    const int buf = use[is_v] & 1;
                    if (!wait(&cempty[is_v * 2 + buf], use[is_v] / 2 - 1)) return false;
                    uint8_t *dst = smem + (is_v ? L::v : L::k) + buf * 2 * L::kTerm;
                    auto put = [&](int i, float4 x, float sc) {
                        uint2 hi, low;
                        split4(x, sc, hi, low);
                        const uint32_t at = swizzled(i * kPer + sub, li, L::kPanel);
                        *reinterpret_cast<uint2 *>(dst + at) = hi;
                        *reinterpret_cast<uint2 *>(dst + L::kTerm + at) = low;
                    };
                    // largest finite magnitude of the row (of all its lanes)
                    auto row_max = [&](float4 x) {
                        uint32_t m = magnitude(x);
                        if constexpr (kLanes == 32) {
                            m = __reduce_max_sync(0xffffffffu, m);
                        } else {
#pragma unroll
                            for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                        }
                        return m;
                    };
                    int used = ex[is_v];
                    if (drafts == kTile) {
                        // The context, which all rows see.  The scale is that of the tile before, which leaves a
                        // factor of 4 to fp16's largest number; a tile that does not fit it, or is far below
                        // it, is done again with its own.
                        for (int round = 0;; ++round) {
                            const float sc = attn_pow2(ex[is_v]);
                            float mf = 0.f;  // (fmaxf passes over NaN)
#pragma unroll 1
                            for (int i = cw; i < kSteps; i += kConvWarps) {
                                const float4 x = src[i * 32];
                                put(i, x, sc);
                                mf = fmaxf(fmaxf(fmaxf(mf, fabsf(x.x)), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
                            }
                            uint32_t m = __float_as_uint(mf);
                            if (m == 0x7F800000u) {  // an infinity, which sets no scale: the largest finite one
                                if (!is_v) kodd[use[0] & 3] = use[0] + 1;
                                m = 0;
                                for (int i = cw; i < kSteps; i += kConvWarps) m = max(m, magnitude(src[i * 32]));
                            }
                            m = __reduce_max_sync(0xffffffffu, m);
                            if (lane == 0) {
                                wmax[(looks & 1) * kConvWarps + cw] = m;
                                tc::mbar_arrive(cmax);
                            }
                            if (!wait(cmax, looks)) return false;
#pragma unroll
                            for (int i = 0; i < kConvWarps; ++i) m = max(m, wmax[(looks & 1) * kConvWarps + i]);
                            ++looks;
                            used = ex[is_v];
                            if (m) ex[is_v] = scale_exp(m) - 1;  // [2^13, 2^14): for the next tile
                            const float top = __uint_as_float(m) * sc;
                            if (round > 0 || m == 0 || (top < 65504.f && top >= 1024.f)) break;
                        }
                    } else if (!is_v) {
                        // Drafts, which some rows see and others do not: a scale for each key, so that none
                        // costs another one bits.
#pragma unroll 1
                        for (int i = cw; i < kSteps; i += kConvWarps) {
                            const float4 x = edge(i);
                            const int e = scale_exp(row_max(x));
                            put(i, x, attn_pow2(e));
                            if (isinf(x.x) || isinf(x.y) || isinf(x.z) || isinf(x.w)) kodd[use[0] & 3] = use[0] + 1;
                            if (li == 0) kexp[(use[0] & 3) * kTile + i * kPer + sub] = (uint8_t)(127 - e);
                        }
                        used = 0;
                    } else {
                        // Drafts' values: one scale, that of the tile's context or else of its first finite draft,
                        // with room for values 16 times as large.  A draft that does not fit, is less than
                        // 1/1024 of it or not finite is set aside (zero here): the rows that see it, and no
                        // others, get it in f32 at the end.
                        volatile uint8_t *ve = vexp + (looks & 1) * kTile;
#pragma unroll 1
                        for (int i = cw; i < kSteps; i += kConvWarps) {
                            const float4 x = edge(i);
                            const int row = i * kPer + sub;
                            const bool odd = !isfinite(x.x) || !isfinite(x.y) || !isfinite(x.z) || !isfinite(x.w);
                            const unsigned odds = __ballot_sync(0xffffffffu, odd && row >= drafts) >> (sub * kLanes);
                            const uint32_t m = row_max(x);
                            if (li == 0) ve[row] = (odds & (0xFFFFFFFFu >> (32 - kLanes))) ? 255 : (uint8_t)(m >> 23);
                        }
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(cmax);
                        if (!wait(cmax, looks)) return false;
                        ++looks;
                        int ref = 0;
                        unsigned fit[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int x = ve[h * 32 + lane];
                            if (h * 32 + lane < drafts) ref = max(ref, x);
                            fit[h] = __ballot_sync(0xffffffffu, x > 0 && x < 255);
                        }
                        ref = __reduce_max_sync(0xffffffffu, ref);
                        if (ref == 0 && (fit[0] | fit[1])) ref = ve[fit[0] ? __ffs(fit[0]) - 1 : 31 + __ffs(fit[1])];
                        used = scale_exp((uint32_t)ref << 23) - 4;  // [2^10, 2^11)
                        const float sc = attn_pow2(used);
#pragma unroll 1
                        for (int i = cw; i < kSteps; i += kConvWarps) {
                            const int row = i * kPer + sub, x = ve[row], at = x - 127 + used;  // values up to 2^(at + 1)
                            const bool out = row >= drafts && x > 0 && (x == 255 || at > 14 || at < 1);
                            put(i, out ? make_float4(0.f, 0.f, 0.f, 0.f) : edge(i), sc);
                            if (out && li == 0) atomicOr(&aside[seg & 3], 1ull << (int)(k0 + row - sh.ctx));
                        }
                    }
                    if (cw == 0 && lane == 0) scale[is_v * 4 + (use[is_v] & 3)] = attn_pow2(-used);
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&empty[slot]);
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&cfull[is_v * 2 + buf]);
                    ++use[is_v];
                    ++e;
                    return true;
                };
                ok = convert(0, 0);
                for (int j = 1; ok && j < T; ++j) ok = convert(0, j) && convert(1, j - 1);
                ok = ok && convert(1, T - 1);
            }
        } else {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoft));
            // ---------------------------------------------------------------- softmax
            const int quad = warp & 3;                // TMEM lanes 32 quad .. 32 quad + 31
            const int sw = warp - kSmWarp0, half = sw >> 2;  // keys [32 half, +32) of each tile, columns [kOH half, +kOH) of O
            const int row = quad * 32 + lane;
            const uint32_t tq = tmem_base + ((uint32_t)(quad * 32) << 16), tOh = tq + kOCol + (uint32_t)(half * kOH);
            const float sign = p.scale2 < 0.f ? -1.f : 1.f;
            auto wait = [&](uint64_t *bar, int phase) -> bool {
                return __all_sync(0xffffffffu, tc::mbar_wait_bounded(bar, (uint32_t)(phase & 1), abort_flag, p.err, kErrSoft,
                                                                     kTimeoutNs));
            };
            int n = 0;      // tiles so far
            int swaps = 0;  // exchanges with the rows' other warp: they alternate between two buffers
            bool ok = true;
            for (int seg = 0; w.next(p, a.n_seq); ++seg) {
                const int T = w.te - w.tb, kvh = w.kvh(), r0 = w.row0();
                const SeqShape &sh = w.w.sh;
                const int rows = min(sh.nodes * p.group - r0, kRows);
                const bool active = quad * 32 < rows;  // the warp has rows
                // ---- Q into TMEM, this row's half of the dims; the last segment's MMAs are done (odone)
                float qscale = 1.f;  // 2^-e of the row
                if (active) {
                    constexpr int kQ4 = kOH / 4;
                    float4 x[kQ4];
                    const int t = (r0 + row) / p.group;
                    const float *src = reinterpret_cast<const float *>(
                                           p.q + (sh.row0 + t) * p.q_row + (kvh * p.group + r0 + row - t * p.group) * p.q_head) +
                                       half * kOH;
                    uint32_t m = 0;
#pragma unroll
                    for (int i = 0; i < kQ4; ++i) {
                        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (row < rows)
                            x[i] = a.vec_q ? reinterpret_cast<const float4 *>(src)[i]
                                           : make_float4(src[4 * i], src[4 * i + 1], src[4 * i + 2], src[4 * i + 3]);
                    }
#pragma unroll
                    for (int i = 0; i < kQ4; ++i) m = max(m, magnitude(x[i]));
                    float *rd = red + (swaps++ & 1) * 2 * kRows;
                    rd[half * kRows + row] = __uint_as_float(m);
                    named_bar(1 + quad, 64);
                    m = max(m, __float_as_uint(rd[(1 - half) * kRows + row]));
                    const int ex = scale_exp(m);
                    const float sc = sign * attn_pow2(ex);
                    qscale = attn_pow2(-ex);
#pragma unroll
                    for (int ch = 0; ch < kQ4 / 8; ++ch) {  // 32 dims: 16 columns of each term
                        uint32_t hi[16], low[16];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            uint2 h2, l2;
                            split4(x[ch * 8 + i], sc, h2, l2);
                            hi[2 * i] = h2.x, hi[2 * i + 1] = h2.y, low[2 * i] = l2.x, low[2 * i + 1] = l2.y;
                        }
                        tmem_st16(tq + kQCol + (uint32_t)(half * (kOH / 2) + ch * 16), hi);
                        tmem_st16(tq + kQCol + (uint32_t)(HD / 2 + half * (kOH / 2) + ch * 16), low);
                    }
                    tc::tmem_wait_st();
                    tc::tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(qfull);
                unsigned long long mask = 0;
                if (row < rows) {
                    const int t = (r0 + row) / p.group;
                    mask = p.tree_mask ? p.tree_mask[sh.row0 + t] : (2ull << t) - 1;
                }
                const float c2row = fabsf(p.scale2) * qscale;
                float m_run = -INFINITY, l = 0.f;
                float unit = 0.f;  // the tile before's unit of weight, 2^(its maximum - kTop), in terms of 2^m_run
                float acc[kOH];
#pragma unroll
                for (int i = 0; i < kOH; ++i) acc[i] = 0.f;
                // (O unit + acc) of tile m into acc, then times alpha
                auto fold = [&](int m, float alpha) -> bool {
                    if (!wait(&odone[m & 1], m / 2)) return false;
                    if (active) {
                        tc::tc_fence_after();
                        const float vs = scale[4 + (m & 3)] * unit;
#pragma unroll
                        for (int ch = 0; ch < kOH / 32; ++ch) {
                            uint32_t o[32];
                            tc::tmem_ld32_async(tOh + (uint32_t)((m & 1) * HD + ch * 32), o);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) acc[ch * 32 + i] = fmaf(__uint_as_float(o[i]), vs, acc[ch * 32 + i]) * alpha;
                        }
                        tc::tc_fence_before();
                    }
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&ofree[m & 1]);
                    return true;
                };
                // after a failed wait the loops run on without work, so that the barriers of a row's two
                // warps keep their counts
                for (int j = 0; j < T; ++j, ++n) {
                    const int b = n & 1;
                    const long long k0 = (long long)(w.tb + j) * kTile;
                    const uint32_t tS = tq + (uint32_t)(b * kTile);
                    const bool tail = k0 + kTile > sh.ctx;
                    ok = ok && wait(&sfull[b], n / 2);
                    float alpha = 1.f, next_unit = 0.f;
                    if (active) {
                        float s[32];
                        float mt = -INFINITY, c2 = 0.f;
                        if (ok) {
                            tc::tc_fence_after();
                            // log2 units: acc 2^-(eq + ek) scale log2 e (a masked score stays -inf with scale 0, too)
                            c2 = fmaxf(c2row * scale[n & 3], 1e-37f);
                            if (kodd[n & 3] == n + 1) {
                                // A key with an infinity has no second term and its products are NaN, which the
                                // maximum passes over; where its score is -inf, its weight is zero.
                                const int t = (r0 + row) / p.group;
                                const float *q = reinterpret_cast<const float *>(
                                    p.q + (sh.row0 + t) * p.q_row + (kvh * p.group + r0 + row - t * p.group) * p.q_head);
#pragma unroll 1
                                for (int i = half * 32; i < half * 32 + 32; ++i) {
                                    float x = tmem_ld1(tS + (uint32_t)i);
                                    if (row < rows && isnan(x) && k0 + i < sh.total &&
                                        key_score<HD>(p, q, w.seq, kvh, k0 + i) * p.scale2 == -INFINITY)
                                        x = -INFINITY;
                                    __syncwarp();
                                    tmem_st1(tS + (uint32_t)i, x);
                                }
                                tc::tmem_wait_st();
                            }
                            tc::tmem_ld32(tS + (uint32_t)(half * 32), s);
                            if (tail) {
                                const uint32_t *ke = reinterpret_cast<const uint32_t *>(kexp + (n & 3) * kTile + half * 32);
#pragma unroll
                                for (int i = 0; i < 32; ++i) s[i] *= __uint_as_float((ke[i >> 2] >> (8 * (i & 3)) & 0xFFu) << 23);
                                // bit i: the row sees key k0 + 32 half + i -- the context, and its mask's drafts
                                const long long d0 = sh.ctx - k0 - half * 32;  // the first draft's column
                                const int avail = (int)(sh.total - sh.ctx);
                                const unsigned long long m = avail >= 64 ? mask : mask & ((1ull << avail) - 1);
                                const uint32_t vis =
                                    (uint32_t)(d0 >= 32 ? ~0ull : d0 > 0 ? ((1ull << d0) - 1) | m << d0 : d0 > -64 ? m >> -d0 : 0ull);
#pragma unroll
                                for (int i = 0; i < 32; ++i) s[i] = (vis & (1u << i)) ? s[i] : -INFINITY;
                            }
                            float x[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                            for (int i = 4; i < 32; ++i) x[i & 3] = fmaxf(x[i & 3], s[i]);
                            mt = c2 * fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                        }
                        // the row's maximum over both halves; past this barrier both have read S, so P may
                        // be written over it
                        float *rd = red + (swaps++ & 1) * 2 * kRows;
                        rd[half * kRows + row] = mt;
                        named_bar(1 + quad, 64);
                        mt = fmaxf(mt, rd[(1 - half) * kRows + row]);
                        const float m_new = fmaxf(m_run, mt);
                        alpha = mt > m_run ? ex2(m_run - mt) : 1.f;
                        next_unit = mt == -INFINITY ? 0.f : ex2(mt - m_new - kTop);
                        m_run = m_new;
                        if (ok) {
                            const float base = mt == -INFINITY ? 0.f : mt - kTop;
                            uint32_t ph[16], pl[16];
                            float sum = 0.f;
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float p0 = ex2(fmaf(s[2 * i], c2, -base)), p1 = ex2(fmaf(s[2 * i + 1], c2, -base));
                                sum += p0 + p1;
                                const __half2 h = __floats2half2_rn(p0, p1);
                                const float2 f = __half22float2(h);
                                const __half2 q = __floats2half2_rn(p0 - f.x, p1 - f.y);
                                ph[i] = *reinterpret_cast<const uint32_t *>(&h);
                                pl[i] = *reinterpret_cast<const uint32_t *>(&q);
                            }
                            l = fmaf(sum, next_unit, l * alpha);
                            tmem_st16(tS + (uint32_t)(half * 16), ph);
                            tmem_st16(tS + (uint32_t)(kTile / 2 + half * 16), pl);
                            tc::tmem_wait_st();
                            tc::tc_fence_before();
                        }
                    }
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&pfull[b]);
                    // the previous tile's P V, at the previous maximum, then this tile's rescale
                    if (j > 0) ok = ok && fold(n - 1, alpha);
                    unit = next_unit;
                }
                ok = ok && fold(n - 1, 1.0f);
                if (active) {  // the row sum of both halves
                    float *rd = red + (swaps++ & 1) * 2 * kRows;
                    rd[half * kRows + row] = l;
                    named_bar(1 + quad, 64);
                    l += rd[(1 - half) * kRows + row];
                }
                bool odd = false;  // some of the row's sums are not finite; where they have been written
                char *first = nullptr;
                int step = 0;
                if (active && ok && row < rows) {
                    const bool whole = w.whole();
                    const int t = (r0 + row) / p.group, h = kvh * p.group + (r0 + row) % p.group;
                    // the drafts that were set aside, for the rows that see them
                    for (unsigned long long rest = aside[seg & 3] & mask; rest; rest &= rest - 1) {
                        const long long pos = sh.ctx + __ffsll((long long)rest) - 1;
                        const int page = min(max(p.block_table[w.seq * p.table_stride + pos / p.page_size], 0), p.num_pages - 1);
                        const long long key = page * p.page_stride + (pos % p.page_size) * p.slot_stride + kvh * p.head_stride;
                        const float *k = reinterpret_cast<const float *>(p.k + key), *v = reinterpret_cast<const float *>(p.v + key);
                        const float *q = reinterpret_cast<const float *>(p.q + (sh.row0 + t) * p.q_row + h * p.q_head);
                        float x = 0.f;
#pragma unroll 4
                        for (int i = 0; i < HD; ++i) x = fmaf(q[i], k[i], x);
                        const float weight = ex2(x * p.scale2 - (m_run == -INFINITY ? 0.f : m_run));
#pragma unroll
                        for (int i = 0; i < kOH; ++i) {
                            const float y = v[half * kOH + i];
                            acc[i] += isfinite(y) ? weight * y : y;
                        }
                    }
                    const long long at = ((long long)(c * 2 + (w.from_before ? 0 : 1)) * kRows + row);
                    float *part = a.part_o + (at - row) * HD + (half * kOH) * kRows + row;  // column-major
                    char *dst = p.out + (sh.row0 + t) * p.out_row + h * p.out_head + half * (kOH * 4);
                    if (whole) {
                        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                        for (int ch = 0; ch < kOH / 8; ++ch) {
                            uint32_t u[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(acc[ch * 8 + i] * inv);
                            write_row<8, 4>(dst + ch * 32, u, a.vec_out);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < kOH; ++i) part[i * kRows] = acc[i];
                        if (half == 0) a.part_ml[at * 2] = m_run, a.part_ml[at * 2 + 1] = l;
                        if (half == 0 && !w.from_before && row == 0) {
                            const long long end = lo + count + (w.w.tiles - w.te) - 1;  // the unit's last tile
                            a.shared[c] = Shared{(int)(((end + 1) * g + total - 1) / total) - 1, sh.row0, kvh, r0, rows};
                        }
                    }
                    odd = isfinite(l) && isnan(odd_mark(acc));
                    first = whole ? dst : reinterpret_cast<char *>(part);
                    step = whole ? 4 : kRows * 4;
                }
                if (__any_sync(0xffffffffu, odd)) {
                    // An infinite value has no second term, and a weight's may be zero or negative: a sum over values
                    // that are not finite is taken from the values (a row whose weights are NaN is NaN).
                    constexpr int kC = kOH / 32;  // columns per lane
                    const long long c0 = (long long)w.tb * kTile, c1 = (long long)w.te * kTile;
                    const float4 bad = odd_columns<float, kC>(p, sh, w.seq, kvh, half * kOH, c0, c1);
#pragma unroll 1
                    for (int i = 0; i < kOH; ++i) {
                        float x = __shfl_sync(0xffffffffu, i % kC ? bad.y : bad.x, i / kC);
                        float *y = reinterpret_cast<float *>(first + i * step);  // (read back: acc stays in registers)
                        if (!odd || isfinite(*y)) continue;
                        x += odd_drafts<float>(p, sh, w.seq, kvh, half * kOH + i, mask, c0, c1);
                        if (x != 0.f) *y = x;
                    }
                }
                __syncwarp();
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == kMmaWarp) tc::tmem_dealloc(tmem_base, kTmemCols);
}

// [page][slot][head] of K or V, whole rows of f32
bool make_map(CUtensorMap *m, const void *base, const pyxis_kv_pages &kv, int box_rows) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const auto stride = [&](int n, int64_t s) { return (cuuint64_t)(n > 1 ? s : kv.head_dim) * 4; };  // of an axis of one: any
    cuuint64_t dims[4] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.n_kv_heads, (cuuint64_t)kv.page_size,
                          (cuuint64_t)kv.num_pages};
    cuuint64_t strides[3] = {stride(kv.n_kv_heads, kv.head_stride), stride(kv.page_size, kv.slot_stride),
                             stride(kv.num_pages, kv.page_stride)};
    cuuint32_t box[4] = {(cuuint32_t)kv.head_dim, 1, (cuuint32_t)box_rows, 1};
    cuuint32_t es[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, const_cast<void *>(base), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD>
cudaError_t run_tc32(const CUtensorMap &k, const CUtensorMap &v, const TcParams &a, int grid, cudaStream_t st) {
    auto kern = tree_attention_tc32_kernel<HD>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = once_per_device(done, [&] {
        cudaFuncAttributes at;
        const cudaError_t x = cudaFuncGetAttributes(&at, kern);
        if (x != cudaSuccess) return x;
        // the softmax warps' share is taken from the launch's registers: with fewer they would wait for good
        if (at.numRegs * 4 < 2 * kRegsFew + 2 * kRegsSoft) return cudaErrorInvalidConfiguration;
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Smem<HD>::bytes);
    });
    if (e != cudaSuccess) return e;
    PdlScope pdl;
    e = launch_kernel(kern, dim3(grid), dim3(kThreads), Smem<HD>::bytes, st, k, v, a);
    if (e != cudaSuccess) return e;
    return launch_tree_join<float, HD>(a, grid, st);
}

}  // namespace

// A page of 2 to 64 slots that tiles 64 keys (a lane of the producer per page), or a multiple of 64 slots.
bool tree_attention_tc32_supported(const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv) {
    (void)a;
    const int64_t most = (int64_t)1 << 37;
    return kv.dtype == PYXIS_DTYPE_F32 && kv.page_size >= 2 && (kTile % kv.page_size == 0 || kv.page_size % kTile == 0) &&
           kv.page_stride < most && kv.slot_stride < most && kv.head_stride < most;
}

size_t tree_attention_tc32_workspace(const pyxis_kv_pages &kv, int num_sms) { return tree_tc_workspace(kv.head_dim, num_sms); }

cudaError_t launch_tree_attention_tc32(const TreeParams &p, const pyxis_tree_attention_args &args, const pyxis_kv_pages &kv,
                                       void *workspace, int num_sms, cudaStream_t st) {
    TcParams a;
    a.t = p;
    a.n_seq = (int)args.n_seq;
    a.box_rows = std::min(kv.page_size, kTile);
    a.tile_pages = kTile / a.box_rows;
    a.page_tiles = std::max(1, kv.page_size / kTile);
    const auto vec = [](const void *base, int64_t row, int64_t head) {
        return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && row % 4 == 0 && head % 4 == 0;
    };
    a.q_sign = 0;
    a.vec_q = vec(args.q, args.q_row, args.q_head);
    a.vec_out = vec(args.out, args.out_row, args.out_head);
    set_tc_workspace(a, workspace, kv.head_dim, num_sms);
    CUtensorMap k, v;
    if (!make_map(&k, kv.k, kv, a.box_rows) || !make_map(&v, kv.v, kv, a.box_rows)) return cudaErrorInvalidValue;
    return kv.head_dim == 128 ? run_tc32<128>(k, v, a, num_sms, st) : run_tc32<64>(k, v, a, num_sms, st);
}

}  // namespace pyxis
