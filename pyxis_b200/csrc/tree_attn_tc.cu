// tree_attn_tc.cu -- tree attention over bf16 pages on the tensor cores (tcgen05, TMEM, TMA).
//
//   S = Q K^T;  p = 2^(s - m);  O = sum p v;  out = O / sum p      (include/pyxis_serve.h)
//
// The rows of one (sequence, kv head) -- its nodes times the query heads that share the kv head --
// are the 128 TMEM lanes of a unit, so the cache is read once for all of them and the arithmetic of
// up to 128 rows (two 128 x 128 x HD products per 128 keys, about 1000 tensor cycles) stays below the
// time those keys take to arrive (64 KB per SM: about 2800 cycles): HBM bounds it.  Rows that are
// not there cost nothing but tensor cycles that are idle anyway.
//
// One CTA per SM.  The 128-key tiles of all units, in order, are dealt out evenly: CTA c takes tiles
// [W c / G, W (c + 1) / G), whatever sequences and heads they belong to, so ragged lengths and few
// sequences load all SMs alike.  A unit inside one CTA is written out at once; one that several
// CTAs share leaves unnormalised partial sums (at most two per CTA) that a second kernel joins.
//
// Warps: 0 producer, 1 MMA issuer (and TMEM owner), 2-5 softmax, a row per thread.
//   producer   a tile's pages by TMA (one box per page and 64 columns, 128-byte swizzle) through a
//              ring of tiles in the order S_0, S_1, O_0, S_2, O_1, ... of the MMAs
//   MMA        S_j into one of three TMEM buffers; O += P_j V_j with P_j from TMEM and V_j as an
//              MN-major operand, as it lies in the cache
//   softmax    reads S_j, masks the tiles that hold drafts or end inside, writes P_j over S_j.  The
//              running maximum is raised only when a tile exceeds it by more than 2^8 (then the row
//              of O in TMEM is rescaled); O / l does not depend on it.
// P is rounded to bf16 (2^-9 of each weight), and l sums the rounded weights, so that rounding
// changes the weights' proportions, never their sum.
#include <algorithm>
#include <atomic>

#include "tc_ptx.cuh"
#include "tmap.cuh"
#include "tree_attn.cuh"

namespace pyxis {
namespace {

constexpr int kRows = 128, kTile = 128;
constexpr int kProdWarp = 0, kMmaWarp = 1, kSmWarp0 = 2, kSmWarps = 4;
constexpr int kThreads = (kSmWarp0 + kSmWarps) * 32;
constexpr int kSBufs = 3;
constexpr uint32_t kTmemCols = 512, kOCol = kSBufs * kTile;
constexpr uint64_t kTimeoutNs = 2000000000ull;
constexpr float kRaise = 8.0f;
constexpr int kMinTiles = 2;  // tiles per CTA before the next CTA gets any
enum { kErrProd = 0x711, kErrMma = 0x712, kErrSoft = 0x713, kErrDrain = 0x714 };

template <int HD>
struct Smem {
    static constexpr int kDB = HD / 64;                  // 64-column panels of a row
    static constexpr uint32_t kPanel = kTile * 128;      // 128 rows x 128 B
    static constexpr uint32_t kEntry = kDB * kPanel;     // a tile of K or of V
    static constexpr int kRing = HD == 128 ? 6 : 12;
    static constexpr uint32_t q = 0;
    static constexpr uint32_t ring = q + kEntry;
    static constexpr uint32_t bar = ring + kRing * kEntry;
    static constexpr int kBars = 2 * kRing + 2 + 3 * kSBufs;
    static constexpr uint32_t misc = bar + kBars * 8;
    static constexpr uint32_t bytes = misc + 64 + 1024;  // + alignment slack
};
static_assert(Smem<128>::bytes <= 232448 && Smem<64>::bytes <= 232448, "227 KB of shared memory per CTA");

struct TcParams {
    TreeParams t;
    int n_seq;
    int box_rows;       // rows of a TMA box: a page, or a tile of a larger page
    int tile_pages;     // boxes per tile
    int vec_q, vec_out; // 16-byte accesses to q's and out's rows
    uint32_t q_sign;    // flips q's signs for a negative scale
    float *part_o, *part_ml;  // [CTA][2][HD][128], [CTA][2][128][2]
    struct Shared *shared;    // [CTA]
};

// A unit that begins in a CTA and goes on in the next ones, up to CTA `last` (-1: the CTA has none).
// Its sums are in slot 1 of the first CTA and slot 0 of the others.
struct Shared {
    int last, row0, kvh, r0, rows;
};

PYXIS_DEVINL void tma_load_4d(void *dst, const void *tmap, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(tc::smem_u32(bar))
        : "memory");
}

// bf16 A and B, f32 D; B MN-major or K-major.
__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
// MN-major operand, 128-byte swizzle: 64-element panels `panel` bytes apart, 8-row groups 1024 bytes apart.
PYXIS_DEVINL uint64_t desc_mn_sw128(uint32_t smem_addr, uint32_t panel) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(panel >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
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

PYXIS_DEVINL uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&x);
}
// 2 N consecutive bf16 of an output row.
template <int N>
PYXIS_DEVINL void write_row(char *dst, const uint32_t (&u)[N], int vec) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < N; i += 4) reinterpret_cast<uint4 *>(dst)[i / 4] = make_uint4(u[i], u[i + 1], u[i + 2], u[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            reinterpret_cast<uint16_t *>(dst)[2 * i] = (uint16_t)u[i];
            reinterpret_cast<uint16_t *>(dst)[2 * i + 1] = (uint16_t)(u[i] >> 16);
        }
    }
}

// Units of a sequence: (kv head, 128-row tile); key tiles of each.
struct SeqWork {
    SeqShape sh;
    int row_tiles, units;
    long long tiles;
    PYXIS_DEVINL long long work() const { return units * tiles; }
};
PYXIS_DEVINL SeqWork seq_work(const TreeParams &p, int seq) {
    SeqWork w;
    w.sh = seq_shape(p, seq);
    w.row_tiles = (w.sh.nodes * p.group + kRows - 1) / kRows;
    w.units = w.row_tiles * p.n_kv;
    w.tiles = (w.sh.total + kTile - 1) / kTile;
    if (w.tiles < 1) w.tiles = 1;  // rows without keys still get their zeros
    return w;
}

// CTAs that share `total` tiles, and the first tile of CTA c.
PYXIS_DEVINL int shares(long long total, int grid) {
    const long long most = (total + kMinTiles - 1) / kMinTiles;
    return (int)(most < grid ? most : grid);
}
PYXIS_DEVINL long long first_tile(long long total, int c, int g) { return total * c / g; }

// The segments (a unit's tiles, or part of them) of a CTA's range, one after another.
struct Walk {
    SeqWork w;
    int seq, unit;
    long long tile, left;  // next tile of the unit, tiles left to this CTA
    long long tb, te;      // the segment
    bool from_before;      // its unit began in an earlier CTA
    bool first;
    PYXIS_DEVINL void begin(const TreeParams &p, int seq0, long long offset, long long count) {
        seq = seq0;
        w = seq_work(p, seq);
        unit = (int)(offset / w.tiles);
        tile = offset - unit * w.tiles;
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
                    w = seq_work(p, seq);
                } while (w.units == 0);
            }
        }
        from_before = tile > 0;  // only the CTA's first segment can start inside a unit
        first = false;
        tb = tile;
        te = w.tiles - tile < left ? w.tiles : tile + left;
        left -= te - tb;
        tile = te;
        return true;
    }
    PYXIS_DEVINL int kvh() const { return unit / w.row_tiles; }
    PYXIS_DEVINL int row0() const { return (unit % w.row_tiles) * kRows; }
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
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) x += warp_sum[w];
        *all += warp_sum[w];
    }
    return x;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attention_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                             const TcParams a) {
    using L = Smem<HD>;
    constexpr int kDB = L::kDB, kRing = L::kRing;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::bar);
    uint64_t *full = bars, *empty = bars + kRing, *qfull = bars + 2 * kRing, *drain = qfull + 1;
    // per score buffer: sfull (S_j landed), pfull (P_j written, V_j fit to be multiplied), odone (P_j V_j done)
    uint64_t *sfull = drain + 1, *pfull = sfull + kSBufs, *odone = pfull + kSBufs;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::misc);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::misc + 4);
    volatile int *bad = reinterpret_cast<volatile int *>(smem + L::misc + 8);  // [2]: a draft's value was not finite
    __shared__ long long warp_sum[kThreads / 32], start_off;
    __shared__ int start_seq;
    const TreeParams &p = a.t;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kRing; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        tc::mbar_init(qfull, kSmWarps);
        tc::mbar_init(drain, 1);
        for (int b = 0; b < kSBufs; ++b) {
            tc::mbar_init(&sfull[b], 1);
            tc::mbar_init(&pfull[b], kSmWarps);
            tc::mbar_init(&odone[b], 1);
        }
        *abort_flag = 0;
        bad[0] = bad[1] = 0;
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
    long long total = 0, mine = 0, incl = 0, sum;
    for (int s0 = 0; s0 < a.n_seq; s0 += kThreads) {
        const int s = s0 + threadIdx.x;
        mine = s < a.n_seq ? seq_work(p, s).work() : 0;
        incl = block_scan(mine, warp_sum, &sum);
        total += sum;
    }
    const int g = shares(total, gridDim.x), c = blockIdx.x;
    const long long lo = c < g ? first_tile(total, c, g) : 0, count = c < g ? first_tile(total, c + 1, g) - lo : 0;
    if (threadIdx.x == 0) a.shared[c].last = -1;
    if (count > 0) {
        long long before = 0;
        for (int s0 = 0; s0 < a.n_seq; s0 += kThreads) {
            const int s = s0 + threadIdx.x;
            if (a.n_seq > kThreads) {  // else they are still at hand
                mine = s < a.n_seq ? seq_work(p, s).work() : 0;
                incl = block_scan(mine, warp_sum, &sum);
            }
            const long long first = before + incl - mine;
            if (mine > 0 && lo >= first && lo < first + mine) start_seq = s, start_off = lo - first;
            before += sum;
        }
        __syncthreads();
        Walk w;
        w.begin(p, start_seq, start_off, count);
        if (warp == kProdWarp) {
            // ---------------------------------------------------------------- TMA producer
            int e = 0;
            bool ok = true;
            while (ok && w.next(p, a.n_seq)) {
                const int T = (int)(w.te - w.tb), kvh = w.kvh();
                const int32_t *table = p.block_table + w.seq * p.table_stride;
                // this lane's page of tile tb + j (-1: none), and how many of the tile's pages exist
                auto page_count = [&](int j) -> int {
                    const long long rest = w.w.sh.total - (w.tb + j) * kTile;
                    if (rest <= 0 || j >= T) return 0;
                    const long long n = (rest + a.box_rows - 1) / a.box_rows;
                    return (int)(n < a.tile_pages ? n : a.tile_pages);
                };
                auto page_of = [&](int j) -> int {
                    if (lane >= page_count(j)) return 0;
                    const int id = __ldg(table + ((w.tb + j) * kTile + lane * a.box_rows) / p.page_size);
                    return min(max(id, 0), p.num_pages - 1);
                };
                auto issue = [&](bool is_k, int j, int page) -> bool {
                    const int s = e % kRing;
                    if (e >= kRing && !__all_sync(0xffffffffu, tc::mbar_wait_bounded(&empty[s], (uint32_t)((e / kRing - 1) & 1),
                                                                                      abort_flag, p.err, kErrProd, kTimeoutNs)))
                        return false;
                    const int n = page_count(j);
                    if (lane == 0) tc::mbar_arrive_expect_tx(&full[s], (uint32_t)(n * a.box_rows * HD * 2));
                    __syncwarp();
                    if (lane < n) {
                        uint8_t *dst = smem + L::ring + s * L::kEntry + lane * a.box_rows * 128;
                        const int slot = (int)(((w.tb + j) * kTile + lane * a.box_rows) % p.page_size);
#pragma unroll
                        for (int x = 0; x < kDB; ++x)
                            tma_load_4d(dst + x * L::kPanel, is_k ? &tm_k : &tm_v, x * 64, kvh, slot, page, &full[s]);
                    }
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
                for (int x = e > kRing ? e - kRing : 0; x < e; ++x)
                    tc::mbar_wait_bounded(&full[x % kRing], (uint32_t)((x / kRing) & 1), &no_abort, p.err, kErrDrain,
                                          100000000ull);
            }
        } else if (warp == kMmaWarp) {
            // ---------------------------------------------------------------- MMA issuer
            if (lane == 0) {
                constexpr uint32_t idesc_s = idesc_bf16(kRows, kTile, false), idesc_o = idesc_bf16(kRows, HD, true);
                const uint64_t q_d = tc::desc_sw128(tc::smem_u32(smem + L::q));
                const uint64_t k_d = tc::desc_sw128(tc::smem_u32(smem + L::ring));
                const uint64_t v_d = desc_mn_sw128(tc::smem_u32(smem + L::ring), L::kPanel);
                const uint32_t tO = tmem_base + kOCol;
                int e = 0, seg = 0;
                long long n0 = 0;  // tiles of earlier segments
                bool ok = true;
                auto score = [&](long long n) -> bool {
                    const int b = (int)(n % kSBufs), s = e % kRing;
                    const long long use = n / kSBufs;
                    // the buffer's earlier probabilities have been multiplied
                    if (use > 0 && !tc::mbar_wait_bounded(&odone[b], (uint32_t)((use - 1) & 1), abort_flag, p.err, kErrMma,
                                                          kTimeoutNs))
                        return false;
                    if (!tc::mbar_wait_bounded(&full[s], (uint32_t)((e / kRing) & 1), abort_flag, p.err, kErrMma, kTimeoutNs))
                        return false;
                    tc::tc_fence_after();
                    const uint32_t tS = tmem_base + (uint32_t)(b * kTile);
#pragma unroll
                    for (int x = 0; x < kDB; ++x)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            tc::mma_f16(tS, q_d + (uint64_t)(x * (L::kPanel >> 4) + kk * 2),
                                        k_d + (uint64_t)(s * (L::kEntry >> 4) + x * (L::kPanel >> 4) + kk * 2), idesc_s,
                                        (uint32_t)(x | kk));
                    tc::mma_commit(&empty[s]);
                    tc::mma_commit(&sfull[b]);
                    ++e;
                    return true;
                };
                auto output = [&](long long n, bool add) -> bool {
                    const int b = (int)(n % kSBufs), s = e % kRing;
                    const long long use = n / kSBufs;
                    if (!tc::mbar_wait_bounded(&full[s], (uint32_t)((e / kRing) & 1), abort_flag, p.err, kErrMma, kTimeoutNs) ||
                        !tc::mbar_wait_bounded(&pfull[b], (uint32_t)(use & 1), abort_flag, p.err, kErrMma, kTimeoutNs))
                        return false;
                    tc::tc_fence_after();
                    const uint32_t tS = tmem_base + (uint32_t)(b * kTile);
#pragma unroll
                    for (int kk = 0; kk < kTile / 16; ++kk)  // 16 keys: 8 columns of P, 16 rows of V
                        tc::mma_f16_ts(tO, tS + (uint32_t)(kk * 8), v_d + (uint64_t)(s * (L::kEntry >> 4) + kk * (2048 >> 4)),
                                       idesc_o, (uint32_t)(add || kk > 0));
                    tc::mma_commit(&empty[s]);
                    tc::mma_commit(&odone[b]);
                    ++e;
                    return true;
                };
                for (; ok && w.next(p, a.n_seq); ++seg) {
                    const int T = (int)(w.te - w.tb);
                    ok = tc::mbar_wait_bounded(qfull, (uint32_t)(seg & 1), abort_flag, p.err, kErrMma, kTimeoutNs) && score(n0);
                    for (int j = 1; ok && j < T; ++j) ok = score(n0 + j) && output(n0 + j - 1, j > 1);
                    ok = ok && output(n0 + T - 1, T > 1);
                    n0 += T;
                }
                // every MMA this thread issued must complete before TMEM is released
                tc::mma_commit(drain);
                volatile int no_abort = 0;
                tc::mbar_wait_bounded(drain, 0, &no_abort, p.err, kErrDrain, kTimeoutNs);
            }
        } else {
            // ---------------------------------------------------------------- softmax
            const int quad = warp & 3;  // TMEM lanes 32 quad .. 32 quad + 31
            const int row = quad * 32 + lane, tid = threadIdx.x - kSmWarp0 * 32;
            const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
            const uint32_t tO = tmem_base + lane_off + kOCol;
            const float c2 = fmaxf(fabsf(p.scale2), 1e-37f);  // a masked score stays -inf with scale 0, too
            auto wait = [&](uint64_t *bar, long long phase) -> bool {
                return __all_sync(0xffffffffu, tc::mbar_wait_bounded(bar, (uint32_t)(phase & 1), abort_flag, p.err, kErrSoft,
                                                                     kTimeoutNs));
            };
            long long n0 = 0;
            int seg = 0;
            bool ok = true;
            for (; ok && w.next(p, a.n_seq); ++seg) {
                const int T = (int)(w.te - w.tb), kvh = w.kvh(), r0 = w.row0();
                const SeqShape &sh = w.w.sh;
                const int rows = min(sh.nodes * p.group - r0, kRows);
                const bool active = quad * 32 < rows;  // the warp has rows
                // ---- Q of the segment; the last segment's MMAs are done (odone)
                constexpr int kCh = HD / 8, kQUnroll = kCh;  // 16-byte chunks of a row, loads in flight
                for (int i0 = tid; i0 < rows * kCh; i0 += kSmWarps * 32 * kQUnroll) {
                    uint4 x[kQUnroll];
#pragma unroll
                    for (int k = 0; k < kQUnroll; ++k) {
                        const int i = i0 + k * kSmWarps * 32, r = r0 + i / kCh, t = r / p.group;
                        if (i >= rows * kCh) break;
                        const char *src = p.q + (sh.row0 + t) * p.q_row + (kvh * p.group + r - t * p.group) * p.q_head +
                                          (i % kCh) * 16;
                        if (a.vec_q) {
                            x[k] = *reinterpret_cast<const uint4 *>(src);
                        } else {
                            const uint16_t *e = reinterpret_cast<const uint16_t *>(src);
                            x[k] = make_uint4((uint32_t)e[0] | (uint32_t)e[1] << 16, (uint32_t)e[2] | (uint32_t)e[3] << 16,
                                              (uint32_t)e[4] | (uint32_t)e[5] << 16, (uint32_t)e[6] | (uint32_t)e[7] << 16);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kQUnroll; ++k) {
                        const int i = i0 + k * kSmWarps * 32, r = i / kCh, ch = i % kCh;
                        if (i >= rows * kCh) break;
                        x[k].x ^= a.q_sign, x[k].y ^= a.q_sign, x[k].z ^= a.q_sign, x[k].w ^= a.q_sign;
                        *reinterpret_cast<uint4 *>(smem + L::q + (ch >> 3) * L::kPanel + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) =
                            x[k];
                    }
                }
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(qfull);
                unsigned long long mask = 0;
                if (row < rows) {
                    const int t = (r0 + row) / p.group;
                    mask = p.tree_mask ? p.tree_mask[sh.row0 + t] : (2ull << t) - 1;
                }
                float m_run = -INFINITY, l = 0.f;
                for (int j = 0; ok && j < T; ++j) {
                    const long long n = n0 + j;
                    const int b = (int)(n % kSBufs);
                    const long long k0 = (w.tb + j) * kTile;
                    const uint32_t tS = tmem_base + lane_off + (uint32_t)(b * kTile);
                    const bool tail = k0 + kTile > sh.ctx;
                    if (tail) {
                        // V_j: rows that hold no key become zero (their weights are zero, but what lies
                        // there may be anything), and so do a draft's values that are not finite: the
                        // rows that do see the draft get them back below
                        const long long ve = 2 * n0 + (j == T - 1 ? 2 * T - 1 : 2 * j + 2);
                        ok = wait(&full[ve % kRing], ve / kRing);
                        if (!ok) break;
                        uint8_t *v = smem + L::ring + (ve % kRing) * L::kEntry;
                        const int valid = (int)min((long long)kTile, max(sh.total - k0, 0ll));
                        const int drafts = (int)min((long long)valid, max(sh.ctx - k0, 0ll));  // first draft's row
                        for (int i = tid; i < (kTile - drafts) * (HD / 8); i += kSmWarps * 32) {
                            const int r = drafts + i / (HD / 8), ch = i % (HD / 8);
                            uint4 *at = reinterpret_cast<uint4 *>(v + (ch >> 3) * L::kPanel + r * 128 + ((ch & 7) << 4));
                            if (r >= valid) {
                                *at = make_uint4(0, 0, 0, 0);
                                continue;
                            }
                            uint4 x = *at;
                            uint32_t *u = &x.x;
                            bool any = false;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if ((u[k] & 0x7F80u) == 0x7F80u) u[k] &= 0xFFFF0000u, any = true;
                                if ((u[k] & 0x7F800000u) == 0x7F800000u) u[k] &= 0xFFFFu, any = true;
                            }
                            if (any) {
                                *at = x;
                                bad[seg & 1] = 1;
                            }
                        }
                        tc::fence_proxy_async_smem();
                    }
                    ok = wait(&sfull[b], n / kSBufs);
                    if (!ok) break;
                    if (active) {
                        tc::tc_fence_after();
                        float s[4][32];
#pragma unroll
                        for (int ch = 0; ch < 4; ++ch)
                            tc::tmem_ld32_async(tS + (uint32_t)(ch * 32), reinterpret_cast<uint32_t(&)[32]>(s[ch]));
                        tc::tmem_wait_ld();
                        if (tail) {
                            // bit i: the row sees key k0 + i -- the context, and the drafts of its mask
                            const long long d0 = sh.ctx - k0;  // the first draft's column
                            const int avail = (int)(sh.total - sh.ctx);
                            const unsigned long long m = avail >= 64 ? mask : mask & ((1ull << avail) - 1);
                            unsigned long long v0 = ~0ull, v1 = ~0ull;
                            if (d0 < 128) {
                                const int d = d0 < -64 ? -64 : (int)d0;
                                v0 = d >= 64 ? ~0ull : d > 0 ? ((1ull << d) - 1) | m << d : d > -64 ? m >> -d : 0;
                                v1 = d > 64 ? ((1ull << (d - 64)) - 1) | m << (d - 64) : d == 64 ? m : d > 0 ? m >> (64 - d) : 0;
                            }
                            const uint32_t vis[4] = {(uint32_t)v0, (uint32_t)(v0 >> 32), (uint32_t)v1, (uint32_t)(v1 >> 32)};
#pragma unroll
                            for (int ch = 0; ch < 4; ++ch)
#pragma unroll
                                for (int i = 0; i < 32; ++i) s[ch][i] = (vis[ch] & (1u << i)) ? s[ch][i] : -INFINITY;
                        }
                        float x[4] = {s[0][0], s[1][0], s[2][0], s[3][0]};
#pragma unroll
                        for (int i = 1; i < 32; ++i)
#pragma unroll
                            for (int ch = 0; ch < 4; ++ch) x[ch] = fmaxf(x[ch], s[ch][i]);
                        const float mt = c2 * fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                        const bool raise = mt > m_run + kRaise || (m_run == -INFINITY && mt > m_run);
                        if (__any_sync(0xffffffffu, raise)) {
                            const float alpha = raise ? ex2(m_run - mt) : 1.0f;
                            if (raise) m_run = mt, l *= alpha;
                            if (j > 0) {
                                // O of the tiles before, in TMEM, once they are all in
                                ok = wait(&odone[(n - 1) % kSBufs], (n - 1) / kSBufs);
                                if (!ok) break;
                                tc::tc_fence_after();
#pragma unroll
                                for (int ch = 0; ch < HD / 32; ++ch) {
                                    uint32_t o[32];
                                    tc::tmem_ld32_async(tO + (uint32_t)(ch * 32), o);
                                    tc::tmem_wait_ld();
#pragma unroll
                                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                    tc::tmem_st32(tO + (uint32_t)(ch * 32), o);
                                }
                                tc::tmem_wait_st();
                            }
                        }
                        const float base = m_run == -INFINITY ? 0.f : m_run;
                        const float2 c22 = f2(c2, c2), base2 = f2(-base, -base);
                        float2 sum[4];
#pragma unroll
                        for (int ch = 0; ch < 4; ++ch) {
                            uint32_t pk[16];
                            sum[ch] = f2(0.f, 0.f);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 y = ffma2(f2(s[ch][i], s[ch][i + 1]), c22, base2);
                                const uint32_t u = pack_bf16(ex2(y.x), ex2(y.y));
                                pk[i / 2] = u;
                                sum[ch] = fadd2(sum[ch], f2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)));
                            }
                            tmem_st16(tS + (uint32_t)(ch * 16), pk);
                        }
                        sum[0] = fadd2(fadd2(sum[0], sum[1]), fadd2(sum[2], sum[3]));
                        l += sum[0].x + sum[0].y;
                        tc::tmem_wait_st();
                        tc::tc_fence_before();
                    }
                    // the next segment's flag: every warp has read it (two segments ago, before it
                    // loaded this one's Q), none is past this segment before this arrival
                    if (j == T - 1 && tid == 0) bad[(seg + 1) & 1] = 0;
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&pfull[b]);
                }
                if (!ok) break;
                n0 += T;
                ok = wait(&odone[(n0 - 1) % kSBufs], (n0 - 1) / kSBufs);
                if (!ok) break;
                if (active) {
                    tc::tc_fence_after();
                    const bool fix = bad[seg & 1] != 0, whole = w.whole();
                    const int t = (r0 + row) / p.group, h = kvh * p.group + (r0 + row) % p.group;
                    const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
                    const long long at = ((long long)(c * 2 + (w.from_before ? 0 : 1)) * kRows + row);
                    char *dst = p.out + (sh.row0 + t) * p.out_row + h * p.out_head;
                    float *part = a.part_o + (at - row) * HD + row;  // column-major: a warp's rows are adjacent
#pragma unroll 1
                    for (int ch = 0; ch < HD / 32; ++ch) {
                        float o[32];
                        tc::tmem_ld32(tO + (uint32_t)(ch * 32), o);
                        // the drafts' values that are not finite, for the rows that see them
                        if (fix && row < rows)
                            for (int d = 0; d < sh.nodes; ++d) {
                                const long long pos = sh.ctx + d;
                                if (!((mask >> d) & 1) || pos >= sh.total || pos < w.tb * kTile || pos >= w.te * kTile) continue;
                                const int page = min(max(p.block_table[w.seq * p.table_stride + pos / p.page_size], 0),
                                                     p.num_pages - 1);
                                const __nv_bfloat16 *v = reinterpret_cast<const __nv_bfloat16 *>(
                                    p.v + page * p.page_stride + (pos % p.page_size) * p.slot_stride + kvh * p.head_stride);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float x = __bfloat162float(v[ch * 32 + i]);
                                    if (!isfinite(x)) o[i] += x;
                                }
                            }
                        if (row < rows && whole) {
                            uint32_t u[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) u[i] = pack_bf16(o[2 * i] * inv, o[2 * i + 1] * inv);
                            write_row(dst + ch * 64, u, a.vec_out);
                        } else if (row < rows) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) part[(ch * 32 + i) * kRows] = o[i];
                        }
                        __syncwarp();  // tcgen05.ld is the whole warp's
                    }
                    if (!whole && row < rows) a.part_ml[at * 2] = m_run, a.part_ml[at * 2 + 1] = l;
                    if (!whole && !w.from_before && row == 0) {
                        const long long end = lo + count + (w.w.tiles - w.te) - 1;  // the unit's last tile
                        a.shared[c] = Shared{(int)(((end + 1) * g + total - 1) / total) - 1, sh.row0, kvh, r0, rows};
                    }
                    tc::tc_fence_before();
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == kMmaWarp) tc::tmem_dealloc(tmem_base, kTmemCols);
}

// Joins the unit that CTA blockIdx.x of the first kernel left unfinished, kJoinCols columns: a row per
// thread.  Many small blocks and several CTAs' sums in flight per thread: a unit shared by all the
// SMs' CTAs is read at L2 speed, not one latency per CTA.
constexpr int kJoinCols = 8, kJoinUnroll = 4;
template <int HD>
__global__ void __launch_bounds__(kRows) tree_join_tc_kernel(const TcParams a) {
    const TreeParams &p = a.t;
    pdl_wait();
    pdl_trigger();
    const int c0 = blockIdx.x, row = threadIdx.x, col = blockIdx.y * kJoinCols;
    const Shared u = a.shared[c0];
    if (u.last < 0 || row >= u.rows) return;
    const auto slot = [&](int c) -> long long { return c == c0 ? c * 2 + 1 : c * 2; };
    const auto ml_of = [&](int c) { return reinterpret_cast<const float2 *>(a.part_ml)[slot(c) * kRows + row]; };
    float o[kJoinCols] = {}, l = 0.f, m = -INFINITY;
    for (int c = c0; c <= u.last; c += kJoinUnroll) {
        float2 ml[kJoinUnroll];
        float x[kJoinUnroll][kJoinCols];
#pragma unroll
        for (int k = 0; k < kJoinUnroll; ++k) {
            ml[k] = c + k <= u.last ? ml_of(c + k) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < kJoinCols; ++i)
                x[k][i] = c + k <= u.last ? a.part_o[(slot(c + k) * HD + col + i) * kRows + row] : 0.f;
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
    uint32_t w[kJoinCols / 2];
#pragma unroll
    for (int i = 0; i < kJoinCols / 2; ++i) w[i] = pack_bf16(o[2 * i] * inv, o[2 * i + 1] * inv);
    write_row(p.out + (u.row0 + t) * p.out_row + head * p.out_head + col * 2, w, a.vec_out);
}

// [page][slot][head][64-column panel] of K or V
bool make_map(CUtensorMap *m, const void *base, const pyxis_kv_pages &kv, int box_rows) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const auto stride = [&](int n, int64_t s) { return (cuuint64_t)(n > 1 ? s : kv.head_dim) * 2; };  // of an axis of one: any
    cuuint64_t dims[4] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.n_kv_heads, (cuuint64_t)kv.page_size,
                          (cuuint64_t)kv.num_pages};
    cuuint64_t strides[3] = {stride(kv.n_kv_heads, kv.head_stride), stride(kv.page_size, kv.slot_stride),
                             stride(kv.num_pages, kv.page_stride)};
    cuuint32_t box[4] = {64, 1, (cuuint32_t)box_rows, 1};
    cuuint32_t es[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD>
cudaError_t run_tc(const CUtensorMap &k, const CUtensorMap &v, const TcParams &a, int grid, cudaStream_t st) {
    auto kern = tree_attention_tc_kernel<HD>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = once_per_device(done, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Smem<HD>::bytes);
    });
    if (e != cudaSuccess) return e;
    PdlScope pdl;
    e = launch_kernel(kern, dim3(grid), dim3(kThreads), Smem<HD>::bytes, st, k, v, a);
    if (e != cudaSuccess) return e;
    return launch_kernel(tree_join_tc_kernel<HD>, dim3(grid, HD / kJoinCols), dim3(kRows), 0, st, a);
}

}  // namespace

// Boxes of whole 8-row swizzle groups: a page of 8 to 128 slots that tiles 128 keys, or a multiple of
// 128 slots.  Strides within the tensor map's 2^40 bytes.
bool tree_attention_tc_supported(const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv) {
    const int64_t most = (int64_t)1 << 38;
    return kv.dtype == PYXIS_DTYPE_BF16 && kv.page_size % 8 == 0 &&
           (kTile % kv.page_size == 0 || kv.page_size % kTile == 0) && kv.page_stride < most &&
           kv.slot_stride < most && kv.head_stride < most;
}

size_t tree_attention_tc_workspace(const pyxis_kv_pages &kv, int num_sms) {
    return (size_t)num_sms * (2 * kRows * (kv.head_dim + 2) * 4 + sizeof(Shared));
}

cudaError_t launch_tree_attention_tc(const TreeParams &p, const pyxis_tree_attention_args &args, const pyxis_kv_pages &kv,
                                     void *workspace, int num_sms, cudaStream_t st) {
    TcParams a;
    a.t = p;
    a.n_seq = (int)args.n_seq;
    a.box_rows = std::min(kv.page_size, kTile);
    a.tile_pages = kTile / a.box_rows;
    const auto vec = [](const void *base, int64_t row, int64_t head) {
        return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && row % 8 == 0 && head % 8 == 0;
    };
    a.vec_q = vec(args.q, args.q_row, args.q_head);
    a.vec_out = vec(args.out, args.out_row, args.out_head);
    a.q_sign = p.scale2 < 0.f ? 0x80008000u : 0u;
    a.part_o = (float *)workspace;
    a.part_ml = a.part_o + (size_t)num_sms * 2 * kRows * kv.head_dim;
    a.shared = reinterpret_cast<Shared *>(a.part_ml + (size_t)num_sms * 2 * kRows * 2);
    CUtensorMap k, v;
    if (!make_map(&k, kv.k, kv, a.box_rows) || !make_map(&v, kv.v, kv, a.box_rows)) return cudaErrorInvalidValue;
    return kv.head_dim == 128 ? run_tc<128>(k, v, a, num_sms, st) : run_tc<64>(k, v, a, num_sms, st);
}

}  // namespace pyxis
