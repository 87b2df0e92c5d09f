// tree_attn_tc.cu -- tree attention over bf16 pages on the tensor cores (tcgen05, TMEM, TMA).
//
//   S = Q K^T;  p = 2^(s - m);  O = sum p v;  out = O / sum p      (include/pyxis_serve.h)
//
// The rows of one (sequence, kv head) -- its nodes times the query heads that share the kv head --
// are the 128 TMEM lanes of a unit, so the cache is read once for all of them and the arithmetic of
// up to 128 rows (three 128 x 128 x HD products per 128 keys, about 1600 tensor cycles) stays below the
// time those keys take to arrive (64 KB per SM: about 2800 cycles): HBM bounds it.  Rows that are
// not there cost nothing but tensor cycles that are idle anyway.
//
// One CTA per SM.  The 128-key tiles of all units, in order, are dealt out evenly: CTA c takes tiles
// [W c / G, W (c + 1) / G), whatever sequences and heads they belong to, so ragged lengths and few
// sequences load all SMs alike.  A unit inside one CTA is written out at once; one that several
// CTAs share leaves unnormalised partial sums (at most two per CTA) that a second kernel joins.
//
// Warps: 0, 2 and 3 producers (of K, of V and of Q), 1 MMA issuer (and TMEM owner), 4-11 softmax: a row
// per thread, half of a tile's keys per warp.
//   producers  a tile's pages by TMA (one box per page, 128-byte swizzle) through a ring of tiles in the
//              order S_0, S_1, O_0, S_2, O_1, ... of the MMAs; the next segment's Q rows by cp.async while
//              the current one runs (the first segment's, which everything waits for, by the softmax warps)
//   MMA        S_j into one of three TMEM buffers; O += lo(P_j) V_j + hi(P_j) V_j with P_j from TMEM and
//              V_j as an MN-major operand, as it lies in the cache
//   softmax    reads S_j, masks the tiles that hold drafts or end inside, writes P_j over S_j.  The
//              running maximum is raised only when a tile exceeds it by more than 2^8 (then the row
//              of O in TMEM is rescaled); O / l does not depend on it.
// P is two bf16 terms, hi = bf16(p) and lo = bf16(p - hi), which leaves 2^-16 of each weight at most: O is
// f32 until its one rounding, as in the forms on the CUDA cores.  The tensor cores have the time for the
// second product (1600 of the 2800 cycles that a tile takes to arrive), and TMEM the room: both terms lie
// over the scores.  The softmax warps pay for it: with one term, off by 2^-9 of a weight, the two cases below
// took 103 and 38 us where they take 110 and 39 (2.3e-3 from 64 bits in place of 1.7e-3, relative l2).  O
// adds up in TMEM, where sums are cut off: 3e-4 of the sum over 64000 positions of one CTA, an eighth of
// the output's rounding.
//
// Measured (16 query and 8 kv heads of 128): one sequence of 131000 positions and 64 nodes 107 to 124 us, 4.3
// to 5.0 TB/s (a floor of 83 us), 16 sequences of 2303 positions 39 to 45 us with 16 nodes and 38 to 41 with
// one (20 and 21), 64 of them with one node 103 to 121 (84): the tiles pass at HBM's rate; the rest is the
// dealing and the first tiles' latency (about 4 us), the last tile's (3 us) and the join of the shared units
// (2 to 7 us).  The softmax warps have all 168 registers that a thread can have: for heads of 128 they spill
// 64 bytes.
#include <algorithm>
#include <atomic>

#include "tree_attn_tc.cuh"

namespace pyxis {
namespace {

constexpr int kRows = kTcRows, kTile = 128;
constexpr int kProdWarp = 0, kMmaWarp = 1, kProdWarpV = 2, kProdWarpQ = 3, kSmWarp0 = 4, kSmWarps = 8;
constexpr int kThreads = (kSmWarp0 + kSmWarps) * 32;
constexpr int kSBufs = 3;
constexpr uint32_t kTmemCols = 512, kOCol = kSBufs * kTile;
constexpr uint64_t kTimeoutNs = 2000000000ull;
constexpr float kRaise = 8.0f;
enum { kErrProd = 0x711, kErrMma = 0x712, kErrSoft = 0x713, kErrDrain = 0x714, kErrAlign = 0x715 };

template <int HD>
struct Smem {
    static constexpr int kDB = HD / 64;                  // 64-column panels of a row
    static constexpr uint32_t kPanel = kTile * 128;      // 128 rows x 128 B
    static constexpr uint32_t kEntry = kDB * kPanel;     // a tile of K or of V (or Q, panel after panel):
    static constexpr uint32_t kGroup = kDB * 1024;       // groups of 8 rows, each panel after panel
    static constexpr int kRing = HD == 128 ? 5 : 12;
    static constexpr uint32_t q = 0;  // two buffers: the next segment's rows come while this one runs
    static constexpr uint32_t ring = q + 2 * kEntry;
    static constexpr uint32_t bar = ring + kRing * kEntry;
    static constexpr int kBars = 2 * kRing + 5 + 3 * kSBufs;
    static constexpr uint32_t misc = bar + kBars * 8;
    static constexpr uint32_t red = misc + 64;               // [2 tiles][2 halves][128 rows] f32
    static constexpr uint32_t bytes = red + 2 * 2 * kRows * 4;
};
static_assert(Smem<128>::bytes <= 232448 && Smem<64>::bytes <= 232448, "227 KB of shared memory per CTA");

// bf16 A and B, f32 D; B MN-major or K-major.
__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attention_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                             const TcParams a) {
    using L = Smem<HD>;
    constexpr int kDB = L::kDB, kRing = L::kRing;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::bar);
    uint64_t *full = bars, *empty = bars + kRing, *qfull = bars + 2 * kRing, *qempty = qfull + 2, *drain = qempty + 2;
    // per score buffer: sfull (S_j landed), pfull (P_j written, V_j fit to be multiplied), odone (P_j V_j done)
    uint64_t *sfull = drain + 1, *pfull = sfull + kSBufs, *odone = pfull + kSBufs;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::misc);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::misc + 4);
    volatile int *bad = reinterpret_cast<volatile int *>(smem + L::misc + 8);  // [2]: 1 + the last segment of that parity with a draft's value that is not finite
    long long &start_off = *reinterpret_cast<long long *>(smem + L::misc + 16);
    int &start_seq = *reinterpret_cast<int *>(smem + L::misc + 24);
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
            tc::mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&qfull[b], 1);
            tc::mbar_init(&qempty[b], 1);
        }
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
    Walk<kTile> w;
    const Range r = begin_walk(a, w, warp_sum, start_seq, start_off);
    const long long total = r.total, lo = r.lo, count = r.count;
    const int g = r.ctas, c = blockIdx.x;
    if (count > 0) {
        // A segment's Q into buffer b, 16 bytes per copy, in the 128-byte swizzle, by `of` warps, of which this
        // is number `part`; rows past the unit's are left as they are (their lanes' results are never
        // written).  Done once the copies of all the warps' lanes are waited for and fenced.
        auto load_q = [&](const Walk<kTile> &s, int b, int part, int of) {
            uint8_t *dst = smem + L::q + b * L::kEntry;
            constexpr int kCh = HD / 8;  // 16-byte chunks of a row; a lane keeps its chunk
            const int r0 = s.row0(), rows = min(s.w.sh.nodes * p.group - r0, kRows), ch = lane % kCh;
            const char *head0 = p.q + s.w.sh.row0 * p.q_row + s.kvh() * p.group * p.q_head + ch * 16;
#pragma unroll 1
            for (int r = part * (32 / kCh) + lane / kCh; r < rows; r += of * (32 / kCh)) {
                const int t = (r0 + r) / p.group, h = r0 + r - t * p.group;
                const char *src = head0 + t * p.q_row + h * p.q_head;
                uint8_t *at = dst + (ch >> 3) * L::kPanel + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
                if (a.vec_q) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tc::smem_u32(at)), "l"(src) : "memory");
                } else {
                    const uint16_t *e = reinterpret_cast<const uint16_t *>(src);
                    uint32_t x[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = ((uint32_t)e[2 * k] | (uint32_t)e[2 * k + 1] << 16) ^ a.q_sign;
                    *reinterpret_cast<uint4 *>(at) = make_uint4(x[0], x[1], x[2], x[3]);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            tc::fence_proxy_async_smem();
            __syncwarp();
        };
        if (warp == kProdWarp || warp == kProdWarpV) {
            // ---------------------------------------------------------------- producers of K and of V
            const bool is_k = warp == kProdWarp;
            int e0 = 0, newest = -1;  // ring places of earlier segments; the latest place filled
            bool ok = true;
            auto wait = [&](uint64_t *bar, int phase) -> bool {
                return __all_sync(0xffffffffu, tc::mbar_wait_bounded(bar, (uint32_t)(phase & 1), abort_flag, p.err, kErrProd,
                                                                     kTimeoutNs));
            };
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
                auto issue = [&](int j, int page) -> bool {
                    const int e = e0 + (is_k ? (j == 0 ? 0 : 2 * j - 1) : (j == T - 1 ? 2 * T - 1 : 2 * j + 2));
                    const int slot = e % kRing;
                    if (!wait(&empty[slot], e / kRing - 1)) return false;
                    const int n = page_count(j);
                    if (lane == 0) tc::mbar_arrive_expect_tx(&full[slot], (uint32_t)(n * a.box_rows * HD * 2));
                    __syncwarp();
                    if (lane < n) {
                        uint8_t *dst = smem + L::ring + slot * L::kEntry + lane * a.box_rows * (HD * 2);
                        const int row = a.page_tiles == 1 ? 0 : (w.tb + j) % a.page_tiles * kTile;
                        const void *map = is_k ? &tm_k : &tm_v;
                        if (kDB == 1 || a.head_units) {
                            tma_load_5d(dst, map, 0, 0, kDB == 1 ? kvh : kvh * a.head_units, row / 8, page, &full[slot]);
                        } else {
                            for (int i = 0; i < a.box_rows / 8 * kDB; ++i)
                                tma_load_5d(dst + i * 1024, map, i % kDB * 64, 0, kvh, row / 8 + i / kDB, page, &full[slot]);
                        }
                    }
                    newest = e;
                    return true;
                };
                int cur = page_of(0);
                for (int j = 0; ok && j < T; ++j) {
                    const int next = page_of(j + 1);
                    ok = issue(j, cur);
                    cur = next;
                }
                e0 += 2 * T;
            }
            if (*abort_flag && lane == 0) {  // let the copies already issued land before the CTA exits
                volatile int no_abort = 0;
                for (int e = max(0, newest - kRing + 1); e <= newest; ++e)
                    tc::mbar_wait_bounded(&full[e % kRing], (uint32_t)((e / kRing) & 1), &no_abort, p.err, kErrDrain, 100000000ull);
            }
        } else if (warp == kMmaWarp) {
            // ---------------------------------------------------------------- MMA issuer
            if (elect_one()) {
                constexpr uint32_t idesc_s = idesc_bf16(kRows, kTile, false), idesc_o = idesc_bf16(kRows, HD, true);
                const uint64_t q_d = tc::desc_sw128(tc::smem_u32(smem + L::q));
                const uint64_t k_d = desc_rows_sw128(tc::smem_u32(smem + L::ring), 1024, L::kGroup), v_d = k_d;
                const uint32_t tO = tmem_base + kOCol;
                int slot = 0, fills = 0;   // ring
                int sb = 0, suse = 0;      // score buffer of the next S, and how often it was used
                int ob = 0, ouse = 0;      // of the next O
                auto wait = [&](uint64_t *bar, int phase) -> bool {
                    return tc::mbar_wait_bounded(bar, (uint32_t)(phase & 1), abort_flag, p.err, kErrMma, kTimeoutNs);
                };
                bool ok = true;
                auto score = [&](uint64_t qd) -> bool {
                    // the buffer's earlier probabilities have been multiplied, and K is there
                    if (!wait(&odone[sb], suse - 1) || !wait(&full[slot], fills)) return false;
                    tc::tc_fence_after();
                    const uint32_t tS = tmem_base + (uint32_t)(sb * kTile);
                    const uint64_t kd = k_d + (uint64_t)(slot * (L::kEntry >> 4));
#pragma unroll
                    for (int x = 0; x < kDB; ++x)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            tc::mma_f16(tS, qd + (uint64_t)(x * (L::kPanel >> 4) + kk * 2),
                                        kd + (uint64_t)(x * (1024 >> 4) + kk * 2), idesc_s, (uint32_t)(x | kk));
                    tc::mma_commit(&empty[slot]);
                    tc::mma_commit(&sfull[sb]);
                    if (++slot == kRing) slot = 0, ++fills;
                    if (++sb == kSBufs) sb = 0, ++suse;
                    return true;
                };
                auto output = [&](bool add) -> bool {
                    if (!wait(&full[slot], fills) || !wait(&pfull[ob], ouse)) return false;
                    tc::tc_fence_after();
                    const uint32_t tS = tmem_base + (uint32_t)(ob * kTile);
                    const uint64_t vd = v_d + (uint64_t)(slot * (L::kEntry >> 4));
#pragma unroll
                    for (int kk = 0; kk < kTile / 8; ++kk)  // 16 keys: 8 columns of P, 16 rows of V; lo, then hi
                        tc::mma_f16_ts(tO, tS + (uint32_t)((kk ^ (kTile / 16)) * 8),
                                       vd + (uint64_t)(kk % (kTile / 16) * (2 * L::kGroup >> 4)), idesc_o, (uint32_t)(add || kk > 0));
                    tc::mma_commit(&empty[slot]);
                    tc::mma_commit(&odone[ob]);
                    if (++slot == kRing) slot = 0, ++fills;
                    if (++ob == kSBufs) ob = 0, ++ouse;
                    return true;
                };
                for (int seg = 0; ok && w.next(p, a.n_seq); ++seg) {
                    const int T = w.te - w.tb;
                    const uint64_t qd = q_d + (uint64_t)((seg & 1) * (L::kEntry >> 4));
                    ok = wait(&qfull[seg & 1], seg >> 1) && score(qd);
                    for (int j = 1; ok && j < T; ++j) {
                        ok = score(qd);
                        if (ok && j == T - 1) tc::mma_commit(&qempty[seg & 1]);
                        ok = ok && output(j > 1);
                    }
                    if (ok && T == 1) tc::mma_commit(&qempty[seg & 1]);
                    ok = ok && output(T > 1);
                }
                // every MMA this thread issued must complete before TMEM is released
                tc::mma_commit(drain);
                volatile int no_abort = 0;
                tc::mbar_wait_bounded(drain, 0, &no_abort, p.err, kErrDrain, kTimeoutNs);
            }
        } else if (warp == kProdWarpQ) {
            // ---------------------------------------------------------------- producer of the next segment's Q
            bool ok = w.next(p, a.n_seq);  // the softmax warps load the first one's
            for (int seg = 1; ok && w.next(p, a.n_seq); ++seg) {
                ok = __all_sync(0xffffffffu, tc::mbar_wait_bounded(&qempty[seg & 1], (uint32_t)((seg / 2 - 1) & 1), abort_flag,
                                                                   p.err, kErrProd, kTimeoutNs));
                if (ok) load_q(w, seg & 1, 0, 1);
                if (ok && lane == 0) tc::mbar_arrive(&qfull[seg & 1]);
            }
        } else if (warp >= kSmWarp0) {
            // ---------------------------------------------------------------- softmax
            {
                Walk<kTile> first = w;
                if (first.next(p, a.n_seq)) load_q(first, 0, warp - kSmWarp0, kSmWarps);
                named_bar(5, kSmWarps * 32);
                if (threadIdx.x == kSmWarp0 * 32) tc::mbar_arrive(&qfull[0]);
            }
            const int quad = warp & 3;                 // TMEM lanes 32 quad .. 32 quad + 31
            const int half = (warp - kSmWarp0) >> 2;   // keys [64 half, +64) of each tile, columns [HD/2 half, +HD/2) of O
            const int row = quad * 32 + lane, tid = threadIdx.x - kSmWarp0 * 32;
            const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
            const uint32_t tO = tmem_base + lane_off + kOCol, tOh = tO + (uint32_t)(half * (HD / 2));
            const float c2 = fmaxf(fabsf(p.scale2), 1e-37f);  // a masked score stays -inf with scale 0, too
            auto wait = [&](uint64_t *bar, int phase) -> bool {
                return __all_sync(0xffffffffu, tc::mbar_wait_bounded(bar, (uint32_t)(phase & 1), abort_flag, p.err, kErrSoft,
                                                                     kTimeoutNs));
            };
            int b = 0, use = 0;    // score buffer and how often it was used
            int n0 = 0, seg = 0;   // tiles of earlier segments
            int swaps = 0;         // exchanges with the rows' other warp: they alternate between two buffers
            bool ok = true;
            for (; w.next(p, a.n_seq); ++seg) {
                const int T = w.te - w.tb, kvh = w.kvh(), r0 = w.row0();
                const SeqShape &sh = w.w.sh;
                const int rows = min(sh.nodes * p.group - r0, kRows);
                const bool active = quad * 32 < rows;  // the warp has rows
                unsigned long long mask = 0;
                if (row < rows) {
                    const int t = (r0 + row) / p.group;
                    mask = p.tree_mask ? p.tree_mask[sh.row0 + t] : (2ull << t) - 1;
                }
                float m_run = -INFINITY, l = 0.f;
                // after a failed wait the loops run on without work, so that the barriers of a row's two
                // warps keep their counts
                for (int j = 0; j < T; ++j) {
                    const long long k0 = (long long)(w.tb + j) * kTile;
                    const int pb = b == 0 ? kSBufs - 1 : b - 1, puse = b == 0 ? use - 1 : use;  // the tile before
                    const uint32_t tS = tmem_base + lane_off + (uint32_t)(b * kTile);
                    const bool tail = k0 + kTile > sh.ctx;
                    if (tail && ok) {
                        // V_j: rows that hold no key become zero (their weights are zero, but what lies
                        // there may be anything), and so do a draft's values that are not finite: the
                        // rows that do see the draft get them back below
                        const int ve = 2 * n0 + (j == T - 1 ? 2 * T - 1 : 2 * j + 2);  // its place in the ring's order
                        ok = wait(&full[ve % kRing], ve / kRing);
                        uint8_t *v = smem + L::ring + (ve % kRing) * L::kEntry;
                        const int valid = (int)min((long long)kTile, max(sh.total - k0, 0ll));
                        const int drafts = (int)min((long long)valid, max(sh.ctx - k0, 0ll));  // first draft's row
                        for (int i = tid; ok && i < (kTile - drafts) * (HD / 8); i += kSmWarps * 32) {
                            const int r = drafts + i / (HD / 8), ch = i % (HD / 8);
                            uint4 *at = reinterpret_cast<uint4 *>(v + (r >> 3) * L::kGroup + (ch >> 3) * 1024 + ((r & 7) << 7) + ((ch & 7) << 4));
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
                                bad[seg & 1] = seg + 1;
                            }
                        }
                        tc::fence_proxy_async_smem();
                    }
                    ok = ok && wait(&sfull[b], use);
                    if (active) {
                        float s[2][32];
                        float mt = -INFINITY;
                        if (ok) {
                        tc::tc_fence_after();
#pragma unroll
                        for (int ch = 0; ch < 2; ++ch)
                            tc::tmem_ld32_async(tS + (uint32_t)(half * 64 + ch * 32), reinterpret_cast<uint32_t(&)[32]>(s[ch]));
                        tc::tmem_wait_ld();
                        if (tail) {
                            // bit i: the row sees key k0 + 64 half + i -- the context, and the drafts of its mask
                            const long long d0 = sh.ctx - k0 - half * 64;  // the first draft's column
                            const int avail = (int)(sh.total - sh.ctx);
                            const unsigned long long m = avail >= 64 ? mask : mask & ((1ull << avail) - 1);
                            const unsigned long long vis = d0 >= 64 ? ~0ull : d0 > 0 ? ((1ull << d0) - 1) | m << d0 : d0 > -64 ? m >> -d0 : 0;
#pragma unroll
                            for (int ch = 0; ch < 2; ++ch)
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    s[ch][i] = ((uint32_t)(vis >> (ch * 32)) & (1u << i)) ? s[ch][i] : -INFINITY;
                        }
                        float x[4] = {s[0][0], s[0][1], s[1][0], s[1][1]};
#pragma unroll
                        for (int i = 2; i < 32; ++i)
#pragma unroll
                            for (int ch = 0; ch < 2; ++ch) x[ch * 2 + (i & 1)] = fmaxf(x[ch * 2 + (i & 1)], s[ch][i]);
                        mt = c2 * fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                        }
                        // the row's maximum over both halves; past this barrier both have read S, so P may
                        // be written over it
                        float *rd = red + (swaps++ & 1) * 2 * kRows;
                        rd[half * kRows + row] = mt;
                        named_bar(1 + quad, 64);
                        mt = fmaxf(mt, rd[(1 - half) * kRows + row]);
                        const bool raise = mt > m_run + kRaise || (m_run == -INFINITY && mt > m_run);
                        if (ok) {
                        if (__any_sync(0xffffffffu, raise)) {
                            const float alpha = raise ? ex2(m_run - mt) : 1.0f;
                            if (raise) m_run = mt, l *= alpha;
                            if (j > 0) {
                                // O of the tiles before, in TMEM, once they are all in
                                ok = wait(&odone[pb], puse);
                                tc::tc_fence_after();
#pragma unroll
                                for (int ch = 0; ch < HD / 64; ++ch) {
                                    uint32_t o[32];
                                    tc::tmem_ld32_async(tOh + (uint32_t)(ch * 32), o);
                                    tc::tmem_wait_ld();
#pragma unroll
                                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                    tc::tmem_st32(tOh + (uint32_t)(ch * 32), o);
                                }
                                tc::tmem_wait_st();
                            }
                        }
                        const float base = m_run == -INFINITY ? 0.f : m_run;
                        const float2 c22 = f2(c2, c2), base2 = f2(-base, -base);
                        float2 sum[2];
#pragma unroll
                        for (int ch = 0; ch < 2; ++ch) {
                            uint32_t hi[16], low[16];
                            sum[ch] = f2(0.f, 0.f);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 y = ffma2(f2(s[ch][i], s[ch][i + 1]), c22, base2), e = f2(ex2(y.x), ex2(y.y));
                                const uint32_t u = pack_bf16(e.x, e.y);
                                const float2 rest = ffma2(f2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)), f2(-1.f, -1.f), e);
                                hi[i / 2] = u;
                                low[i / 2] = pack_bf16(rest.x, rest.y);
                                sum[ch] = fadd2(sum[ch], e);
                            }
                            tmem_st16(tS + (uint32_t)(half * 32 + ch * 16), hi);
                            tmem_st16(tS + (uint32_t)(kTile / 2 + half * 32 + ch * 16), low);
                        }
                        sum[0] = fadd2(sum[0], sum[1]);
                        l += sum[0].x + sum[0].y;
                        tc::tmem_wait_st();
                        tc::tc_fence_before();
                        }
                    }
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&pfull[b]);
                    if (++b == kSBufs) b = 0, ++use;
                }
                n0 += T;
                ok = ok && wait(&odone[b == 0 ? kSBufs - 1 : b - 1], b == 0 ? use - 1 : use);
                if (active) {
                    float *rd = red + (swaps++ & 1) * 2 * kRows;
                    rd[half * kRows + row] = l;
                    named_bar(1 + quad, 64);
                    l += rd[(1 - half) * kRows + row];
                }
                if (active && ok) {
                    tc::tc_fence_after();
                    const bool fix = bad[seg & 1] == seg + 1, whole = w.whole();
                    const int t = (r0 + row) / p.group, h = kvh * p.group + (r0 + row) % p.group;
                    const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
                    const long long at = ((long long)(c * 2 + (w.from_before ? 0 : 1)) * kRows + row);
                    char *dst = p.out + (sh.row0 + t) * p.out_row + h * p.out_head;
                    float *part = a.part_o + (at - row) * HD + row;  // column-major: a warp's rows are adjacent
#pragma unroll 1
                    for (int ch = half * (HD / 64); ch < (half + 1) * (HD / 64); ++ch) {
                        float o[32];
                        tc::tmem_ld32(tO + (uint32_t)(ch * 32), o);
                        // the drafts' values that are not finite, for the rows that see them
                        if (fix && row < rows)
                            for (int d = 0; d < sh.nodes; ++d) {
                                const long long pos = sh.ctx + d;
                                if (!((mask >> d) & 1) || pos >= sh.total || pos < (long long)w.tb * kTile || pos >= (long long)w.te * kTile) continue;
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
                        // A weight's second term may be zero or negative: a sum over values that are not finite
                        // is taken from the values (a row whose weights are NaN is NaN).
                        const bool odd = row < rows && isfinite(l) && isnan(odd_mark(o));
                        if (__any_sync(0xffffffffu, odd)) {
                            const long long k0 = (long long)w.tb * kTile, k1 = (long long)w.te * kTile;
                            const float bad_ctx = odd_columns<__nv_bfloat16, 1>(p, sh, w.seq, kvh, ch * 32, k0, k1).x;
#pragma unroll 1
                            for (int i = 0; i < 32; ++i) {
                                const int d = ch * 32 + i;
                                float x = __shfl_sync(0xffffffffu, bad_ctx, i);
                                __nv_bfloat16 *y = reinterpret_cast<__nv_bfloat16 *>(dst) + d;
                                // (read back: o stays in registers)
                                if (!odd || isfinite(whole ? __bfloat162float(*y) : part[d * kRows])) continue;
                                x += odd_drafts<__nv_bfloat16>(p, sh, w.seq, kvh, d, mask, k0, k1);
                                if (x == 0.f) continue;
                                if (whole)
                                    store(y, x);
                                else
                                    part[d * kRows] = x;
                            }
                        }
                        __syncwarp();  // tcgen05.ld is the whole warp's
                    }
                    if (!whole && half == 0 && row < rows) a.part_ml[at * 2] = m_run, a.part_ml[at * 2 + 1] = l;
                    if (!whole && half == 0 && !w.from_before && row == 0) {
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

// K or V as [page][8-slot group][panel][slot of 8][64 columns], with panels counted over all heads, so that
// a page is one box in the order in which it lies in shared memory; heads that are not a whole number of
// panels apart are an axis of their own, and boxes are a group's panel.
bool make_map(CUtensorMap *m, const void *base, const pyxis_kv_pages &kv, int box_rows, int head_units) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const bool panels = head_units > 0 || kv.head_dim == 64;
    const int db = kv.head_dim / 64;
    const auto stride = [&](int n, int64_t s) { return (cuuint64_t)(n > 1 ? s : kv.head_dim) * 2; };  // of an axis of one: any
    cuuint64_t dims[5] = {(cuuint64_t)(panels ? 64 : kv.head_dim), 8, (cuuint64_t)kv.n_kv_heads, (cuuint64_t)kv.page_size / 8,
                          (cuuint64_t)kv.num_pages};
    cuuint64_t strides[4] = {(cuuint64_t)kv.slot_stride * 2, stride(kv.n_kv_heads, kv.head_stride),
                             stride(kv.page_size / 8, kv.slot_stride * 8), stride(kv.num_pages, kv.page_stride)};
    cuuint32_t box[5] = {64, 8, 1, (cuuint32_t)box_rows / 8, 1};
    if (head_units > 0) {
        dims[2] = (cuuint64_t)(kv.n_kv_heads - 1) * head_units + db;
        strides[1] = 128;
        box[2] = (cuuint32_t)db;
    } else if (!panels) {
        box[3] = 1;
    }
    cuuint32_t es[5] = {1, 1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void *>(base), dims, strides, box, es,
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
    return launch_tree_join<__nv_bfloat16, HD>(a, grid, st);
}

}  // namespace

// Boxes of whole 8-row swizzle groups: a page of 8 to 128 slots that tiles 128 keys, or a multiple of
// 128 slots.  Strides within the tensor map's 2^40 bytes.
bool tree_attention_tc_supported(const pyxis_tree_attention_args &a, const pyxis_kv_pages &kv) {
    const int64_t most = (int64_t)1 << 35;  // (a group of 8 slots is an axis)
    return kv.dtype == PYXIS_DTYPE_BF16 && kv.page_size % 8 == 0 &&
           (kTile % kv.page_size == 0 || kv.page_size % kTile == 0) && kv.page_stride < most &&
           kv.slot_stride < most && kv.head_stride < most;
}

size_t tree_attention_tc_workspace(const pyxis_kv_pages &kv, int num_sms) {
    return tree_tc_workspace(kv.head_dim, num_sms);
}

cudaError_t launch_tree_attention_tc(const TreeParams &p, const pyxis_tree_attention_args &args, const pyxis_kv_pages &kv,
                                     void *workspace, int num_sms, cudaStream_t st) {
    TcParams a;
    a.t = p;
    a.n_seq = (int)args.n_seq;
    a.box_rows = std::min(kv.page_size, kTile);
    a.tile_pages = kTile / a.box_rows;
    a.page_tiles = std::max(1, kv.page_size / kTile);
    const auto vec = [](const void *base, int64_t row, int64_t head) {
        return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && row % 8 == 0 && head % 8 == 0;
    };
    a.q_sign = p.scale2 < 0.f ? 0x80008000u : 0u;
    a.vec_q = a.q_sign == 0 && vec(args.q, args.q_row, args.q_head);
    a.vec_out = vec(args.out, args.out_row, args.out_head);
    set_tc_workspace(a, workspace, kv.head_dim, num_sms);
    // panels counted over all heads, as far as a coordinate reaches
    const int64_t units = kv.n_kv_heads == 1 ? kv.head_dim / 64 : kv.head_stride % 64 == 0 ? kv.head_stride / 64 : 0;
    a.head_units = kv.head_dim == 128 && units > 0 && units * kv.n_kv_heads < (1ll << 31) ? (int)units : 0;
    CUtensorMap k, v;
    if (!make_map(&k, kv.k, kv, a.box_rows, a.head_units) || !make_map(&v, kv.v, kv, a.box_rows, a.head_units))
        return cudaErrorInvalidValue;
    return kv.head_dim == 128 ? run_tc<128>(k, v, a, num_sms, st) : run_tc<64>(k, v, a, num_sms, st);
}

}  // namespace pyxis
