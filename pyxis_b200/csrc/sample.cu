// sample.cu -- temperature, top-k, top-p and min-p sampling of one token per row from given uniform
// numbers (src/sampler.rs:23-110 on the device; definition in include/pyxis_serve.h).
//
// Every filter keeps a prefix of the order "largest logit first, equal ones by index", so the
// prefixes are nested and the kept weight is the smallest of the prefixes' weights.  With that
// total Z the drawn token is the first one in the order whose running sum of weights exceeds u Z:
// nothing is sorted and no mask is kept; three times at most one element of the order is located
// -- by count (the k-th), by weight (p Z_k) and by weight (u Z).
//
// A cluster of CTAs holds a row in shared memory (one pass over HBM).  Elements are located in two
// steps: the cluster gathers a small set that holds the element into the leader CTA's shared memory,
// and the leader narrows that set down by histograms over the 64-bit (value, index) key until a
// warp can rank what is left.  The set is
//   - with top_k up to kMaxTopK: everything from the k-th largest of the threads' maxima up (each of
//     them is an element of its own, so the k-th largest element is not below it); about k elements,
//     and the other filters and the draw are settled among them without another pass;
//   - else: the bin of a histogram of the row (weights by (max - x) / temperature, 1/32 nat a bin)
//     that the running sum over the bins names, one gather per element sought.
// A set that is too large (flat or heavily tied rows) is cut down first, by the cluster's
// histograms over the same key.
//
// Weights are exp() in f64 rounded to 2^-44 (less for rows of over 2^18 tokens, so that a row's sum
// stays below 2^63): integer sums are exact in any order, so neither the atomics' order nor the
// cluster's size changes a token, and the sums are far finer than the spacing of uniform numbers.
//
// Latency bounds it: a row is read once (0.6 MB: 0.1 us of the memory's time), but maximum, histogram,
// gather and narrowing follow one another, with a cluster barrier between.  Measured, 151936 tokens: one
// f32 row with top-p 23 us, 64 bf16 rows with top-k, top-p and min-p 16.4 us, with top-p alone 78 us
// (the weights' exponentials and the histograms' shared-memory atomics).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "serve.h"

namespace pyxis {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;  // 1/32 nat each: 32 nats, past which a weight rounds to 0
constexpr int kPerThread = kBins / kThreads;
constexpr float kBinsPerNat = 32.0f;
constexpr int kCand = 2048;  // elements that the leader takes
constexpr int kMaxTopK = 1024;
constexpr int kRank = 128;   // elements that are ranked against one another
constexpr int kMaxCluster = 16;     // 8 is portable; 16 where the device takes it
constexpr int kTable = 256;  // steps of 2 in the exponentials' table

struct SampleArgs {
    const void *logits;
    size_t n, ld;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int32_t top_k_all;
    int32_t *idx;
    float *prob;
    int shift;     // weights are multiples of 2^-shift
    int last_bin;  // elements of later bins have weight 0
    unsigned cap;  // elements of a segment that shared memory holds
};

using u64 = unsigned long long;

struct Histogram {
    unsigned lo[kBins], hi[kBins], cnt[kBins];  // weight as two words, count
};

// A part of the order: keys lo .. hi, and the weight and count of what comes before it.
struct Range {
    u64 lo, hi, ex_mass;
    unsigned ex_count, count;
};

struct Shared {
    union {
        u64 cand[kCand];
        Histogram sub;  // of a key range, while the cluster cuts a set down
    };
    Histogram row;      // of the row; then, in the leader, of the candidates' key range
    double table[kTable];  // 2^(shift - j / 256)
    u64 scan[kWarps];
    unsigned scan_cnt[kWarps];
    u64 rank_min[kMaxCluster], rank_max[kMaxCluster], rank_mass[kMaxCluster];
    float rank_top[kMaxCluster];
    Range ctl[4];       // what the leader tells the cluster: per element sought
    int bin[4];         // its bin (the last bin of a top-k set), -1: nothing to seek
    unsigned ncand;
    Range narrow;
    u64 few[kRank], few_w[kRank];
    unsigned nfew;
    u64 found_mass, found_w, found_key;
    double temperature, top_p, min_p, u;  // the row's parameters, read while the row arrives
    int top_k;
};

PYXIS_DEVINL float widen(float x) { return x; }
PYXIS_DEVINL float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
PYXIS_DEVINL T lowest() {
    return T(-INFINITY);
}

// Order-preserving key of a finite or infinite value and its index: larger values first, then
// smaller indexes; -0 ties with +0.
PYXIS_DEVINL u64 key_of(float v, unsigned idx) {
    if (v == 0.0f) v = 0.0f;
    const unsigned u = __float_as_uint(v);
    const unsigned ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((u64)ord << 32) | (0xFFFFFFFFu - idx);
}
PYXIS_DEVINL float value_of(u64 key) {
    const unsigned ord = (unsigned)(key >> 32);
    return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7FFFFFFFu) : ~ord);
}

// 64-bit add into two 32-bit words of (this or another CTA's) shared memory: the carry goes with
// the value the low word had, so the pair is exact once all adds are done.
PYXIS_DEVINL void add_wide(unsigned *lo, unsigned *hi, u64 w) {
    const unsigned wl = (unsigned)w;
    const unsigned old = atomicAdd(lo, wl);
    const unsigned c = (unsigned)(w >> 32) + (old + wl < old ? 1u : 0u);
    if (c) atomicAdd(hi, c);
}
// The adds of four elements (b < 0: none) into this CTA's own histogram: the four low words' atomics
// are all in flight before the first one's old value is needed for its carry.
PYXIS_DEVINL void add_wide4(Histogram &h, const int (&b)[4], const u64 (&w)[4], bool count) {
    const unsigned lo = (unsigned)__cvta_generic_to_shared(h.lo), hi = (unsigned)__cvta_generic_to_shared(h.hi),
                   cnt = (unsigned)__cvta_generic_to_shared(h.cnt);
    unsigned old[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        asm volatile("{\n .reg .pred p;\n setp.ge.s32 p, %3, 0;\n mov.u32 %0, 0;\n @p atom.shared.add.u32 %0, [%1], %2;\n}\n"
                     : "=r"(old[j])
                     : "r"(lo + 4 * b[j]), "r"((unsigned)w[j]), "r"(b[j])
                     : "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned c = b[j] < 0 ? 0 : (unsigned)(w[j] >> 32) + (old[j] + (unsigned)w[j] < old[j] ? 1u : 0u);
        asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %1, 0;\n @p red.shared.add.u32 [%0], %1;\n}\n" ::"r"(hi + 4 * b[j]), "r"(c)
                     : "memory");
        if (count)
            asm volatile("{\n .reg .pred p;\n setp.ge.s32 p, %1, 0;\n @p red.shared.add.u32 [%0], 1;\n}\n" ::"r"(cnt + 4 * b[j]),
                         "r"(b[j])
                         : "memory");
    }
}
PYXIS_DEVINL u64 wide(const Histogram &h, int b) { return ((u64)h.hi[b] << 32) | h.lo[b]; }

struct Row {
    float top;            // largest logit
    float bin_scale;      // bins per unit of logit
    double steps;         // 2^(1/256) steps per unit of logit
    int shift, last_bin;
    const double *table;
    // the bin of x, or -1 if its weight is 0
    PYXIS_DEVINL int bin(float x) const {
        const float f = (top - x) * bin_scale;
        const int b = f < (float)(last_bin + 1) ? (int)f : -1;  // NaN and infinite distances: -1
        return x == top ? 0 : b;
    }
    // a bound: values below it are in later bins than b (the bins' own rounding is far within 1e-3 bins)
    PYXIS_DEVINL float floor_of(int b) const {
        return b >= last_bin || isinf(top) ? -INFINITY : top - (float)(b + 1) * (1.001f / bin_scale) - fabsf(top) * 1e-6f;
    }
    // exp((x - top) / temperature) 2^shift, rounded: 2^(shift - k / 256) from the table, times exp of
    // the rest d ln 2 / 256, |d| <= 1/2, by its Taylor polynomial (of degree four: off by 2^-54 of the weight)
    PYXIS_DEVINL u64 weight(float x) const {
        constexpr double c = 0.69314718055994530942 / kTable;
        constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: rounds to a whole number
        const double u = ((double)top - (double)x) * steps;
        const double m = u + kRound;
        const int k = __double2loint(m);  // valid bins: u < 2^14
        const double d = (m - kRound) - u;
        double e = fma(d, fma(d, fma(d, fma(d, c * c * c * c / 24.0, c * c * c / 6.0), c * c / 2.0), c), 1.0) * table[k & (kTable - 1)];
        e = __hiloint2double(__double2hiint(e) - ((k >> 8) << 20), __double2loint(e));  // 2^-(k / 256)
        // to a whole number in the low bits
        const u64 w = (u64)__double_as_longlong(e + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
        return x == top ? 1ull << shift : w;
    }
};

// Inclusive sums over the CTA's threads.
PYXIS_DEVINL void block_scan(u64 &mass, unsigned &cnt, Shared &s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 m = __shfl_up_sync(0xffffffffu, mass, o);
        const unsigned c = __shfl_up_sync(0xffffffffu, cnt, o);
        if (lane >= o) mass += m, cnt += c;
    }
    __syncthreads();
    if (lane == 31) s.scan[warp] = mass, s.scan_cnt[warp] = cnt;
    __syncthreads();
    for (int w = 0; w < warp; ++w) mass += s.scan[w], cnt += s.scan_cnt[w];
}
PYXIS_DEVINL u64 block_sum(u64 x, Shared &s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.scan[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < kWarps; ++w) x += s.scan[w];
    return x;
}
// Smallest and largest of the threads' keys.
PYXIS_DEVINL void block_range(u64 &lo, u64 &hi, Shared &s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 x = __shfl_xor_sync(0xffffffffu, lo, o), y = __shfl_xor_sync(0xffffffffu, hi, o);
        lo = x < lo ? x : lo;
        hi = y > hi ? y : hi;
    }
    __shared__ u64 lows[kWarps], highs[kWarps];
    __syncthreads();
    if ((threadIdx.x & 31) == 0) lows[threadIdx.x >> 5] = lo, highs[threadIdx.x >> 5] = hi;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) {
        lo = lows[w] < lo ? lows[w] : lo;
        hi = highs[w] > hi ? highs[w] : hi;
    }
}

PYXIS_DEVINL void clear(Histogram &h) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) h.lo[b] = h.hi[b] = h.cnt[b] = 0;
}
PYXIS_DEVINL int shift_for(u64 lo, u64 hi) {  // (hi - key) >> shift is a bin
    static_assert(kBins == 1 << 10, "");
    const int bits = 64 - __clzll((long long)(hi - lo));
    return bits > 10 ? bits - 10 : 0;
}

// The bin of a key-range histogram where the running count (by_count) or weight passes t becomes
// the range; *out is written by one thread (after a barrier: in may be *out).
PYXIS_DEVINL void pick_bin(const Histogram &h, const Range &in, int sh, bool by_count, u64 t, Range *out, Shared &s) {
    u64 m = 0;
    unsigned c = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) m += wide(h, threadIdx.x * kPerThread + j), c += h.cnt[threadIdx.x * kPerThread + j];
    const Range r = in;
    u64 em = m;
    unsigned ec = c;
    block_scan(em, ec, s);
    em += r.ex_mass - m, ec += r.ex_count - c;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int b = threadIdx.x * kPerThread + j;
        const u64 before = by_count ? ec : em, size = by_count ? h.cnt[b] : wide(h, b);
        if (t >= before && t - before < size) {
            const u64 hi = r.hi - ((u64)b << sh), width = (1ull << sh) - 1;
            *out = Range{hi - r.lo > width ? hi - width : r.lo, hi, em, ec, h.cnt[b]};
        }
        em += wide(h, b), ec += h.cnt[b];
    }
    __syncthreads();
}

// Ranks n <= kRank keys of s.few against one another (weights in s.few_w), kRankLanes threads to a key:
// the first of them, few_owner(n), adds the weight and the number of those before it.
constexpr int kRankLanes = kThreads / kRank;
static_assert(kRankLanes == 4, "");
PYXIS_DEVINL unsigned few_index() { return threadIdx.x / kRankLanes; }
PYXIS_DEVINL bool few_owner(unsigned n) { return threadIdx.x % kRankLanes == 0 && few_index() < n; }
PYXIS_DEVINL void rank_few(const Shared &s, unsigned n, u64 &before, unsigned &rank) {
    u64 m = 0;
    unsigned c = 0;
    if (few_index() < n) {
        const u64 k = s.few[few_index()];
        for (unsigned i = threadIdx.x % kRankLanes; i < n; i += kRankLanes)
            if (s.few[i] > k) m += s.few_w[i], ++c;
    }
#pragma unroll
    for (int o = 1; o < kRankLanes; o <<= 1) {
        m += __shfl_xor_sync(0xffffffffu, m, o);
        c += __shfl_xor_sync(0xffffffffu, c, o);
    }
    before += m, rank += c;
}

// Leader: among the candidates, whose first follows ex_mass and ex_count, the element where the
// running count or weight passes t: its weight, its key and the running weight with it.
PYXIS_DEVINL void locate(Shared &s, const Row &r, unsigned n, u64 ex_mass, unsigned ex_count, bool by_count, u64 t) {
    u64 lo = ~0ull, hi = 0;
    for (unsigned i = threadIdx.x; i < n; i += kThreads) {
        const u64 k = s.cand[i];
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
    }
    block_range(lo, hi, s);
    if (threadIdx.x == 0) s.narrow = Range{lo, hi, ex_mass, ex_count, n};
    __syncthreads();
    while (s.narrow.count > kRank) {
        lo = s.narrow.lo, hi = s.narrow.hi;
        const int sh = shift_for(lo, hi);
        clear(s.row);
        __syncthreads();
        for (unsigned i = threadIdx.x; i < n; i += kThreads) {
            const u64 k = s.cand[i];
            if (k < lo || k > hi) continue;
            const int b = (int)((hi - k) >> sh);
            add_wide(&s.row.lo[b], &s.row.hi[b], r.weight(value_of(k)));
            atomicAdd(&s.row.cnt[b], 1u);
        }
        __syncthreads();
        pick_bin(s.row, s.narrow, sh, by_count, t, &s.narrow, s);
    }
    if (threadIdx.x == 0) s.nfew = 0;
    __syncthreads();
    lo = s.narrow.lo, hi = s.narrow.hi;
    for (unsigned i = threadIdx.x; i < n; i += kThreads) {
        const u64 k = s.cand[i];
        if (k < lo || k > hi) continue;
        const unsigned at = atomicAdd(&s.nfew, 1u);
        s.few[at] = k;
        s.few_w[at] = r.weight(value_of(k));
    }
    __syncthreads();
    u64 before = s.narrow.ex_mass;
    unsigned rank = s.narrow.ex_count;
    rank_few(s, s.nfew, before, rank);
    if (few_owner(s.nfew)) {
        const u64 w = s.few_w[few_index()];
        if (by_count ? rank == t : t >= before && t - before < w) {
            s.found_mass = before + w;
            s.found_w = w;
            s.found_key = s.few[few_index()];
        }
    }
    __syncthreads();
}

// What the filters and the draw ask for, the same for every CTA of a row.
struct Params {
    int top_k;
    double top_p, min_p, u;
    PYXIS_DEVINL u64 top_p_target(u64 prefix) const {  // the first element with a running weight >= p prefix
        const double goal = ceil(top_p * (double)prefix);
        return goal > 1.0 ? (u64)goal - 1 : 0;
    }
    PYXIS_DEVINL u64 draw_target(u64 kept) const {
        const double v = u > 0.0 ? u : 0.0;  // NaN: 0
        const u64 t = v < 1.0 ? (u64)(v * (double)kept) : kept;
        return t < kept ? t : kept - 1;
    }
};

PYXIS_DEVINL void write_result(const SampleArgs &a, size_t row, const Shared &s, u64 kept) {
    if (threadIdx.x != 0) return;
    a.idx[row] = (int32_t)(0xFFFFFFFFu - (unsigned)(s.found_key & 0xFFFFFFFFu));
    if (a.prob) a.prob[row] = (float)((double)s.found_w / (double)kept);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared &s = *reinterpret_cast<Shared *>(smem);
    T *vals = reinterpret_cast<T *>(smem + (sizeof(Shared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), ranks = cluster.num_blocks();
    Shared &leader = *cluster.map_shared_rank(&s, 0);
    const size_t row = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // first half of the barrier that tells every CTA of the cluster that the others have started (their
    // shared memory may be written): waited on before the maxima are sent
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

    if (tid == 0) {
        s.temperature = a.temperature ? (double)a.temperature[row] : a.temperature_all;
        s.top_k = a.top_k ? a.top_k[row] : a.top_k_all;
        s.top_p = a.top_p ? (double)a.top_p[row] : a.top_p_all;
        s.min_p = a.min_p ? (double)a.min_p[row] : a.min_p_all;
        s.u = (double)a.u[row];
    }
    // ---- this CTA's segment of the row, and the threads' maxima
    const size_t per = (a.n + ranks - 1) / ranks;
    const size_t beg = rank * per < a.n ? rank * per : a.n, end = beg + per < a.n ? beg + per : a.n;
    const T *src = reinterpret_cast<const T *>(a.logits) + row * a.ld + beg;
    const unsigned len = (unsigned)(end - beg), held = len < a.cap ? len : a.cap;
    constexpr unsigned V = 16 / sizeof(T);
    // shared memory holds the segment at the 16-byte phase it has in global memory
    const unsigned phase = (unsigned)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    T *own = vals + phase;

    // (elements before and after it in its 16-byte vectors are -inf there)
    float mine = -INFINITY;
    const unsigned head = min(held, (V - phase) % V), vecs = (held - head) / V, all_vecs = (phase + held + V - 1) / V;
    {
        const uint4 *g = reinterpret_cast<const uint4 *>(src + head);
        uint4 *d = reinterpret_cast<uint4 *>(own + head);
#pragma unroll 8
        for (unsigned i = tid; i < vecs; i += kThreads) {
            const uint4 x = __ldg(g + i);
            d[i] = x;
            const T *e = reinterpret_cast<const T *>(&x);
#pragma unroll
            for (unsigned j = 0; j < V; ++j) mine = fmaxf(mine, widen(e[j]));
        }
    }
    const T none = lowest<T>();
    if (tid < (int)phase) vals[tid] = none;
    if (phase + held + tid < all_vecs * V) own[held + tid] = none;
    if (tid < (int)head) own[tid] = src[tid], mine = fmaxf(mine, widen(src[tid]));
    for (unsigned i = head + vecs * V + tid; i < held; i += kThreads) own[i] = src[i], mine = fmaxf(mine, widen(src[i]));
    for (unsigned i = held + tid; i < len; i += kThreads) mine = fmaxf(mine, widen(src[i]));
    // fn(values, index of the first, how many) for every element: four at a time from shared memory,
    // then one by one what it does not hold
    auto scan = [&](auto &&fn) {
        constexpr unsigned H = V / 4;
        for (unsigned i = tid; i < all_vecs * H; i += kThreads) {
            float x[4];
            if constexpr (sizeof(T) == 4) {
                const float4 v = reinterpret_cast<const float4 *>(vals)[i];
                x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
            } else {
                const uint2 v = reinterpret_cast<const uint2 *>(vals)[i];
                x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xFFFF0000u);
                x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xFFFF0000u);
            }
            fn(x, (int)(i * 4) - (int)phase);
        }
        for (unsigned i = held + tid; i < len; i += kThreads) {
            const float x[4] = {widen(src[i]), -INFINITY, -INFINITY, -INFINITY};
            fn(x, (int)i);
        }
    };
    clear(s.row);
    if (tid == 0) s.ncand = 0;
    if (tid < kTable) s.table[tid] = exp2(a.shift - (double)tid / kTable);
    float top = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float *wtop = reinterpret_cast<float *>(s.scan);
    if (lane == 0) wtop[warp] = top;
    __syncthreads();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid < (int)ranks) {
        float t = wtop[0];
        for (int w = 1; w < kWarps; ++w) t = fmaxf(t, wtop[w]);
        cluster.map_shared_rank(&s, tid)->rank_top[rank] = t;
    }
    cluster.sync();
    Row r;
    r.top = s.rank_top[0];
    for (unsigned i = 1; i < ranks; ++i) r.top = fmaxf(r.top, s.rank_top[i]);
    if (!(r.top > -INFINITY)) {  // the same for the whole cluster
        if (rank == 0 && tid == 0) {
            a.idx[row] = -1;
            if (a.prob) a.prob[row] = 0.f;
        }
        return;
    }
    const double temperature = s.temperature;
    if (!(temperature > 0.0)) {  // greedy: the first maximum
        u64 best = 0, least = ~0ull;
        scan([&](const float (&x)[4], int i) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (x[j] == r.top) {
                    const u64 k = key_of(r.top, (unsigned)(beg + i + j));
                    best = k > best ? k : best;
                }
        });
        block_range(least, best, s);
        if (tid == 0) leader.rank_max[rank] = best;
        cluster.sync();
        if (rank == 0 && tid == 0) {
            for (unsigned i = 0; i < ranks; ++i) best = s.rank_max[i] > best ? s.rank_max[i] : best;
            a.idx[row] = (int32_t)(0xFFFFFFFFu - (unsigned)(best & 0xFFFFFFFFu));
            if (a.prob) a.prob[row] = 1.0f;
        }
        return;
    }
    r.bin_scale = (float)(kBinsPerNat / temperature);
    r.steps = kTable * 1.44269504088896340736 / temperature;
    r.shift = a.shift;
    r.last_bin = a.last_bin;
    r.table = s.table;
    Params q;
    q.top_k = s.top_k;
    q.top_p = s.top_p;
    q.min_p = s.min_p;
    q.u = s.u;
    // weights that min_p keeps: w >= min_p 2^shift
    const u64 least = q.min_p > 0.0 ? (u64)ceil(fmin(q.min_p, 1.0) * (double)(1ull << r.shift)) : 0;

    // every element of bins first .. last of key lo .. hi into the leader's candidates
    auto gather = [&](int first, int last, u64 lo, u64 hi) {
        const float floor = r.floor_of(last);
        scan([&](const float (&x)[4], int i) {
            if (!(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= floor)) return;  // most are far below
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = r.bin(x[j]);
                if (b < first || b > last) continue;
                const u64 k = key_of(x[j], (unsigned)(beg + i + j));
                if (k < lo || k > hi) continue;
                const unsigned at = atomicAdd(&leader.ncand, 1u);
                if (at < kCand) leader.cand[at] = k;
            }
        });
    };

    // ---- a set that settles everything: the whole row, or what top_k can keep
    const bool small = a.n <= kCand;
    if (small || (q.top_k > 0 && q.top_k <= kMaxTopK)) {
        if (!small) {
            const int b = r.bin(mine);
            if (b >= 0) atomicAdd(&leader.row.cnt[b], 1u);
            cluster.sync();
        }
        if (rank == 0) {
            if (tid == 0) s.bin[3] = r.last_bin;
            __syncthreads();
            if (!small) {
                u64 unused = 0;
                unsigned c = 0;
#pragma unroll
                for (int j = 0; j < kPerThread; ++j) c += s.row.cnt[tid * kPerThread + j];
                unsigned incl = c;
                block_scan(unused, incl, s);
                unsigned before = incl - c;
#pragma unroll
                for (int j = 0; j < kPerThread; ++j) {
                    const unsigned x = s.row.cnt[tid * kPerThread + j];
                    if (before < (unsigned)q.top_k && before + x >= (unsigned)q.top_k) s.bin[3] = tid * kPerThread + j;
                    before += x;
                }
            }
        }
        cluster.sync();
        gather(0, leader.bin[3], 0, ~0ull);
        cluster.sync();
        const unsigned n = leader.ncand;
        if (n <= kCand) {
            if (rank != 0) {
                cluster.sync();  // the leader's count has been read
                return;
            }
            cluster.sync();
            if (n <= kRank) {  // one ranking answers all three
                u64 w = 0, before = 0;
                unsigned at = 0;
                if (tid < (int)n) s.few[tid] = s.cand[tid], s.few_w[tid] = r.weight(value_of(s.cand[tid]));
                __syncthreads();
                rank_few(s, n, before, at);
                const bool in = few_owner(n) && (q.top_k <= 0 || at < (unsigned)q.top_k);  // top-k keeps it
                if (in) w = s.few_w[few_index()];
                const u64 total = block_sum(in ? w : 0, s);
                u64 kept = total;
                if (q.min_p > 0.0) {
                    const u64 above = block_sum(in && w >= least ? w : 0, s);
                    kept = above < kept ? above : kept;
                }
                if (q.top_p < 1.0) {
                    const u64 t = q.top_p_target(total);
                    if (in && t >= before && t - before < w) s.found_mass = before + w;
                    __syncthreads();
                    kept = s.found_mass < kept ? s.found_mass : kept;
                }
                const u64 t = q.draw_target(kept);
                if (in && t >= before && t - before < w) {
                    s.found_w = w;
                    s.found_key = s.few[few_index()];
                }
                __syncthreads();
                write_result(a, row, s, kept);
                return;
            }
            u64 total = 0, above = 0;
            for (unsigned i = tid; i < n; i += kThreads) {
                const u64 w = r.weight(value_of(s.cand[i]));
                total += w;
                if (w >= least) above += w;
            }
            total = block_sum(total, s);
            if (q.top_k > 0 && (unsigned)q.top_k < n) {
                locate(s, r, n, 0, 0, true, (u64)q.top_k - 1);
                total = s.found_mass;
                __syncthreads();
            }
            u64 kept = total;
            if (q.min_p > 0.0) {
                above = block_sum(above, s);
                kept = above < kept ? above : kept;
            }
            if (q.top_p < 1.0) {
                locate(s, r, n, 0, 0, false, q.top_p_target(total));
                kept = s.found_mass < kept ? s.found_mass : kept;
                __syncthreads();
            }
            locate(s, r, n, 0, 0, false, q.draw_target(kept));
            write_result(a, row, s, kept);
            return;
        }
        cluster.sync();  // everyone has read the count
        clear(s.row);
        cluster.sync();
    }

    // ---- the histogram of the row, in the leader
    {
        u64 above = 0;  // weight of the elements that min_p keeps
        const bool count = q.top_k > 0;
        scan([&](const float (&x)[4], int) {
            int b[4];
            u64 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = r.bin(x[j]), w[j] = r.weight(x[j]);
            add_wide4(s.row, b, w, count);
#pragma unroll
            for (int j = 0; j < 4; ++j) above += b[j] >= 0 && w[j] >= least ? w[j] : 0;
        });
        above = block_sum(above, s);
        if (tid == 0) leader.rank_mass[rank] = above;
        if (rank != 0)
            for (int b = tid; b < kBins; b += kThreads) {
                const u64 w = wide(s.row, b);
                if (w) add_wide(&leader.row.lo[b], &leader.row.hi[b], w);
                if (s.row.cnt[b]) atomicAdd(&leader.row.cnt[b], s.row.cnt[b]);
            }
    }
    cluster.sync();

    // ---- leader: running sums over the bins (thread t holds bins kPerThread t ..)
    u64 bin_mass[kPerThread], ex_mass = 0, total = 0, kept = 0;
    unsigned bin_cnt[kPerThread], ex_cnt = 0, total_cnt = 0;
    if (rank == 0) {
        u64 m = 0;
        unsigned c = 0;
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            bin_mass[j] = wide(s.row, tid * kPerThread + j);
            bin_cnt[j] = s.row.cnt[tid * kPerThread + j];
            m += bin_mass[j];
            c += bin_cnt[j];
        }
        ex_mass = m, ex_cnt = c;
        block_scan(ex_mass, ex_cnt, s);
        if (tid == kThreads - 1) s.found_mass = ex_mass, s.nfew = ex_cnt;
        __syncthreads();
        total = s.found_mass;
        total_cnt = s.nfew;
        ex_mass -= m, ex_cnt -= c;
        kept = total;
        if (q.min_p > 0.0) {
            u64 above = 0;
            for (unsigned i = 0; i < ranks; ++i) above += s.rank_mass[i];
            kept = above < kept ? above : kept;
        }
        __syncthreads();
    }
    u64 prefix = total;  // weight of the top-k prefix
    // stage 0: top-k, 1: top-p, 2: the draw.  Each locates the first element whose running count
    // (stage 0) or weight exceeds t.
    for (int stage = 0; stage < 3; ++stage) {
        if (stage == 0 && q.top_k <= 0) continue;
        if (stage == 1 && !(q.top_p < 1.0)) continue;
        u64 t = 0;
        if (rank == 0) {
            t = stage == 0 ? (u64)q.top_k - 1 : stage == 1 ? q.top_p_target(prefix) : q.draw_target(kept);
            if (tid == 0) s.bin[stage] = -1, s.ncand = 0;
            __syncthreads();
            u64 m = ex_mass;
            unsigned c = ex_cnt;
#pragma unroll
            for (int j = 0; j < kPerThread; ++j) {
                const u64 before = stage == 0 ? c : m, size = stage == 0 ? bin_cnt[j] : bin_mass[j];
                if (t >= before && t - before < size) {
                    s.bin[stage] = tid * kPerThread + j;
                    s.ctl[stage] = Range{0, ~0ull, m, c, bin_cnt[j]};
                }
                m += bin_mass[j], c += bin_cnt[j];
            }
        }
        cluster.sync();
        const int bin = leader.bin[stage];
        if (bin < 0) continue;  // top-k keeps the whole row
        gather(bin, bin, 0, ~0ull);
        cluster.sync();
        unsigned count = leader.ncand;
        if (count > kCand) {
            // the bin's range of keys; then each round leaves 1 / kBins of it, down to single keys
            u64 lo = ~0ull, hi = 0;
            scan([&](const float (&x)[4], int i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (r.bin(x[j]) != bin) continue;
                    const u64 k = key_of(x[j], (unsigned)(beg + i + j));
                    lo = k < lo ? k : lo;
                    hi = k > hi ? k : hi;
                }
            });
            block_range(lo, hi, s);
            if (tid == 0) leader.rank_min[rank] = lo, leader.rank_max[rank] = hi;
            cluster.sync();
            lo = ~0ull, hi = 0;
            for (unsigned i = 0; i < ranks; ++i) {
                lo = leader.rank_min[i] < lo ? leader.rank_min[i] : lo;
                hi = leader.rank_max[i] > hi ? leader.rank_max[i] : hi;
            }
            while (count > kCand) {
                const int sh = shift_for(lo, hi);
                clear(s.sub);
                cluster.sync();
                scan([&](const float (&x)[4], int i) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (r.bin(x[j]) != bin) continue;
                        const u64 k = key_of(x[j], (unsigned)(beg + i + j));
                        if (k < lo || k > hi) continue;
                        const unsigned b = (unsigned)((hi - k) >> sh);
                        add_wide(&s.sub.lo[b], &s.sub.hi[b], r.weight(x[j]));
                        atomicAdd(&s.sub.cnt[b], 1u);
                    }
                });
                __syncthreads();
                if (rank != 0)
                    for (int b = tid; b < kBins; b += kThreads)
                        if (s.sub.cnt[b]) {
                            add_wide(&leader.sub.lo[b], &leader.sub.hi[b], wide(s.sub, b));
                            atomicAdd(&leader.sub.cnt[b], s.sub.cnt[b]);
                        }
                cluster.sync();
                if (rank == 0) {
                    if (tid == 0) s.ctl[stage].lo = lo, s.ctl[stage].hi = hi, s.ncand = 0;
                    __syncthreads();
                    pick_bin(s.sub, s.ctl[stage], sh, stage == 0, t, &s.ctl[stage], s);
                }
                cluster.sync();
                lo = leader.ctl[stage].lo, hi = leader.ctl[stage].hi, count = leader.ctl[stage].count;
            }
            gather(bin, bin, lo, hi);
            cluster.sync();
        }
        if (rank == 0) {
            locate(s, r, count, s.ctl[stage].ex_mass, s.ctl[stage].ex_count, stage == 0, t);
            const u64 cum = s.found_mass;
            if (stage == 0) prefix = cum;
            if (stage < 2)
                kept = cum < kept ? cum : kept;
            else
                write_result(a, row, s, kept);
            __syncthreads();
        }
    }
    cluster.sync();  // no CTA leaves while another may still read the leader's
}

template <typename T>
cudaError_t run_sample(SampleArgs &a, size_t M, int num_sms, cudaStream_t st) {
    auto kern = sample_kernel<T>;
    static std::atomic<uint64_t> done{0};
    constexpr size_t fixed = (sizeof(Shared) + 15) / 16 * 16, most = 200 * 1024;
    constexpr size_t pad = 2 * 16 / sizeof(T);  // a segment's phase, and its last vector's end
    cudaError_t e = once_per_device(done, [&] {
        const cudaError_t x = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        return x != cudaSuccess ? x : cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (e != cudaSuccess) return e;
    // one CTA per 4096 tokens, up to 16 while the rows leave SMs idle, else up to 8 (one row of 151936
    // f32: 31 us with 8, 25 us with 16); fewer where the rows fill the GPU (two CTAs an SM) without
    // them and two such segments still fit an SM
    int ranks = 1;
    const int widest = M * kMaxCluster <= (size_t)num_sms ? kMaxCluster : 8;
    while (ranks < widest && (size_t)ranks * 4096 < a.n) ranks *= 2;
    while (ranks > 1 && M * ranks > (size_t)num_sms * 2 && (a.n / (ranks / 2)) * sizeof(T) + fixed < 112 * 1024) ranks /= 2;
    for (;; ranks = 8) {
        const size_t per = (a.n + ranks - 1) / ranks, room = (most - fixed) / sizeof(T) - pad;
        a.cap = (unsigned)std::min(per, room);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ranks, (unsigned)M);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = fixed + (a.cap + pad) * sizeof(T);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ranks;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (ranks > 8) {  // not every device places 16 CTAs side by side
            int clusters = 0;
            e = cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg);
            if (e != cudaSuccess || clusters < 1) {
                cudaGetLastError();
                continue;
            }
        }
        return cudaLaunchKernelEx(&cfg, kern, a);
    }
}

}  // namespace

cudaError_t launch_sample(const void *logits, int dtype, size_t M, size_t n, size_t ld, const float *uniforms,
                          const pyxis_sample_params &p, int32_t *idx, float *prob, int num_sms, cudaStream_t st) {
    SampleArgs a;
    a.logits = logits;
    a.n = n;
    a.ld = ld;
    a.u = uniforms;
    a.temperature = p.temperature;
    a.top_p = p.top_p;
    a.min_p = p.min_p;
    a.top_k = p.top_k;
    a.temperature_all = p.temperature_all;
    a.top_p_all = p.top_p_all;
    a.min_p_all = p.min_p_all;
    a.top_k_all = p.top_k_all;
    a.idx = idx;
    a.prob = prob;
    int bits = 0;
    while ((1ull << bits) < n) ++bits;
    a.shift = bits > 18 ? 62 - bits : 44;
    // a weight below 2^-(shift + 1) rounds to 0: beyond (shift + 1) ln 2 nats, and a bin to spare
    a.last_bin = (int)((a.shift + 1) * 0.6931471805599453 * kBinsPerNat) + 1;
    return dtype == PYXIS_DTYPE_F32 ? run_sample<float>(a, M, num_sms, st) : run_sample<__nv_bfloat16>(a, M, num_sms, st);
}

}  // namespace pyxis
