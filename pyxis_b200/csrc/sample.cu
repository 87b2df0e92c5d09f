// sample.cu -- temperature, top-k, top-p and min-p sampling of one token per row from given uniform
// numbers (src/sampler.rs:23-110 on the device; definition in include/pyxis_serve.h).
//
// Every filter keeps a prefix of the order "largest logit first, equal ones by index", so the
// prefixes are nested and the kept weight is the smallest of the prefixes' weights.  With that
// total Z the drawn token is the first one in the order whose running sum of weights exceeds u Z:
// nothing is sorted and no mask is kept; three times at most one element of the order is located
// -- by count (the k-th), by weight (p Z_k) and by weight (u Z).
//
// A cluster of CTAs holds a row in shared memory (one pass over HBM) and histograms it by
// (max - x) / temperature in bins of 1/64 nat, weights and counts.  The leader CTA finds the bin
// that holds the element sought, the cluster gathers the bin's elements into the leader's shared
// memory, and the leader sorts and scans them.  A bin of more elements than that holds (flat or
// heavily tied rows) is first cut down by histograms over the 64-bit (value, index) key.
//
// Weights are exp() in f64 rounded to 2^-44 (less for rows of over 2^18 tokens, so that a row's sum
// stays below 2^63): integer sums are exact in any order, so neither the atomics' order nor the
// cluster's size changes a token, and the sums are far finer than the spacing of uniform numbers.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <atomic>

#include "common.cuh"
#include "serve.h"

namespace pyxis {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;        // 1/64 nat each: 32 nats, past which a weight rounds to 0
constexpr int kCand = 2048;        // elements of a bin that the leader sorts
constexpr int kMaxCluster = 8;
constexpr int kPerThread = kBins / kThreads;
constexpr float kBinsPerNat = 64.0f;

struct SampleArgs {
    const void *logits;
    size_t n, ld;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int32_t top_k_all;
    int32_t *idx;
    float *prob;
    int shift;       // weights are multiples of 2^-shift
    int last_bin;    // elements of later bins have weight 0
    unsigned cap;    // elements of a segment that shared memory holds
};

// What the leader tells the cluster about the element being located.
struct Control {
    int skip;                        // the prefix is the whole row
    int bin;                         // first-level bin
    unsigned count;                  // elements in [lo, hi] of the bin
    unsigned long long lo, hi;       // key range
    unsigned long long ex_mass;      // weight and count before the range
    unsigned ex_count;
};

struct Shared {
    union {
        unsigned long long cand[kCand];
        struct {
            unsigned lo[kBins], hi[kBins], cnt[kBins];
        } sub;  // histogram of a key range
    };
    unsigned lo[kBins], hi[kBins], cnt[kBins];  // the row's histogram (leader): weight as two words, count
    unsigned long long scan[kWarps];
    unsigned scan_cnt[kWarps];
    unsigned long long rank_min[kMaxCluster], rank_max[kMaxCluster], rank_mass[kMaxCluster];
    float rank_top[kMaxCluster];
    Control ctl[3];
    unsigned ncand;
    unsigned long long found_mass, found_w, found_key;
    int which;
};

PYXIS_DEVINL float widen(float x) { return x; }
PYXIS_DEVINL float widen(__nv_bfloat16 x) { return __bfloat162float(x); }

// Order-preserving key of a finite or infinite value and its index: larger values first, then
// smaller indexes; -0 ties with +0.
PYXIS_DEVINL unsigned long long key_of(float v, unsigned idx) {
    if (v == 0.0f) v = 0.0f;
    const unsigned u = __float_as_uint(v);
    const unsigned ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)ord << 32) | (0xFFFFFFFFu - idx);
}
PYXIS_DEVINL float value_of(unsigned long long key) {
    const unsigned ord = (unsigned)(key >> 32);
    return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7FFFFFFFu) : ~ord);
}

// 64-bit add into two 32-bit words of (this or another CTA's) shared memory: the carry goes with
// the value the low word had, so the pair is exact once all adds are done.
PYXIS_DEVINL void add_wide(unsigned *lo, unsigned *hi, unsigned long long w) {
    const unsigned wl = (unsigned)w;
    const unsigned old = atomicAdd(lo, wl);
    const unsigned c = (unsigned)(w >> 32) + (old + wl < old ? 1u : 0u);
    if (c) atomicAdd(hi, c);
}

struct Row {
    float top;        // largest logit
    float bin_scale;  // bins per unit of logit
    double inv_t;
    bool greedy;
    int shift, last_bin;
    // the bin of x, or -1 if its weight is 0
    PYXIS_DEVINL int bin(float x) const {
        if (x == top) return 0;
        if (greedy) return -1;
        const float f = (top - x) * bin_scale;
        return f < (float)(last_bin + 1) ? (int)f : -1;  // NaN and infinite distances: -1
    }
    PYXIS_DEVINL unsigned long long weight(float x) const {
        if (x == top) return 1ull << shift;
        const double e = exp(-((double)top - (double)x) * inv_t);
        return (unsigned long long)__double2ll_rn(e * (double)(1ull << shift));
    }
};

// Inclusive sums over the CTA's threads.
PYXIS_DEVINL void block_scan(unsigned long long &mass, unsigned &cnt, Shared &s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long m = __shfl_up_sync(0xffffffffu, mass, o);
        const unsigned c = __shfl_up_sync(0xffffffffu, cnt, o);
        if (lane >= o) mass += m, cnt += c;
    }
    __syncthreads();
    if (lane == 31) s.scan[warp] = mass, s.scan_cnt[warp] = cnt;
    __syncthreads();
    for (int w = 0; w < warp; ++w) mass += s.scan[w], cnt += s.scan_cnt[w];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared &s = *reinterpret_cast<Shared *>(smem);
    T *vals = reinterpret_cast<T *>(smem + (sizeof(Shared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), ranks = cluster.num_blocks();
    Shared &leader = *cluster.map_shared_rank(&s, 0);
    const size_t row = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    // this CTA's segment of the row
    const size_t per = (a.n + ranks - 1) / ranks;
    const size_t beg = rank * per < a.n ? rank * per : a.n, end = beg + per < a.n ? beg + per : a.n;
    const T *src = reinterpret_cast<const T *>(a.logits) + row * a.ld + beg;
    const unsigned len = (unsigned)(end - beg), held = len < a.cap ? len : a.cap;
    constexpr unsigned V = 16 / sizeof(T);
    // shared memory holds the segment at the 16-byte phase it has in global memory
    const unsigned phase = (unsigned)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    T *own = vals + phase;
    auto value = [&](unsigned i) -> float { return widen(i < held ? own[i] : src[i]); };

    for (int b = tid; b < kBins; b += kThreads) s.lo[b] = s.hi[b] = s.cnt[b] = 0;
    if (tid == 0) s.ncand = 0;
    float top = -INFINITY;
    const unsigned head = min(held, (V - phase) % V), vecs = (held - head) / V;
    if (tid < head) own[tid] = src[tid], top = fmaxf(top, widen(src[tid]));
    for (unsigned i = head + vecs * V + tid; i < held; i += kThreads) own[i] = src[i], top = fmaxf(top, widen(src[i]));
    for (unsigned i = held + tid; i < len; i += kThreads) top = fmaxf(top, widen(src[i]));
    {
        const uint4 *g = reinterpret_cast<const uint4 *>(src + head);
        uint4 *d = reinterpret_cast<uint4 *>(own + head);
#pragma unroll 4
        for (unsigned i = tid; i < vecs; i += kThreads) {
            const uint4 x = __ldg(g + i);
            d[i] = x;
            const T *e = reinterpret_cast<const T *>(&x);
#pragma unroll
            for (unsigned j = 0; j < V; ++j) top = fmaxf(top, widen(e[j]));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float *wtop = reinterpret_cast<float *>(s.scan);
    if (lane == 0) wtop[warp] = top;
    __syncthreads();
    if (tid < (int)ranks) {
        float t = wtop[0];
        for (int w = 1; w < kWarps; ++w) t = fmaxf(t, wtop[w]);
        cluster.map_shared_rank(&s, tid)->rank_top[rank] = t;
    }
    cluster.sync();
    Row r;
    r.top = s.rank_top[0];
    for (unsigned i = 1; i < ranks; ++i) r.top = fmaxf(r.top, s.rank_top[i]);
    const float t32 = a.temperature ? a.temperature[row] : 0.f;
    const double temperature = a.temperature ? (double)t32 : a.temperature_all;
    r.greedy = !(temperature > 0.0);
    r.inv_t = r.greedy ? 0.0 : 1.0 / temperature;
    r.bin_scale = (float)(kBinsPerNat * r.inv_t);
    r.shift = a.shift;
    r.last_bin = a.last_bin;
    const int top_k = r.greedy ? 0 : a.top_k ? a.top_k[row] : a.top_k_all;
    const double top_p = r.greedy ? 1.0 : a.top_p ? (double)a.top_p[row] : a.top_p_all;
    const double min_p = r.greedy ? 0.0 : a.min_p ? (double)a.min_p[row] : a.min_p_all;
    if (!(r.top > -INFINITY)) {  // the same for the whole cluster
        if (rank == 0 && tid == 0) {
            a.idx[row] = -1;
            if (a.prob) a.prob[row] = 0.f;
        }
        return;
    }

    // ---- the histogram of the row, in the leader
    {
        const double least = fmin(min_p, 1.0) * (double)(1ull << r.shift);
        unsigned long long above = 0;  // weight of the elements that min_p keeps
        for (unsigned i = tid; i < len; i += kThreads) {
            const float x = value(i);
            const int b = r.bin(x);
            if (b < 0) continue;
            const unsigned long long w = r.weight(x);
            if ((double)w >= least) above += w;
            add_wide(&s.lo[b], &s.hi[b], w);
            atomicAdd(&s.cnt[b], 1u);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
        __syncthreads();
        if (lane == 0) s.scan[warp] = above;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kWarps; ++w) above += s.scan[w];
            leader.rank_mass[rank] = above;
        }
        if (rank != 0)
            for (int b = tid; b < kBins; b += kThreads)
                if (s.cnt[b]) {
                    add_wide(&leader.lo[b], &leader.hi[b], ((unsigned long long)s.hi[b] << 32) | s.lo[b]);
                    atomicAdd(&leader.cnt[b], s.cnt[b]);
                }
    }
    cluster.sync();

    // ---- leader: running sums over the bins (thread t holds bins kPerThread t ..)
    unsigned long long bin_mass[kPerThread], ex_mass = 0;
    unsigned bin_cnt[kPerThread], ex_cnt = 0;
    unsigned long long total = 0, kept = 0;
    unsigned total_cnt = 0;
    if (rank == 0) {
        unsigned long long m = 0;
        unsigned c = 0;
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            const int b = tid * kPerThread + j;
            bin_mass[j] = ((unsigned long long)s.hi[b] << 32) | s.lo[b];
            bin_cnt[j] = s.cnt[b];
            m += bin_mass[j];
            c += bin_cnt[j];
        }
        ex_mass = m, ex_cnt = c;
        block_scan(ex_mass, ex_cnt, s);
        if (tid == kThreads - 1) s.found_mass = ex_mass, s.which = (int)ex_cnt;
        __syncthreads();
        total = s.found_mass;
        total_cnt = (unsigned)s.which;
        ex_mass -= m, ex_cnt -= c;
        kept = total;
        if (min_p > 0.0) {
            unsigned long long above = 0;
            for (unsigned i = 0; i < ranks; ++i) above += s.rank_mass[i];
            kept = above < kept ? above : kept;
        }
        __syncthreads();
    }

    unsigned long long prefix = total;  // weight of the top-k prefix
    // stage 0: top-k, 1: top-p, 2: the draw.  Each locates the first element whose running count
    // (stage 0) or weight exceeds `t`.
    for (int stage = 0; stage < 3; ++stage) {
        if (stage == 0 && top_k <= 0) continue;
        if (stage == 1 && !(top_p < 1.0)) continue;
        Control &ctl = s.ctl[stage];
        unsigned long long t = 0;
        if (rank == 0) {
            bool skip = false;
            if (stage == 0) {
                t = (unsigned long long)top_k - 1;
                skip = t >= total_cnt;
            } else if (stage == 1) {
                const double goal = ceil(top_p * (double)prefix);
                t = goal > 1.0 ? (unsigned long long)goal - 1 : 0;
                skip = t >= total;
            } else {
                double u = (double)a.u[row];
                u = r.greedy || !(u > 0.0) ? 0.0 : u;
                t = u < 1.0 ? (unsigned long long)(u * (double)kept) : kept;
                if (t >= kept) t = kept - 1;
            }
            if (tid == 0) ctl.skip = skip, s.ncand = 0;
            if (!skip) {
                unsigned long long m = ex_mass;
                unsigned c = ex_cnt;
#pragma unroll
                for (int j = 0; j < kPerThread; ++j) {
                    const unsigned long long before = stage == 0 ? c : m, size = stage == 0 ? bin_cnt[j] : bin_mass[j];
                    if (t >= before && t - before < size) {
                        ctl.bin = tid * kPerThread + j;
                        ctl.count = bin_cnt[j];
                        ctl.lo = 0, ctl.hi = ~0ull;
                        ctl.ex_mass = m, ctl.ex_count = c;
                    }
                    m += bin_mass[j], c += bin_cnt[j];
                }
            }
        }
        cluster.sync();
        const Control &shared_ctl = leader.ctl[stage];
        if (shared_ctl.skip) continue;
        const int bin = shared_ctl.bin;
        unsigned count = shared_ctl.count;
        unsigned long long lo = 0, hi = ~0ull;
        if (count > kCand) {
            // the bin's range of keys
            unsigned long long kmin = ~0ull, kmax = 0;
            for (unsigned i = tid; i < len; i += kThreads) {
                const float x = value(i);
                if (r.bin(x) != bin) continue;
                const unsigned long long k = key_of(x, (unsigned)(beg + i));
                kmin = k < kmin ? k : kmin;
                kmax = k > kmax ? k : kmax;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long x = __shfl_xor_sync(0xffffffffu, kmin, o), y = __shfl_xor_sync(0xffffffffu, kmax, o);
                kmin = x < kmin ? x : kmin;
                kmax = y > kmax ? y : kmax;
            }
            __syncthreads();
            if (lane == 0) s.scan[warp] = kmin;
            __syncthreads();
            if (tid == 0) {
                for (int w = 0; w < kWarps; ++w) kmin = s.scan[w] < kmin ? s.scan[w] : kmin;
                leader.rank_min[rank] = kmin;
            }
            __syncthreads();
            if (lane == 0) s.scan[warp] = kmax;
            __syncthreads();
            if (tid == 0) {
                for (int w = 0; w < kWarps; ++w) kmax = s.scan[w] > kmax ? s.scan[w] : kmax;
                leader.rank_max[rank] = kmax;
            }
            cluster.sync();
            lo = ~0ull, hi = 0;
            for (unsigned i = 0; i < ranks; ++i) {
                lo = leader.rank_min[i] < lo ? leader.rank_min[i] : lo;
                hi = leader.rank_max[i] > hi ? leader.rank_max[i] : hi;
            }
            // each round leaves 1/kBins of the range, down to single keys
            while (count > kCand) {
                int sh = 0;
                while (((hi - lo) >> sh) >= kBins) ++sh;
                for (int b = tid; b < kBins; b += kThreads) s.sub.lo[b] = s.sub.hi[b] = s.sub.cnt[b] = 0;
                cluster.sync();
                for (unsigned i = tid; i < len; i += kThreads) {
                    const float x = value(i);
                    if (r.bin(x) != bin) continue;
                    const unsigned long long k = key_of(x, (unsigned)(beg + i));
                    if (k < lo || k > hi) continue;
                    const unsigned b = (unsigned)((hi - k) >> sh);
                    add_wide(&s.sub.lo[b], &s.sub.hi[b], r.weight(x));
                    atomicAdd(&s.sub.cnt[b], 1u);
                }
                __syncthreads();
                if (rank != 0)
                    for (int b = tid; b < kBins; b += kThreads)
                        if (s.sub.cnt[b]) {
                            add_wide(&leader.sub.lo[b], &leader.sub.hi[b],
                                     ((unsigned long long)s.sub.hi[b] << 32) | s.sub.lo[b]);
                            atomicAdd(&leader.sub.cnt[b], s.sub.cnt[b]);
                        }
                cluster.sync();
                if (rank == 0) {
                    unsigned long long m = 0;
                    unsigned c = 0;
#pragma unroll
                    for (int j = 0; j < kPerThread; ++j) {
                        const int b = tid * kPerThread + j;
                        m += ((unsigned long long)s.sub.hi[b] << 32) | s.sub.lo[b];
                        c += s.sub.cnt[b];
                    }
                    unsigned long long em = m;
                    unsigned ec = c;
                    block_scan(em, ec, s);
                    em += ctl.ex_mass - m, ec += ctl.ex_count - c;
                    __syncthreads();  // ctl is rewritten below
#pragma unroll
                    for (int j = 0; j < kPerThread; ++j) {
                        const int b = tid * kPerThread + j;
                        const unsigned long long bm = ((unsigned long long)s.sub.hi[b] << 32) | s.sub.lo[b];
                        const unsigned long long before = stage == 0 ? ec : em, size = stage == 0 ? s.sub.cnt[b] : bm;
                        if (t >= before && t - before < size) {
                            ctl.hi = hi - ((unsigned long long)b << sh);
                            const unsigned long long width = (1ull << sh) - 1;
                            ctl.lo = ctl.hi - lo > width ? ctl.hi - width : lo;
                            ctl.count = s.sub.cnt[b];
                            ctl.ex_mass = em, ctl.ex_count = ec;
                        }
                        em += bm, ec += s.sub.cnt[b];
                    }
                }
                cluster.sync();
                lo = shared_ctl.lo, hi = shared_ctl.hi, count = shared_ctl.count;
            }
        }
        // ---- gather the elements of the range into the leader, sort and scan them there
        for (unsigned i = tid; i < len; i += kThreads) {
            const float x = value(i);
            if (r.bin(x) != bin) continue;
            const unsigned long long k = key_of(x, (unsigned)(beg + i));
            if (k < lo || k > hi) continue;
            const unsigned at = atomicAdd(&leader.ncand, 1u);
            if (at < kCand) leader.cand[at] = k;
        }
        cluster.sync();
        if (rank == 0) {
            int size = 32;
            while (size < (int)count) size <<= 1;
            for (int i = (int)count + tid; i < size; i += kThreads) s.cand[i] = 0;
            __syncthreads();
            for (int k = 2; k <= size; k <<= 1)
                for (int j = k >> 1; j > 0; j >>= 1) {
                    for (int i = tid; i < size / 2; i += kThreads) {
                        const int x = 2 * i - (i & (j - 1)), y = x + j;  // j is a power of two
                        const unsigned long long p = s.cand[x], q = s.cand[y];
                        if ((p < q) == ((x & k) == 0)) s.cand[x] = q, s.cand[y] = p;
                    }
                    __syncthreads();
                }
            // running weights; thread t holds `each` consecutive candidates
            const int each = (size + kThreads - 1) / kThreads;
            unsigned long long w[kCand / kThreads], m = 0;
            for (int j = 0; j < each; ++j) {
                const int i = tid * each + j;
                w[j] = i < (int)count ? r.weight(value_of(s.cand[i])) : 0;
                m += w[j];
            }
            unsigned long long em = m;
            unsigned unused = 0;
            block_scan(em, unused, s);
            em += ctl.ex_mass - m;
            for (int j = 0; j < each; ++j) {
                const int i = tid * each + j;
                if (i < (int)count &&
                    (stage == 0 ? (unsigned long long)ctl.ex_count + i == t : t >= em && t - em < w[j])) {
                    s.found_mass = em + w[j];
                    s.found_w = w[j];
                    s.found_key = s.cand[i];
                }
                em += w[j];
            }
            __syncthreads();
            const unsigned long long cum = s.found_mass;
            if (stage == 0) prefix = cum;
            if (stage < 2) {
                if (cum < kept) kept = cum;
            } else if (tid == 0) {
                a.idx[row] = (int32_t)(0xFFFFFFFFu - (unsigned)(s.found_key & 0xFFFFFFFFu));
                if (a.prob) a.prob[row] = r.greedy ? 1.0f : (float)((double)s.found_w / (double)kept);
            }
            __syncthreads();
        }
    }
}

template <typename T>
cudaError_t run_sample(SampleArgs &a, size_t M, int ranks, cudaStream_t st) {
    auto kern = sample_kernel<T>;
    static std::atomic<uint64_t> done{0};
    constexpr size_t fixed = (sizeof(Shared) + 15) / 16 * 16, most = 200 * 1024;
    cudaError_t e = once_per_device(done, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    });
    if (e != cudaSuccess) return e;
    const size_t per = (a.n + ranks - 1) / ranks, room = (most - fixed) / sizeof(T) - 16 / sizeof(T);
    a.cap = (unsigned)(per < room ? per : room);
    const size_t bytes = fixed + (a.cap + 16 / sizeof(T)) * sizeof(T);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks, (unsigned)M);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace

cudaError_t launch_sample(const void *logits, int dtype, size_t M, size_t n, size_t ld, const float *uniforms,
                          const pyxis_sample_params &p, int32_t *idx, float *prob, cudaStream_t st) {
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
    // one CTA per 4096 tokens, up to eight
    int ranks = 1;
    while (ranks < kMaxCluster && (size_t)ranks * 4096 < n) ranks *= 2;
    return dtype == PYXIS_DTYPE_F32 ? run_sample<float>(a, M, ranks, st) : run_sample<__nv_bfloat16>(a, M, ranks, st);
}

}  // namespace pyxis
