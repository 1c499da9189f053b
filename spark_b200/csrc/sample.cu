// sample.cu -- sampling with temperature, top-k, top-p and min-p from given random
// numbers, and the same cut of logits for what samples later (a tree's verification).
//
// With M the largest logit, e(v) = exp((l(v) - M) / T).  In falling order of l, the
// lower index first, the first k entries stay; of those the shortest prefix whose sum
// of e is top_p of theirs or more; of those the entries with e >= min_p.  Each is a
// prefix of one order, so that all three are one cut (value, index).  The token is
// argmax e(v) / noise(v) over what stays: with exponential variates a sample.
//
// No sort.  The cut is found by counting: a histogram of the row over its distance
// from M (1024 bins over 32 T, below which e is under 2^-45), with counts and sums of
// e; a scan gives the bin that the cut is in; the few entries of that bin are compared
// with one another.  A bin of more than kList entries is divided again, by the
// integers in the order of the floats, then, if all are equal, by their index.  The
// sums decide borders, so that they have to be good, and may not depend on the order of
// atomics: e in 64 bits, added as multiples of 2^-44 in integers (409,600 entries of at
// most 1 fit 64 bits).
//
// One thread-block cluster of 8 CTAs (fewer where there are many rows) per row, each
// CTA a slice of the vocabulary that it keeps in shared memory, so that a row is read
// once; noise is read where an entry stays.  Bins are added and scans are exchanged
// through distributed shared memory; all CTAs take the same decisions.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace spark {
namespace tc {
int sm_count_cached(int dev);
}

namespace sm {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 1024;             // the last one: all that is further away
constexpr int kList = 512;              // entries that are compared with one another
constexpr int kRowBytes = 200 * 1024;   // of a CTA's slice
constexpr int kMaxVocab = kMaxCluster * kRowBytes / 4;
constexpr int kSmemSm = 228 * 1024;     // shared memory of an SM

struct Params {
    SparkSample a;
    int slice;   // vocabulary entries of a CTA, a multiple of 16
};

struct Note {
    float a, b;
    int i, pad;
};
// An entry of the list: its place in the falling order is (key, index), rising.
struct Entry {
    uint32_t key;
    int index;
};
// Where a cut was found: what lies before the bin, and in it.
struct Found {
    int bin, count, in;
    unsigned long long mass;
};
struct Cut {
    uint32_t key;               // what stays: smaller keys, of equal ones the indices up to this
    int index;
    unsigned long long mass;    // of all that stays
};
struct Shared {
    union {
        struct {
            unsigned count[kBins], low[kBins], high[kBins];  // of this CTA
        };
        struct {
            Entry list[kList];                               // (rank 0's, when the bins are added)
            unsigned long long list_mass[kList];
        };
    };
    unsigned long long mass[kBins];                          // of the row
    unsigned counts[kBins];
    Note note[2][kMaxCluster];
    Note red[kWarps];
    unsigned long long scan_mass[kWarps];
    unsigned scan_count[kWarps];
    unsigned listed;
    Found found;
    Cut cut;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The same variable of another CTA of the cluster.
template <typename T>
__device__ __forceinline__ T* of_rank(T* p, uint32_t rank) {
    uint64_t q;
    asm volatile("mapa.u64 %0, %1, %2;" : "=l"(q) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
    return reinterpret_cast<T*>(q);
}

// Integers that rise where the floats fall (no NaN; both zeros are one value).
__device__ __forceinline__ uint32_t key_of(float x) {
    const int i = __float_as_int(x + 0.f);
    return 0x7fffffffu - (uint32_t)(i ^ ((i >> 31) & 0x7fffffff));
}

// How notes are joined: the largest a with its lowest index i (-1: none), b summed.
__device__ __forceinline__ Note none() { return Note{-INFINITY, 0.f, -1, 0}; }
__device__ __forceinline__ void add(Note& v, float a, int i) {
    if (v.i < 0 || a > v.a) v.a = a, v.i = i;   // indexes come in increasing order
}
__device__ __forceinline__ Note join_warp(Note v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float a = __shfl_xor_sync(0xffffffffu, v.a, o);
        const int i = __shfl_xor_sync(0xffffffffu, v.i, o);
        v.b += __shfl_xor_sync(0xffffffffu, v.b, o);
        if (i >= 0 && (v.i < 0 || a > v.a || (a == v.a && i < v.i))) v.a = a, v.i = i;
    }
    return v;
}
// Of all threads of the cluster, for every thread, in a fixed order.
__device__ __forceinline__ Note join_all(Shared& s, int& step, Note v) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = (int)cluster_size();
    v = join_warp(v);
    if (lane == 0) s.red[warp] = v;
    __syncthreads();
    Note* slot = s.note[step++ & 1];
    if (warp == 0) {
        v = join_warp(lane < kWarps ? s.red[lane] : none());
        if (lane < n) *of_rank(&slot[cluster_rank()], lane) = v;
    }
    cluster_sync();
    return join_warp(lane < n ? slot[lane] : none());
}

// What a row's entries are measured with.
struct Row {
    float top;         // M
    float bins;        // bins a unit of distance
    double per_temp;
};
__device__ __forceinline__ int bin_of(const Row& r, float x) { return min(__float2int_rz((r.top - x) * r.bins), kBins - 1); }
// e in multiples of 2^-44; 0 where it is below half of that
__device__ __forceinline__ unsigned long long mass_of(const Row& r, float x) {
    const double z = ((double)x - (double)r.top) * r.per_temp;
    return z < -32.0 ? 0ull : __double2ull_rn(exp(z) * 0x1p44);
}

// Which entries a histogram is over, and their bins: by distance; or those with key in [lo, lo + span], by key; or those
// of key lo with index in [from, from + span], by index.
struct Range {
    int mode;
    uint32_t lo, span;
    int from, shift;
    int bin;            // mode 0: the bin that counts for `has`
};
__device__ __forceinline__ bool has(const Range& g, const Row& r, float x, int index) {
    if (g.mode == 0) return bin_of(r, x) == g.bin;
    const uint32_t k = key_of(x);
    return g.mode == 1 ? k - g.lo <= g.span : k == g.lo && (uint32_t)(index - g.from) <= g.span;
}
__device__ __forceinline__ int bin_in(const Range& g, float x, int index) {
    return g.mode == 1 ? (int)((key_of(x) - g.lo) >> g.shift) : (index - g.from) >> g.shift;
}

template <typename L>
struct Slice {
    const L* v;     // in shared memory
    int v0, n;      // index of the first, how many
};

__device__ __forceinline__ void count_one(Shared& s, int bin, unsigned long long mass) {
    atomicAdd(&s.count[bin], 1u);
    if (mass == 0) return;
    // 64 bits in two words: the low one says when it wrapped
    const unsigned low = (unsigned)mass, was = atomicAdd(&s.low[bin], low);
    const unsigned high = (unsigned)(mass >> 32) + (was + low < was ? 1u : 0u);
    if (high) atomicAdd(&s.high[bin], high);
}

// Fills s.counts and s.mass with the row's bins: mode 0: all entries but those of the last bin; else those of the range.
template <typename L>
__device__ void histogram(Shared& s, const Slice<L>& x, const Row& r, const Range& g, bool masses) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = s.low[i] = s.high[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < x.n; i += kThreads) {
        const float v = (float)x.v[i];
        int bin;
        if (g.mode == 0) {
            bin = bin_of(r, v);
            if (bin == kBins - 1) continue;
        } else {
            if (!has(g, r, v, x.v0 + i)) continue;
            bin = bin_in(g, v, x.v0 + i);
        }
        count_one(s, bin, masses ? mass_of(r, v) : 0ull);
    }
    cluster_sync();
    // each CTA adds its share of the bins and gives the sums to all
    const int n = (int)cluster_size(), share = kBins / n, b0 = (int)cluster_rank() * share;
    for (int b = b0 + threadIdx.x; b < b0 + share; b += kThreads) {
        unsigned count = 0;
        unsigned long long mass = 0;
        for (int k = 0; k < n; ++k) {
            count += *of_rank(&s.count[b], k);
            mass += ((unsigned long long)*of_rank(&s.high[b], k) << 32) + *of_rank(&s.low[b], k);
        }
        for (int k = 0; k < n; ++k) *of_rank(&s.counts[b], k) = count, *of_rank(&s.mass[b], k) = mass;
    }
    cluster_sync();
}

// The bin in which a cut lies: where the count reaches `k` (k > 0), else where the mass reaches `target`; bin -1 where none does.
// Threads with two bins each scan them in order.  mass: of all bins, for every thread.
__device__ unsigned long long find(Shared& s, unsigned k, double target, unsigned count0, unsigned long long mass0) {
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const unsigned c0 = s.counts[2 * t], c1 = s.counts[2 * t + 1];
    const unsigned long long m0 = s.mass[2 * t], m1 = s.mass[2 * t + 1];
    unsigned c = c0 + c1;
    unsigned long long m = m0 + m1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned pc = __shfl_up_sync(0xffffffffu, c, o);
        const unsigned long long pm = __shfl_up_sync(0xffffffffu, m, o);
        if (lane >= o) c += pc, m += pm;
    }
    if (lane == 31) s.scan_count[warp] = c, s.scan_mass[warp] = m;
    if (t == 0) s.found = Found{-1, 0, 0, 0};
    __syncthreads();
    unsigned before = count0;
    unsigned long long mass = mass0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s.scan_count[w], mass += s.scan_mass[w];
        all += s.scan_mass[w];
    }
    before += c - c0 - c1, mass += m - m0 - m1;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const unsigned cj = j ? c1 : c0;
        const unsigned long long mj = j ? m1 : m0;
        const bool here = k ? before < k && k <= before + cj : (double)mass < target && target <= (double)(mass + mj) && mj > 0;
        if (here) s.found = Found{2 * t + j, (int)before, (int)cj, mass};
        before += cj, mass += mj;
    }
    __syncthreads();
    return all;
}

// The cut by count (k > 0) or by mass (target) of the entries that g names, behind count0 entries of mass0: at most kList
// of them are compared with one another.
template <typename L>
__device__ void solve(Shared& s, const Slice<L>& x, const Row& r, const Range& g, unsigned k, double target, unsigned count0,
                      unsigned long long mass0) {
    if (cluster_rank() == 0 && threadIdx.x == 0) s.listed = 0;
    cluster_sync();
    unsigned* listed = of_rank(&s.listed, 0);
    Entry* list = of_rank(&s.list[0], 0);
    for (int i = threadIdx.x; i < x.n; i += kThreads) {
        const float v = (float)x.v[i];
        if (!has(g, r, v, x.v0 + i)) continue;
        const unsigned at = atomicAdd(listed, 1u);
        if (at < kList) list[at] = Entry{key_of(v), x.v0 + i};
    }
    cluster_sync();
    if (cluster_rank() == 0) {
        const int n = min((int)s.listed, kList);
        const int t = threadIdx.x;
        Entry mine{0xffffffffu, 0x7fffffff};
        unsigned long long mass = 0;
        if (t < n) {
            mine = s.list[t];
            const uint32_t o = 0x7fffffffu - mine.key;   // the float again
            mass = mass_of(r, __int_as_float((int)(o ^ (uint32_t)(((int)o >> 31) & 0x7fffffff))));
            s.list_mass[t] = mass;
        }
        __syncthreads();
        if (t < n) {
            unsigned before = count0;
            unsigned long long sum = mass0;
            for (int j = 0; j < n; ++j) {
                const Entry e = s.list[j];
                if (e.key < mine.key || (e.key == mine.key && e.index < mine.index)) ++before, sum += s.list_mass[j];
            }
            const bool last = k ? before + 1 == k : (double)sum < target && target <= (double)(sum + mass) && mass > 0;
            if (last) {
                const Cut cut{mine.key, mine.index, sum + mass};
                for (int j = 0; j < (int)cluster_size(); ++j) *of_rank(&s.cut, j) = cut;
            }
        }
    }
    cluster_sync();
}

// The cut by count (k > 0: behind the first k entries) or by mass (behind the shortest prefix with `target`), from the bins by
// distance, which are in s if `fresh`.  s.cut afterwards.  Returns whether the bins are still there.
template <typename L>
__device__ bool cut_at(Shared& s, int& step, const Slice<L>& x, const Row& r, bool fresh, unsigned k, double target, int vocab,
                       bool masses) {
    Range g{0, 0, 0, 0, 0, 0};
    if (!fresh) histogram(s, x, r, g, masses);
    find(s, k, target, 0, 0);
    Found f = s.found;
    if (f.bin < 0) {
        // behind all bins: the last one has the rest (and no mass)
        f.bin = kBins - 1;
        f.count = (int)(s.scan_count[0]);
        f.mass = s.scan_mass[0];
        for (int w = 1; w < kWarps; ++w) f.count += (int)s.scan_count[w], f.mass += s.scan_mass[w];
        f.in = vocab - f.count;
    }
    g.bin = f.bin;
    fresh = true;
    while (f.in > kList) {
        fresh = false;
        if (g.mode == 0) {
            // the range of the bin's keys (as floats of the row: largest and smallest)
            Note hi = none(), lo = none();
            for (int i = threadIdx.x; i < x.n; i += kThreads) {
                const float v = (float)x.v[i];
                if (bin_of(r, v) == g.bin) add(hi, v, i), add(lo, -v, i);
            }
            const float top = join_all(s, step, hi).a, bottom = -join_all(s, step, lo).a;
            g.mode = 1, g.lo = key_of(top), g.span = key_of(bottom) - g.lo;
        } else if (g.mode == 1) {
            g.lo += (uint32_t)f.bin << g.shift, g.span = min(g.span - ((uint32_t)f.bin << g.shift), (1u << g.shift) - 1);
        } else {
            g.from += f.bin << g.shift, g.span = min(g.span - ((uint32_t)f.bin << g.shift), (1u << g.shift) - 1);
        }
        if (g.mode == 1 && g.span == 0) g.mode = 2, g.from = 0, g.span = (uint32_t)vocab - 1;
        g.shift = max(0, 32 - __clz(g.span) - 10);   // span >> shift < 1024
        histogram(s, x, r, g, masses);
        find(s, k, target, (unsigned)f.count, f.mass);
        f = s.found;
        if (f.in <= kList) {
            // the bin's own range
            const uint32_t at = (uint32_t)f.bin << g.shift;
            if (g.mode == 1) g.lo += at;
            else g.from += (int)at;
            g.span = min(g.span - at, (1u << g.shift) - 1);
        }
    }
    solve(s, x, r, g, k, target, (unsigned)f.count, f.mass);
    return fresh;
}

template <typename L>
__global__ void __launch_bounds__(kThreads) k_sample(const __grid_constant__ Params p) {
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ Shared s;
    const SparkSample& a = p.a;
    const int cs = (int)cluster_size(), rank = (int)cluster_rank(), tid = threadIdx.x;
    const int64_t row = blockIdx.x / cs, b = row / a.nodes, node = row - b * a.nodes;
    const int vocab = (int)a.vocab;
    L* v = reinterpret_cast<L*>(raw);
    Slice<L> x{v, rank * p.slice, max(0, min(p.slice, vocab - rank * p.slice))};
    const L* logits = reinterpret_cast<const L*>(a.logits) + b * a.logits_stride[0] + node * a.logits_stride[1];
    cluster_arrive();
    grid_wait();
    const double temp = a.temperature ? (double)a.temperature[b] : a.temperature_all;
    const int64_t top_k = a.top_k ? (int64_t)a.top_k[b] : a.top_k_all;
    const double top_p = a.top_p ? (double)a.top_p[b] : a.top_p_all, min_p = a.min_p ? (double)a.min_p[b] : a.min_p_all;
    Note best = none();
    for (int i = tid; i < x.n; i += kThreads) {
        const L l = logits[x.v0 + i];
        v[i] = l;
        const float f = (float)l;
        if (f != f) best.b = 1.f;
        add(best, f, x.v0 + i);
    }
    cluster_wait();      // every CTA of the cluster has started: its shared memory may be written
    int step = 0;
    best = join_all(s, step, best);
    const bool none_here = best.b != 0.f || !(best.a > -INFINITY && best.a < INFINITY) || !(temp >= 0);
    Row r;
    r.top = best.a;
    const double t = fmin(fmax(temp, 1e-30), 1e30);
    r.per_temp = 1.0 / t;
    const bool by_k = !none_here && temp != 0 && top_k > 0 && top_k < vocab, by_p = !none_here && temp != 0 && top_p < 1;
    // (a cut by count has nothing to do with the temperature)
    r.bins = (float)((kBins - 1) / (by_k ? fmax(32 * t, 32.0) : 32 * t));
    Cut cut{0xffffffffu, 0x7fffffff, 0};
    float least = -INFINITY;
    if (none_here) {
    } else if (temp == 0) {
        cut = Cut{key_of(best.a), best.i, 0};
    } else {
        bool fresh = false;
        unsigned long long mass = 0;
        if (by_k) {
            fresh = cut_at(s, step, x, r, false, (unsigned)top_k, 0.0, vocab, by_p);
            cut = s.cut;
            mass = cut.mass;
            __syncthreads();
        }
        if (by_p) {
            if (!fresh) histogram(s, x, r, Range{0, 0, 0, 0, 0, 0}, true);
            if (!by_k) mass = find(s, 1, 0.0, 0, 0);
            // (at least half a multiple: the largest entry stays)
            const double target = fmax(top_p * (double)mass, 0.5);
            __syncthreads();
            cut_at(s, step, x, r, true, 0, target, vocab, true);
            cut = s.cut;
        }
        // e >= min_p, where exp's argument is (l - M) / T
        if (min_p > 0) least = __double2float_ru((double)best.a + fmin(log(min_p), 0.0) * t);
        least = fminf(least, best.a);
    }
    auto stays = [&](float f, int index) {
        if (!(f >= least)) return false;
        const uint32_t k = key_of(f);
        return k < cut.key || (k == cut.key && index <= cut.index);
    };
    if (a.out) {
        L* out = reinterpret_cast<L*>(a.out) + b * a.out_stride[0] + node * a.out_stride[1];
        for (int i = tid; i < x.n; i += kThreads)
            out[x.v0 + i] = none_here || stays((float)v[i], x.v0 + i) ? v[i] : (L)-INFINITY;
    }
    if (a.token) {
        Note got = none();
        if (!none_here && temp != 0) {
            const float* noise = a.noise + b * a.noise_stride;
            const float per = (float)r.per_temp;
            for (int i = tid; i < x.n; i += kThreads) {
                const float f = (float)v[i];
                if (!stays(f, x.v0 + i)) continue;
                const float e = expf((f - r.top) * per);
                got.b += e;
                if (e > 0.f) add(got, __fdividef(e, noise[x.v0 + i]), x.v0 + i);
            }
            got = join_all(s, step, got);
            // the owner of the token knows its logit
            if (a.logprob && got.i >= x.v0 && got.i < x.v0 + x.n && tid == 0)
                a.logprob[b] = ((float)v[got.i - x.v0] - r.top) * per - logf(got.b);
        } else if (!none_here) {
            got.i = best.i;
        }
        if (rank == 0 && tid == 0) {
            a.token[b] = got.i;
            if (a.logprob && (got.i < 0 || temp == 0.f)) a.logprob[b] = got.i < 0 ? NAN : 0.f;
        }
    }
    cluster_sync();   // (no CTA ends while another may still write to it)
}

inline int64_t slice_of(int64_t vocab, int cs) { return ((vocab + cs - 1) / cs + 15) / 16 * 16; }

// CTAs of a cluster: as in tree_verify.cu, where there are more rows than fit at once smaller clusters wait less.
int cluster_ctas(int64_t rows, int64_t vocab, int item, int sms) {
    int best = kMaxCluster;
    double least = 0;
    for (int cs = kMaxCluster; cs >= 1; cs /= 2) {
        const int64_t slice = slice_of(vocab, cs);
        if (slice * item > kRowBytes) break;
        const size_t bytes = sizeof(Shared) + slice * item + 1024;
        const double at_once = (double)sms * std::min<size_t>(4, kSmemSm / bytes) / cs;
        const double time = std::max(1.0, rows / at_once) * (16 * kThreads + slice);
        if (cs == kMaxCluster || time < least) best = cs, least = time;
    }
    return best;
}

template <typename L>
int launch(const Params& p, int64_t rows, int cs, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(k_sample<L>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowBytes);
    if (e != cudaSuccess) return set_error((int)e, "spark_sample: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * cs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)p.slice * sizeof(L);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, k_sample<L>, p);
    if (e != cudaSuccess) return set_error((int)e, "spark_sample: launch failed: %s", cudaGetErrorString(e));
    return check_launch("spark_sample");
}

}  // namespace sm
}  // namespace spark

extern "C" {

int spark_sample(const SparkSample* a, void* stream) {
    using namespace spark;
    using namespace spark::sm;
    SPARK_REQUIRE(a, SPARK_ERR_INVALID, "spark_sample: null pointer");
    SPARK_REQUIRE(a->batch >= 0 && a->nodes >= 0 && a->vocab >= 1, SPARK_ERR_INVALID, "spark_sample: bad size");
    SPARK_REQUIRE(a->dtype >= 0 && a->dtype <= 2, SPARK_ERR_INVALID, "spark_sample: bad dtype %d", (int)a->dtype);
    SPARK_REQUIRE(a->vocab <= kMaxVocab, SPARK_ERR_UNSUPPORTED, "spark_sample: a vocabulary of %lld entries is above %d",
                  (long long)a->vocab, kMaxVocab);
    SPARK_REQUIRE(a->batch < (1 << 24) && a->nodes < (1 << 24) && a->batch * a->nodes < (1 << 24), SPARK_ERR_UNSUPPORTED,
                  "spark_sample: more than 2^24 rows");
    if (a->batch == 0 || a->nodes == 0) return SPARK_OK;
    SPARK_REQUIRE(a->logits && (a->token || a->out), SPARK_ERR_INVALID, "spark_sample: null pointer");
    SPARK_REQUIRE(!a->token || (a->noise && a->nodes == 1), SPARK_ERR_INVALID, "spark_sample: a token takes noise, and one row a sequence");
    SPARK_REQUIRE(!a->logprob || a->token, SPARK_ERR_INVALID, "spark_sample: the probability of no token");
    if (a->out) {
        const int64_t extent[2] = {a->batch, a->nodes};
        bool same = true;
        for (int i = 0; i < 2; ++i) {
            SPARK_REQUIRE(extent[i] == 1 || a->out_stride[i] != 0, SPARK_ERR_INVALID, "spark_sample: output rows in one place");
            same = same && (extent[i] == 1 || a->out_stride[i] == a->logits_stride[i]);
        }
        SPARK_REQUIRE(a->out != a->logits || same, SPARK_ERR_INVALID, "spark_sample: in place needs equal strides");
    }
    Params p;
    p.a = *a;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return set_error((int)e, "spark_sample: %s", cudaGetErrorString(e));
    const int64_t rows = a->batch * a->nodes;
    const int item = a->dtype == SPARK_DTYPE_F32 ? 4 : 2;
    const int cs = cluster_ctas(rows, a->vocab, item, tc::sm_count_cached(dev));
    SPARK_REQUIRE(slice_of(a->vocab, cs) * item <= kRowBytes, SPARK_ERR_UNSUPPORTED, "spark_sample: vocabulary");
    p.slice = (int)slice_of(a->vocab, cs);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == SPARK_DTYPE_BF16) return launch<__nv_bfloat16>(p, rows, cs, st);
    if (a->dtype == SPARK_DTYPE_F16) return launch<__half>(p, rows, cs, st);
    return launch<float>(p, rows, cs, st);
}

}  // extern "C"
