// sample.cu -- sampling with temperature, top-k, top-p and min-p from given random
// numbers, and the same cut of logits for what samples later (a tree's verification).
//
// With M the largest logit, e(v) = exp((l(v) - M) / T).  In falling order of l, the
// lower index first, the first k entries stay; of those the shortest prefix whose sum
// of e is top_p of theirs or more; of those the entries with e >= min_p.  Each is a
// prefix of one order, so that all three are one cut (value, index).  The token is
// argmax e(v) / noise(v) over what stays: with exponential variates a sample.
//
// No sort.  Entries are told apart by their distance from M in bins (512 over 32 T,
// below which e is under 2^-45).
//  1. A histogram of the largest entries of 16-byte vectors gives a bin with at least k
//     entries at or before it (without a count: about a thirtieth of the row); what
//     lies there is listed, usually all that can stay.
//  2. A list of at most kPairs entries is compared with itself.  A longer one is
//     divided by a histogram with counts and sums of e, whose scan gives the bin that
//     the cut is in, and that bin again, by the integers in the order of the floats,
//     then, if all are equal, by their index, until so few are left.
//  3. top_p of a whole row takes its sum.  What is not listed is summed in fp32, with a
//     bound of the error; if that leaves the cut open, or the list is too short or too
//     long, step 2 is done on all entries.
// The sums decide borders, so that they have to be good, and may not depend on the order
// of atomics: e in 64 bits, added as multiples of 2^-44 in integers (409,600 entries of
// at most 1 fit 64 bits).
//
// One thread-block cluster of 8 CTAs (fewer where there are many rows) per row, each
// CTA a slice of the vocabulary that it keeps in shared memory, so that a row is read
// once; noise is read where an entry stays.  Bins and lists are exchanged through
// distributed shared memory; all CTAs take the same decisions.
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
constexpr int kBins = 512;              // the last one: all that is further away
constexpr int kPairs = 256;             // entries that are compared with one another
constexpr int kList = 4096;             // entries that a CTA lists
constexpr int kRowBytes = 200 * 1024;   // of a CTA's slice
constexpr int kMaxVocab = kMaxCluster * kRowBytes / 4;
constexpr int kSmemSm = 228 * 1024;     // shared memory of an SM
constexpr int kBatch = 4;               // vectors of a thread on the way together
static_assert(kBins == kThreads, "a thread has a bin");

struct Params {
    SparkSample a;
    int slice;   // vocabulary entries of a CTA, a multiple of 16
};

struct Note {
    float a, b;
    int i, pad;
};
// An entry's place in the falling order is (key, index), rising.
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
    uint32_t key;                       // what stays: smaller keys, of equal ones the indices up to this
    int index;
    unsigned long long before, mass;    // sums of e of what stays, without and with the last entry
    double target;                      // what they were compared with
};
// What a CTA tells the others with its list: entries in it (more than kList: too many), sum of e of the others, of |z| e.
struct Rest {
    int listed, pad;
    double sum, slope;
};
struct Shared {
    unsigned count[kBins];                                    // of this CTA, and the sums of e in two words
    union {
        unsigned low[kBins];
        Entry pair[kPairs];                                   // (rank 0's, when no sums are on the way)
    };
    union {
        unsigned high[kBins];
        unsigned long long pair_mass[kPairs];
    };
    unsigned long long mass[kBins];                           // of the row
    unsigned counts[kBins];
    uint16_t list[kList];
    Note note[2][kMaxCluster];
    Note red[kWarps];
    Rest rest[kMaxCluster];
    double red_sum[kWarps], red_slope[kWarps];
    unsigned long long scan_mass[kWarps];
    unsigned scan_count[kWarps];
    unsigned listed, pairs, base;
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
// Asks for bytes [p, p + n) in L2.
__device__ __forceinline__ void to_l2(const void* p, int64_t n) {
    const uintptr_t a = (reinterpret_cast<uintptr_t>(p) + 15) & ~uintptr_t(15);
    const int64_t m = (reinterpret_cast<intptr_t>(p) + n - (intptr_t)a) & ~int64_t(15);
    if (m > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a), "r"((uint32_t)m) : "memory");
}

// Integers that rise where the floats fall (no NaN; both zeros are one value), and back.
__device__ __forceinline__ uint32_t key_of(float x) {
    const int i = __float_as_int(x + 0.f);
    return 0x7fffffffu - (uint32_t)(i ^ ((i >> 31) & 0x7fffffff));
}
__device__ __forceinline__ float value_of(uint32_t key) {
    const int o = (int)(0x7fffffffu - key);
    return __int_as_float(o ^ ((o >> 31) & 0x7fffffff));
}

// 16 bytes of logits.
template <typename L>
struct Vec {
    static constexpr int N = 16 / sizeof(L);
    union {
        uint4 raw;
        L v[N];
    };
    __device__ __forceinline__ Vec() {}
    __device__ __forceinline__ Vec(const uint4& x) : raw(x) {}
    // the largest, a NaN if there is one
    __device__ __forceinline__ float largest() const;
};
template <>
__device__ __forceinline__ float Vec<float>::largest() const {
    float a, b;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(v[0]), "f"(v[1]));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(v[2]), "f"(v[3]));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
    return a;
}
template <>
__device__ __forceinline__ float Vec<__half>::largest() const {
    const __half2* h = reinterpret_cast<const __half2*>(v);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
}
template <>
__device__ __forceinline__ float Vec<__nv_bfloat16>::largest() const {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(v);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}

// How notes are joined: the largest a with its lowest index i (-1: none), b summed.
__device__ __forceinline__ Note none() { return Note{-INFINITY, 0.f, -1, 0}; }
__device__ __forceinline__ void add(Note& v, float a, int i) {
    if (v.i < 0 || a > v.a || (a == v.a && i < v.i)) v.a = a, v.i = i;
}
__device__ __forceinline__ Note join_warp(Note v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float a = __shfl_xor_sync(0xffffffffu, v.a, o);
        const int i = __shfl_xor_sync(0xffffffffu, v.i, o);
        v.b += __shfl_xor_sync(0xffffffffu, v.b, o);
        if (i >= 0) add(v, a, i);
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

// A CTA's part of a row, in shared memory, and the entries of it that are looked at: those listed, or all.
template <typename L>
struct Slice {
    const L* v;
    int v0, n;               // index of the first, how many
    const uint16_t* list;    // NULL: all
    int listed;

    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        if (list) {
            for (int i = threadIdx.x; i < listed; i += kThreads) f((float)v[list[i]], v0 + list[i]);
        } else {
            for (int i = threadIdx.x; i < n; i += kThreads) f((float)v[i], v0 + i);
        }
    }
};

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
__device__ __noinline__ void histogram(Shared& s, const Slice<L>& x, const Row& r, const Range& g, bool masses) {
    s.count[threadIdx.x] = s.low[threadIdx.x] = s.high[threadIdx.x] = 0;
    __syncthreads();
    x.each([&](float v, int index) {
        int bin;
        if (g.mode == 0) {
            bin = bin_of(r, v);
            if (bin == kBins - 1) return;
        } else {
            if (!has(g, r, v, index)) return;
            bin = bin_in(g, v, index);
        }
        count_one(s, bin, masses ? mass_of(r, v) : 0ull);
    });
    cluster_sync();
    // each CTA adds its share of the bins and gives the sums to all
    const int n = (int)cluster_size(), share = kBins / n, b = (int)cluster_rank() * share + threadIdx.x;
    if (threadIdx.x < share) {
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
// Behind count0 entries of mass0.  Returns the mass of all bins.
__device__ __noinline__ unsigned long long find(Shared& s, unsigned k, double target, unsigned count0, unsigned long long mass0) {
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const unsigned own = s.counts[t];
    const unsigned long long own_mass = s.mass[t];
    unsigned c = own;
    unsigned long long m = own_mass;
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
    before += c - own, mass += m - own_mass;
    const bool here = k ? before < k && k <= before + own
                        : (double)mass < target && target <= (double)(mass + own_mass) && own_mass > 0;
    if (here) s.found = Found{t, (int)before, (int)own, mass};
    __syncthreads();
    return all;
}

// Rank 0 compares its s.pairs entries with one another and tells all CTAs the cut: by count (k > 0), by mass (target > 0), or by
// top_p of the mass of the first k or, without k, of all and `rest`.  Behind count0 entries of mass0.  Where the cut is behind
// them all its mass is 0.
__device__ __noinline__ void solve(Shared& s, const Row& r, unsigned k, double target, double top_p, double rest, unsigned count0,
                                   unsigned long long mass0) {
    if (cluster_rank() == 0) {
        const int n = min((int)s.pairs, kPairs), t = threadIdx.x;
        if (t < n) s.pair_mass[t] = mass_of(r, value_of(s.pair[t].key));
        if (t == 0) s.cut.mass = 0;
        // as many threads an entry as there are
        int a_time = 32;
        while (a_time > kThreads / kPairs && a_time * n > kThreads) a_time >>= 1;
        const int e = t / a_time, sub = t & (a_time - 1);
        __syncthreads();
        Entry mine{0xffffffffu, 0x7fffffff};
        unsigned before = 0;
        unsigned long long sum = 0, mass = 0;
        if (e < n) {
            mine = s.pair[e], mass = s.pair_mass[e];
            for (int j = sub; j < n; j += a_time) {
                const Entry other = s.pair[j];
                if (other.key < mine.key || (other.key == mine.key && other.index < mine.index)) ++before, sum += s.pair_mass[j];
            }
        }
        for (int o = 1; o < a_time; o <<= 1) {
            before += __shfl_xor_sync(0xffffffffu, before, o);
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (!(target > 0) && top_p < 1) {
            // the last of the entries that count has the mass of them all
            if (e < n && sub == 0 && before + 1 == (k ? k : (unsigned)n)) s.scan_mass[0] = sum + mass;
            __syncthreads();
            // (at least half a multiple: the largest entry stays)
            target = fmax(top_p * ((double)s.scan_mass[0] + rest), 0.5);
        }
        before += count0, sum += mass0;
        if (e < n && sub == 0) {
            const bool last = target > 0 ? (double)sum < target && target <= (double)(sum + mass) && mass > 0 : before + 1 == k;
            if (last) s.cut = Cut{mine.key, mine.index, sum, sum + mass, target};
        }
        __syncthreads();
        if (t > 0 && t < (int)cluster_size()) *of_rank(&s.cut, t) = s.cut;
    }
    cluster_sync();
}

// The cut by count (k > 0: behind the first k entries) or by mass (behind the shortest prefix with `target`) of x's entries, from
// their bins by distance, which are in s if `fresh`.  s.cut afterwards.  Returns whether the bins are still there.
template <typename L>
__device__ __noinline__ bool cut_at(Shared& s, int& step, const Slice<L>& x, const Row& r, bool fresh, unsigned k, double target, int entries,
                                    int vocab, bool masses) {
    Range g{0, 0, 0, 0, 0, 0};
    if (!fresh) histogram(s, x, r, g, masses);
    find(s, k, target, 0, 0);
    Found f = s.found;
    if (f.bin < 0) {
        // behind all bins: the last one has the rest (and no mass)
        f = Found{kBins - 1, 0, 0, 0};
        for (int w = 0; w < kWarps; ++w) f.count += (int)s.scan_count[w], f.mass += s.scan_mass[w];
        f.in = entries - f.count;
    }
    g.bin = f.bin;
    fresh = true;
    while (f.in > kPairs) {
        fresh = false;
        if (g.mode == 0) {
            // the range of the bin's keys, from its largest and smallest value
            Note hi = none(), lo = none();
            x.each([&](float v, int index) {
                if (bin_of(r, v) == g.bin) add(hi, v, index), add(lo, -v, index);
            });
            const float top = join_all(s, step, hi).a, bottom = -join_all(s, step, lo).a;
            g.mode = 1, g.lo = key_of(top), g.span = key_of(bottom) - g.lo;
        }
        if (g.mode == 1 && g.span == 0) g.mode = 2, g.from = 0, g.span = (uint32_t)vocab - 1;
        g.shift = max(0, 32 - __clz(g.span) - 9);   // span >> shift < 512
        histogram(s, x, r, g, masses);
        find(s, k, target, (unsigned)f.count, f.mass);
        f = s.found;
        // the bin's own range
        const uint32_t at = (uint32_t)f.bin << g.shift;
        if (g.mode == 1) g.lo += at;
        else g.from += (int)at;
        g.span = min(g.span - at, (1u << g.shift) - 1);
    }
    if (cluster_rank() == 0 && threadIdx.x == 0) s.pairs = 0;
    cluster_sync();
    unsigned* pairs = of_rank(&s.pairs, 0);
    Entry* pair = of_rank(&s.pair[0], 0);
    x.each([&](float v, int index) {
        if (!has(g, r, v, index)) return;
        const unsigned at = atomicAdd(pairs, 1u);
        if (at < kPairs) pair[at] = Entry{key_of(v), index};
    });
    cluster_sync();
    solve(s, r, k, target, 1.0, 0.0, (unsigned)f.count, f.mass);
    return fresh;
}

// The cut of x's entries, which have all that stays: by count, and by top_p of those; or by mass.
template <typename L>
__device__ __forceinline__ void cut_all(Shared& s, int& step, const Slice<L>& x, const Row& r, unsigned k, double top_p, double target,
                                        bool fresh, int entries, int vocab) {
    if (k) {
        fresh = cut_at(s, step, x, r, false, k, 0.0, entries, vocab, top_p < 1);
        if (!(top_p < 1)) return;
        // (at least half a multiple: the largest entry stays)
        target = fmax(top_p * (double)s.cut.mass, 0.5);
        __syncthreads();
    }
    cut_at(s, step, x, r, fresh, 0, target, entries, vocab, true);
}

template <typename L>
__global__ void __launch_bounds__(kThreads, 2) k_sample(const __grid_constant__ Params p) {
    using V = Vec<L>;
    constexpr int N = V::N;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ Shared s;
    const SparkSample& a = p.a;
    const int cs = (int)cluster_size(), rank = (int)cluster_rank(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.x / cs, b = row / a.nodes, node = row - b * a.nodes;
    const int vocab = (int)a.vocab, v0 = rank * p.slice, n = max(0, min(p.slice, vocab - v0));
    const L* logits = reinterpret_cast<const L*>(a.logits) + b * a.logits_stride[0] + node * a.logits_stride[1] + v0;
    cluster_arrive();
    grid_wait();
    const double temp = a.temperature ? (double)a.temperature[b] : a.temperature_all;
    const int64_t top_k = a.top_k ? (int64_t)a.top_k[b] : a.top_k_all;
    const double top_p = a.top_p ? (double)a.top_p[b] : a.top_p_all, min_p = a.min_p ? (double)a.min_p[b] : a.min_p_all;
    bool by_k = top_k > 0 && top_k < vocab, by_p = top_p < 1;
    const float* noise = a.token ? a.noise + b * a.noise_stride + v0 : nullptr;
    if (noise && !by_k && !by_p && !(min_p > 0) && temp > 0 && tid == 0) to_l2(noise, (int64_t)n * 4);

    // the slice, in vectors that lie as they do in memory: `head` entries of the first one belong to another slice, or row
    const int head = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(L)), vectors = n ? (head + n + N - 1) / N : 0;
    uint4* const vec = reinterpret_cast<uint4*>(raw);
    const uint4* const from = reinterpret_cast<const uint4*>(logits - head);
    float most = -INFINITY;
    for (int i0 = tid; i0 < vectors; i0 += kBatch * kThreads) {
        V x[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = i0 + k * kThreads;
            if (i >= vectors) continue;
            if (i * N >= head && (i + 1) * N <= head + n) {
                x[k].raw = from[i];
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int at = i * N + j - head;
                    x[k].v[j] = at >= 0 && at < n ? logits[at] : (L)-INFINITY;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = i0 + k * kThreads;
            if (i >= vectors) continue;
            vec[i] = x[k].raw;
            const float m = x[k].largest();
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(m));
        }
    }
    Slice<L> x{reinterpret_cast<const L*>(raw) + head, v0, n, nullptr, 0};
    cluster_wait();      // every CTA of the cluster has started: its shared memory may be written
    int step = 0;
    Note best{most == most ? most : -INFINITY, most == most ? 0.f : 1.f, 0, 0};
    best = join_all(s, step, best);
    Row r;
    r.top = best.a;
    const bool none_here = best.b != 0.f || !(best.a > -INFINITY && best.a < INFINITY) || !(temp >= 0);
    const bool greedy = !none_here && temp == 0;
    const double t = fmin(fmax(temp, 1e-30), 1e30);
    r.per_temp = 1.0 / t;
    by_k = by_k && !none_here && !greedy, by_p = by_p && !none_here && !greedy;
    // (a cut by count has nothing to do with the temperature)
    r.bins = (float)((kBins - 1) / (by_k ? fmax(32 * t, 32.0) : 32 * t));
    const float per = (float)r.per_temp;
    float limit = -INFINITY;      // what stays: above this, or equal with an index up to `last`
    int last = 0x7fffffff;
    if (greedy) {
        Note first = none();
        x.each([&](float f, int index) {
            if (f == r.top) add(first, f, index);
        });
        limit = r.top, last = join_all(s, step, first).i;
    } else if (by_k || by_p) {
        // the bin by which there are enough entries, from the vectors' largest
        s.count[tid] = 0;
        if (tid == 0) s.listed = s.pairs = 0;
        __syncthreads();
        for (int i = tid; i < vectors; i += kThreads) {
            const int bin = bin_of(r, V(vec[i]).largest());
            if (bin < kBins - 1) atomicAdd(&s.count[bin], 1u);
        }
        cluster_sync();
        {
            unsigned count = 0;
            for (int k = 0; k < cs; ++k) count += *of_rank(&s.count[tid], k);
            s.counts[tid] = count, s.mass[tid] = 0;
        }
        __syncthreads();
        find(s, by_k ? (unsigned)top_k : (unsigned)max(64, vocab / 32), 0.0, 0, 0);
        const int bound = s.found.bin >= 0 ? s.found.bin : kBins - 2;
        const bool reached = !by_k || s.found.bin >= 0;
        // what is not further away; of the rest the sum, where that is asked for
        double sum = 0, slope = 0;
        for (int i = tid; i < vectors && reached; i += kThreads) {
            const V u(vec[i]);
            if (bin_of(r, u.largest()) <= bound) {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (bin_of(r, (float)u.v[j]) <= bound) {
                        const unsigned at = atomicAdd(&s.listed, 1u);
                        if (at < kList) s.list[at] = (uint16_t)(i * N + j - head);
                    }
            }
            if (by_k) continue;
            float e = 0.f, f = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float d = (float)u.v[j] - r.top;
                if (bin_of(r, (float)u.v[j]) <= bound || !(d > -INFINITY)) continue;
                const float z = d * per, q = expf(z);
                e += q, f = fmaf(-z, q, f);
            }
            sum += e, slope += f;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o), slope += __shfl_xor_sync(0xffffffffu, slope, o);
        if (lane == 0) s.red_sum[warp] = sum, s.red_slope[warp] = slope;
        __syncthreads();
        const int listed = (int)s.listed;
        if (tid < cs) {
            Rest mine{listed, 0, 0, 0};
            for (int w = 0; w < kWarps; ++w) mine.sum += s.red_sum[w], mine.slope += s.red_slope[w];
            *of_rank(&s.rest[rank], tid) = mine;
        }
        if (listed <= kPairs) {
            // perhaps all are few: rank 0 has them then
            if (tid == 0) s.base = atomicAdd(of_rank(&s.pairs, 0), (unsigned)listed);
            __syncthreads();
            Entry* pair = of_rank(&s.pair[0], 0);
            if (tid < listed && s.base + tid < kPairs) pair[s.base + tid] = Entry{key_of((float)x.v[s.list[tid]]), v0 + s.list[tid]};
        }
        cluster_sync();
        int total = 0;
        bool fits = reached;
        sum = slope = 0;
        for (int k = 0; k < cs; ++k) {
            const Rest& c = s.rest[k];
            total += c.listed, fits = fits && c.listed <= kList, sum += c.sum, slope += c.slope;
        }
        x.list = s.list, x.listed = listed;
        bool done = false;
        const double scale = 0x1p44, rest = sum * scale;
        const unsigned k = by_k ? (unsigned)top_k : 0;
        if (fits && by_k) {
            if (total <= kPairs) solve(s, r, k, 0.0, top_p, 0.0, 0, 0);
            else cut_all(s, step, x, r, k, top_p, 0.0, false, total, vocab);
            done = true;
        } else if (fits) {
            if (total <= kPairs) {
                solve(s, r, 0, 0.0, top_p, rest, 0, 0);
                done = s.cut.mass > 0;
            } else {
                histogram(s, x, r, Range{0, 0, 0, 0, 0, 0}, true);
                const double whole = (double)find(s, 1, 0.0, 0, 0), target = fmax(top_p * (whole + rest), 0.5);
                __syncthreads();
                done = target <= whole;
                if (done) cut_all(s, step, x, r, 0, 1.0, target, true, total, vocab);
            }
            if (done) {
                // The terms of the rest are off by 2^-23 (expf) and 7 2^-24 (sums of 8) of themselves, and by 3 2^-24 |z| (a
                // difference, a factor and a product); the cut is certain where that does not reach the next entry.
                const double off = top_p * (sum * 0x1p-20 + slope * 0x1p-22) * scale;
                done = (double)s.cut.before < s.cut.target - off && s.cut.target + off <= (double)s.cut.mass;
            }
        }
        if (!done) {
            x.list = nullptr;
            double target = 0;
            __syncthreads();
            if (!by_k) {
                histogram(s, x, r, Range{0, 0, 0, 0, 0, 0}, true);
                target = fmax(top_p * (double)find(s, 1, 0.0, 0, 0), 0.5);
                __syncthreads();
            }
            cut_all(s, step, x, r, k, top_p, target, !by_k, vocab, vocab);
        }
        limit = value_of(s.cut.key), last = s.cut.index;
    }
    // e >= min_p, where exp's argument is (l - M) / T
    if (min_p > 0 && !none_here && !greedy) {
        const float least = fminf(__double2float_ru((double)r.top + fmin(log(min_p), 0.0) * t), r.top);
        if (least > limit) limit = least, last = 0x7fffffff;
    }
    auto stays = [&](float f, int index) { return f > limit || (f == limit && index <= last); };
    if (a.out) {
        L* out = reinterpret_cast<L*>(a.out) + b * a.out_stride[0] + node * a.out_stride[1] + v0;
        const bool alike = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(logits)) & 15) == 0;
        for (int i = tid; i < vectors; i += kThreads) {
            V u(vec[i]);
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (!none_here && !stays((float)u.v[j], v0 + i * N + j - head)) u.v[j] = (L)-INFINITY;
            if (alike && i * N >= head && (i + 1) * N <= head + n) {
                reinterpret_cast<uint4*>(out - head)[i] = u.raw;
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int at = i * N + j - head;
                    if (at >= 0 && at < n) out[at] = u.v[j];
                }
            }
        }
    }
    if (!a.token) return;
    Note got = none();
    if (!none_here && !greedy) {
        auto draw = [&](float f, int index, float e) {
            const float q = expf((f - r.top) * per);
            got.b += q;
            if (q > 0.f) add(got, __fdividef(q, e), index);
        };
        if (x.list) {
            x.each([&](float f, int index) {
                if (stays(f, index)) draw(f, index, noise[index - v0]);
            });
        } else {
            constexpr int kAhead = 8;
            for (int i0 = tid; i0 < n; i0 += kAhead * kThreads) {
                float f[kAhead], e[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int i = i0 + k * kThreads;
                    f[k] = i < n ? (float)x.v[i] : -INFINITY;
                    e[k] = i < n && stays(f[k], v0 + i) ? noise[i] : 0.f;
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int i = i0 + k * kThreads;
                    if (i < n && stays(f[k], v0 + i)) draw(f[k], v0 + i, e[k]);
                }
            }
        }
        got = join_all(s, step, got);
    } else if (greedy) {
        got.i = last;
    }
    // the owner of the token knows its logit
    if (a.logprob && !none_here && !greedy && got.i >= v0 && got.i < v0 + n && tid == 0)
        a.logprob[b] = ((float)x.v[got.i - v0] - r.top) * per - logf(got.b);
    if (rank == 0 && tid == 0) {
        a.token[b] = got.i;
        if (a.logprob && (got.i < 0 || greedy)) a.logprob[b] = got.i < 0 ? NAN : 0.f;
    }
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
    cudaError_t e = cudaFuncSetAttribute(k_sample<L>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowBytes + 16);
    if (e != cudaSuccess) return set_error((int)e, "spark_sample: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * cs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)p.slice * sizeof(L) + 16;   // (a vector more where the slice does not begin with one)
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
