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
//  1. A thread has the largest entries of four groups of its 16-byte vectors.  A
//     histogram of those gives a bin with at least k entries at or before it (without a
//     count: about a thirtieth of the row); what lies there is listed, usually all that
//     can stay.
//  2. A list of at most kPairs entries is compared with itself.  A longer one is
//     divided by a histogram with counts and sums of e, whose scan gives the bin that
//     the cut is in, and that bin again, by the integers in the order of the floats,
//     then, if all are equal, by their index, until so few are left.
//  3. top_p of a whole row takes its sum.  What is not listed is summed in fp32, with a
//     bound of the error; if that leaves the cut open, in 64 bits.  If the list has too
//     little of it, a longer one is made; if that has too, or is too long, step 2 is done on
//     all entries.
// The sums decide borders, so that they have to be good, and may not depend on the order
// of atomics: e in 64 bits, added as multiples of 2^-44 in integers (409,600 entries of
// at most 1 fit 64 bits).
//
// A row is kept in shared memory, so that it is read once; noise is read where an entry
// stays.  A CTA takes a row that fits (up to 200 KB).  A longer one is cut into the
// slices of a thread-block cluster, which exchange bins and lists through distributed
// shared memory and all take the same decisions; a step costs a cluster barrier
// then (2000 cycles or more each, against some hundred).
//
// Few rows are bound by that chain of steps: one of 151,936 in fp32 takes 8.6 us without
// a cut, 12.5 with top_k 50, 12.7 with top_p 0.9 of those, 23 with top_p 0.95 of all.
// Many are bound by the instructions a value (a few to find the largest, some 10 more where
// top_p sums a row): 1024 rows of 32,000 in bf16 61 us without a cut (the noise is read: 3.2
// TB/s; 64 with logprob, whose sum is in integers), 47 with top_k 50, 93 with top_p 0.95.  A flat distribution, of which more stays
// than lists hold, is divided by histograms of all its entries, whose exponentials in 64
// bits bound it (four at a time take no less): 130 to 220 us for 64 rows of 100,003; and a
// row in some hundred whose border the sums in fp32 leave open takes 20 to 50 us more.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "overlap.cuh"

namespace spark {
namespace tc {
int sm_count_cached(int dev);
}

namespace sm {

constexpr int kThreads = 512;           // (1024: 1 to 70% longer, 200 rows of 32,000 19.8 us for 12.2)
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 512;              // the last one: all that is further away
constexpr int kPairs = 256;             // entries that are compared with one another
constexpr int kList = 6144;             // entries that a CTA lists
constexpr int kRowBytes = 200 * 1024;   // of a CTA's slice
constexpr int kSmemSm = 228 * 1024;     // shared memory of an SM
constexpr int kLongBytes = 96 * 1024;   // of a row that a cluster may be faster for
constexpr int kMaxVocab = kMaxCluster * kRowBytes / 4;
constexpr int kGroups = 4;              // of a thread's vectors, which are on the way together

struct Params {
    SparkSample a;
    int slice;   // vocabulary entries of a CTA, a multiple of 16
};

struct Note {
    float a;
    int i;
    unsigned long long b;
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
    unsigned long long target;          // what they were compared with
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
    uint16_t list[kList];                                     // places among the vectors; those from 65536 on from the end back
    Note note[2][kMaxCluster];
    Note red[2][kWarps];
    Rest rest[kMaxCluster];
    double red_sum[kWarps], red_slope[kWarps];
    unsigned long long scan_mass[kWarps];
    unsigned scan_count[kWarps];
    unsigned listed[2], pairs, base;
    double per_temp, reach;                                   // 1 / T; how far below M min_p reaches
    float bins;
    Found found;
    int further;
    Cut cut;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
__device__ __forceinline__ void cluster_sync() {
    if (cluster_size() == 1) {
        __syncthreads();
        return;
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
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

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two values an instruction, and the sum of their bits.
using Two = unsigned long long;
__device__ __forceinline__ Two two(float a, float b) {
    Two v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ Two add(Two a, Two b) {
    Two v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
    Two v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ void add_bits(unsigned& sum, Two v) { sum += (unsigned)v + (unsigned)(v >> 32); }

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

__device__ __forceinline__ Note none() { return Note{-INFINITY, -1, 0}; }
__device__ __forceinline__ void add(Note& v, float a, int i) {
    if (v.i < 0 || a > v.a || (a == v.a && i < v.i)) v.a = a, v.i = i;
}
// Integers in the order of the floats (no NaN), and back.
__device__ __forceinline__ int ordered(float x) {
    const int i = __float_as_int(x);
    return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
// The sum over a warp.
__device__ __forceinline__ unsigned long long sum_of_warp(unsigned long long x) {
    const unsigned a = __reduce_add_sync(0xffffffffu, (unsigned)x & 0x7ffffff), b = __reduce_add_sync(0xffffffffu, (unsigned)(x >> 27) & 0x7ffffff),
                   c = __reduce_add_sync(0xffffffffu, (unsigned)(x >> 54));
    return ((unsigned long long)c << 54) + ((unsigned long long)b << 27) + a;
}
// How notes are joined: the largest a with its lowest index i (-1: none), b summed.
__device__ __forceinline__ Note join_warp(Note v) {
    const float top = unordered(__reduce_max_sync(0xffffffffu, ordered(v.i < 0 ? -INFINITY : v.a)));
    const unsigned first = __reduce_min_sync(0xffffffffu, v.i >= 0 && v.a == top ? (unsigned)v.i : 0xffffffffu);
    return Note{top, (int)first, sum_of_warp(v.b)};
}
// Of all threads of the cluster, for every thread, in a fixed order.
__device__ __forceinline__ Note join_all(Shared& s, int& step, Note v) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = (int)cluster_size();
    v = join_warp(v);
    Note* red = s.red[step & 1];
    if (lane == 0) red[warp] = v;
    __syncthreads();
    Note* slot = s.note[step++ & 1];
    if (n == 1) return join_warp(lane < kWarps ? red[lane] : none());
    if (warp == 0) {
        v = join_warp(lane < kWarps ? red[lane] : none());
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
    int listed, low;         // of them below 65536
    int head;                // places before v

    __device__ __forceinline__ int at(int i) const { return (i < low ? list[i] : 65536 + list[kList - 1 - (i - low)]) - head; }

    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        if (list) {
            for (int i = threadIdx.x; i < listed; i += kThreads) {
                const int j = at(i);
                f((float)v[j], v0 + j);
            }
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

// Adds the bins of the CTAs into s.counts and, if asked, s.mass: each CTA its share, which it gives to all.
__device__ __forceinline__ void add_bins(Shared& s, bool masses) {
    if (cluster_size() == 1) {
        const int b = threadIdx.x;
        __syncthreads();
        if (b < kBins) {
            s.counts[b] = s.count[b];
            if (masses) s.mass[b] = ((unsigned long long)s.high[b] << 32) + s.low[b];
        }
        __syncthreads();
        return;
    }
    cluster_sync();
    const int n = (int)cluster_size(), share = kBins / n, b = (int)cluster_rank() * share + threadIdx.x;
    if (threadIdx.x < share) {
        unsigned count = 0;
        unsigned long long mass = 0;
        for (int k = 0; k < n; ++k) {
            count += *of_rank(&s.count[b], k);
            if (masses) mass += ((unsigned long long)*of_rank(&s.high[b], k) << 32) + *of_rank(&s.low[b], k);
        }
        for (int k = 0; k < n; ++k) {
            *of_rank(&s.counts[b], k) = count;
            if (masses) *of_rank(&s.mass[b], k) = mass;
        }
    }
    cluster_sync();
}
// Fills s.counts and s.mass with the row's bins: mode 0: all entries but those of the last bin; else those of the range.
template <typename L>
__device__ __noinline__ void histogram(Shared& s, const Slice<L>& x, const Row& r, const Range& g, bool masses) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = s.low[i] = s.high[i] = 0;
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
    add_bins(s, true);
}

// The bin in which the count reaches k, from s.counts; bin -1 where none does.  And that for `more`, in s.further.
__device__ __forceinline__ void find_count(Shared& s, unsigned k, unsigned more) {
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const unsigned own = t < kBins ? s.counts[t] : 0;
    unsigned c = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned pc = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c += pc;
    }
    if (lane == 31) s.scan_count[warp] = c;
    if (t == 0) s.found = Found{-1, 0, 0, 0}, s.further = -1;
    __syncthreads();
    const unsigned before = __reduce_add_sync(0xffffffffu, lane < warp ? s.scan_count[lane] : 0) + c - own;
    if (before < k && k <= before + own) s.found = Found{t, (int)before, (int)own, 0};
    if (before < more && more <= before + own) s.further = t;
    __syncthreads();
}

// The mass of all bins, for every thread.
__device__ __noinline__ unsigned long long mass_of_bins(Shared& s) {
    const int t = threadIdx.x, lane = t & 31;
    if (t < kBins) {
        const unsigned long long m = sum_of_warp(s.mass[t]);
        if (lane == 0) s.scan_mass[t >> 5] = m;
    }
    __syncthreads();
    const unsigned long long all = sum_of_warp(lane < kBins / 32 ? s.scan_mass[lane] : 0);
    __syncthreads();
    return all;
}
// The sum over the cluster, for every thread.
__device__ __noinline__ unsigned long long sum_of_all(Shared& s, unsigned long long x) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = (int)cluster_size();
    x = sum_of_warp(x);
    __syncthreads();
    if (lane == 0) s.scan_mass[warp] = x;
    __syncthreads();
    x = sum_of_warp(lane < kWarps ? s.scan_mass[lane] : 0);
    if (n == 1) return x;
    if (threadIdx.x < n) *of_rank(&s.mass[cluster_rank()], threadIdx.x) = x;
    cluster_sync();
    return sum_of_warp(lane < n ? s.mass[lane] : 0);
}
// The bin in which a cut lies: where the count reaches `k` (k > 0), else where the mass reaches `target`.  Behind count0 entries of
// mass0.  Where none does, bin -1, with the count and the mass of all.
__device__ __noinline__ void find(Shared& s, unsigned k, unsigned long long target, unsigned count0, unsigned long long mass0) {
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    unsigned own = 0, c = 0;
    unsigned long long own_mass = 0, m = 0;
    if (t < kBins) {
        c = own = s.counts[t], m = own_mass = s.mass[t];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned pc = __shfl_up_sync(0xffffffffu, c, o);
            const unsigned long long pm = __shfl_up_sync(0xffffffffu, m, o);
            if (lane >= o) c += pc, m += pm;
        }
        if (lane == 31) s.scan_count[warp] = c, s.scan_mass[warp] = m;
    }
    __syncthreads();
    if (t < kBins) {
        const unsigned before = count0 + c - own + __reduce_add_sync(0xffffffffu, lane < warp ? s.scan_count[lane] : 0);
        const unsigned long long mass = mass0 + m - own_mass + sum_of_warp(lane < warp ? s.scan_mass[lane] : 0);
        const bool here = k ? before < k && k <= before + own : mass < target && target <= mass + own_mass;
        if (here) s.found = Found{t, (int)before, (int)own, mass};
        if (t == kBins - 1 && (k ? before + own < k : mass + own_mass < target)) s.found = Found{-1, (int)(before + own), 0, mass + own_mass};
    }
    __syncthreads();
}
// The share top_p of a mass (at least one multiple: the largest entry stays).
__device__ __forceinline__ unsigned long long share_of(double top_p, double mass) { return (unsigned long long)fmax(ceil(top_p * mass), 1.0); }

// Rank 0 compares its s.pairs entries with one another and tells all CTAs the cut: by count (k > 0), by mass (target > 0), or by
// top_p of the mass of the first k or, without k, of all and `rest`.  Behind count0 entries of mass0.  Where the cut is behind
// them all its mass is 0.
__device__ __noinline__ void solve(Shared& s, const Row& r, unsigned k, unsigned long long target, double top_p, double rest, unsigned count0,
                                   unsigned long long mass0) {
    if (cluster_rank() == 0) {
        const int n = min((int)s.pairs, kPairs), t = threadIdx.x;
        if (t < n) s.pair_mass[t] = mass_of(r, value_of(s.pair[t].key));
        if (t == 0) s.cut.mass = 0;
        // a few threads an entry, so that each compares about 16
        int part = 1;
        while (part < 4 && (n >> part) > 16 && (n << (part + 1)) <= kThreads) ++part;
        const int e = t >> part, sub = t & ((1 << part) - 1);
        __syncthreads();
        Entry mine{0xffffffffu, 0x7fffffff};
        unsigned before = 0;
        unsigned long long sum = 0, mass = 0;
        if (e < n) {
            mine = s.pair[e], mass = s.pair_mass[e];
            const uint64_t place = (uint64_t)mine.key << 32 | (uint32_t)mine.index;
            for (int j = sub; j < n; j += 1 << part) {
                const Entry other = s.pair[j];
                const bool first = ((uint64_t)other.key << 32 | (uint32_t)other.index) < place;
                before += first, sum += first ? s.pair_mass[j] : 0;
            }
        }
        for (int o = 1; o < 1 << part; o <<= 1) {
            before += __shfl_xor_sync(0xffffffffu, before, o);
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (target == 0 && top_p < 1) {
            // the last of the entries that count has the mass of them all
            if (e < n && sub == 0 && before + 1 == (k ? k : (unsigned)n)) s.scan_mass[0] = sum + mass;
            __syncthreads();
            target = share_of(top_p, (double)s.scan_mass[0] + rest);
        }
        before += count0, sum += mass0;
        if (e < n && sub == 0) {
            const bool last = target ? sum < target && target <= sum + mass : before + 1 == k;
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
__device__ __noinline__ bool cut_at(Shared& s, int& step, const Slice<L>& x, const Row& r, bool fresh, unsigned k, unsigned long long target, int entries,
                                    int vocab, bool masses) {
    Range g{0, 0, 0, 0, 0, 0};
    if (!fresh) histogram(s, x, r, g, masses);
    find(s, k, target, 0, 0);
    Found f = s.found;
    // behind all bins: the last one has the rest (and no mass)
    if (f.bin < 0) f.bin = kBins - 1, f.in = entries - f.count;
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
__device__ __forceinline__ void cut_all(Shared& s, int& step, const Slice<L>& x, const Row& r, unsigned k, double top_p, unsigned long long target,
                                        bool fresh, int entries, int vocab) {
    if (k) {
        fresh = cut_at(s, step, x, r, false, k, 0ull, entries, vocab, top_p < 1);
        if (!(top_p < 1)) return;
        target = share_of(top_p, (double)s.cut.mass);
        __syncthreads();
    }
    cut_at(s, step, x, r, fresh, 0, target, entries, vocab, true);
}

// Lists x's entries from `edge` on, of the groups of vectors that have some, and gives rank 0 all of them where they are few; with
// `sums`, those of what is not listed.
struct Listed {
    int total;      // of the cluster
    bool fits;
    double sum, slope;
};
template <typename L>
__device__ __forceinline__ Listed list_from(Shared& s, Slice<L>& x, const Row& r, const uint4* vec, int vectors, unsigned groups, bool sums, float per2,
                                         float edge) {
    using V = Vec<L>;
    constexpr int N = V::N;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cs = (int)cluster_size();
    const float per2_low = (float)(r.per_temp * 1.4426950408889634 - (double)per2), lowest = fmaxf(-200.f / per2, -FLT_MAX);
    double sum = 0, slope = 0;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        if (!(groups >> k & 1)) continue;
        for (int i = tid + k * kThreads; i < vectors; i += kGroups * kThreads) {
            const V u(vec[i]);
            if (u.largest() >= edge) {
                unsigned which = 0;
#pragma unroll
                for (int j = 0; j < N; ++j) which |= (float)u.v[j] >= edge ? 1u << j : 0u;
                const int place = i * N, far = place >> 16;
                unsigned at = atomicAdd(&s.listed[far], (unsigned)__popc(which));
                for (; which && at < kList; which &= which - 1, ++at)
                    s.list[far ? kList - 1 - at : at] = (uint16_t)(place + __ffs(which) - 1);
            }
            if (!sums) continue;
            float e[N], f = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                // 2^z, z in two terms: a difference and 1 / T in two
                const float v = (float)u.v[j], d = fmaxf(v - r.top, lowest), z = d * per2;   // (2^-200 is 0)
                const float q = v < edge ? exp2_of(z) : 0.f, low = fmaf(d, per2_low, fmaf(d, per2, -z)) * 0.69314718f;
                e[j] = fmaf(q, low, q), f = fmaf(z, q, f);
            }
#pragma unroll
            for (int o = N / 2; o > 0; o >>= 1)
#pragma unroll
                for (int j = 0; j < o; ++j) e[j] += e[j + o];
            sum += e[0], slope -= f;
        }
    }
    if (sums) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o), slope += __shfl_xor_sync(0xffffffffu, slope, o);
        if (lane == 0) s.red_sum[warp] = sum, s.red_slope[warp] = slope;
    }
    __syncthreads();
    const int listed = (int)(s.listed[0] + s.listed[1]);
    x.list = s.list, x.listed = listed, x.low = (int)s.listed[0];
    if (warp == 0) {
        sum = slope = 0;
        if (sums) {
            if (lane < kWarps) sum = s.red_sum[lane], slope = s.red_slope[lane];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o), slope += __shfl_xor_sync(0xffffffffu, slope, o);
        }
        if (lane < cs) *of_rank(&s.rest[cluster_rank()], lane) = Rest{listed, 0, sum, slope};
    }
    if (listed <= kPairs) {
        // perhaps all are few: rank 0 has them then
        if (tid == 0) s.base = atomicAdd(of_rank(&s.pairs, 0), (unsigned)listed);
        __syncthreads();
        Entry* pair = of_rank(&s.pair[0], 0);
        if (tid < listed && s.base + tid < kPairs) pair[s.base + tid] = Entry{key_of((float)x.v[x.at(tid)]), x.v0 + x.at(tid)};
    }
    cluster_sync();
    Listed all{0, true, 0, 0};
    for (int k = 0; k < cs; ++k) {
        const Rest& c = s.rest[k];
        all.total += c.listed, all.fits = all.fits && c.listed <= kList, all.sum += c.sum, all.slope += c.slope;
    }
    return all;
}

// The cut by top_p of a row of which x's entries are listed, from `edge` on, if it is among them.
template <typename L>
__device__ __forceinline__ bool cut_by_mass(Shared& s, int& step, const Slice<L>& x, const Row& r, const Listed& l, double top_p, int vocab, float edge) {
    // (a mass of all that the list does not reach is found out about by the caller)
    auto cut = [&](double more) {
        if (l.total <= kPairs) {
            solve(s, r, 0, 0ull, top_p, more, 0, 0);
            return s.cut.mass > 0;
        }
        histogram(s, x, r, Range{0, 0, 0, 0, 0, 0}, true);
        const unsigned long long whole = mass_of_bins(s), target = share_of(top_p, (double)whole + more);
        if (target <= whole) cut_all(s, step, x, r, 0, 1.0, target, true, l.total, vocab);
        return target <= whole;
    };
    constexpr double scale = 0x1p44;
    if (!cut(l.sum * scale)) return false;
    // The terms of the rest are off by 2^-22 (the exponential), 2^-24 (its second factor) and 3 2^-24 (sums of 8) of themselves, and by
    // 2^-24 |z| (a difference); the cut is certain where that does not reach the next entry.
    const double off = top_p * (l.sum * 0x1.4p-21 + l.slope * 0x1p-24) * scale;
    if ((double)s.cut.before < (double)s.cut.target - off && (double)s.cut.target + off <= (double)s.cut.mass) return true;
    // it is not: the rest as the list's entries are summed
    unsigned long long exact = 0;
    for (int i = threadIdx.x; i < x.n; i += kThreads)
        if ((float)x.v[i] < edge) exact += mass_of(r, (float)x.v[i]);
    return cut((double)sum_of_all(s, exact));
}

template <typename L, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) k_sample(const __grid_constant__ Params p) {
    using V = Vec<L>;
    constexpr int N = V::N;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ Shared s;
    const SparkSample& a = p.a;
    const int cs = (int)cluster_size(), rank = (int)cluster_rank(), tid = threadIdx.x;
    const int64_t row = blockIdx.x / cs, b = row / a.nodes, node = row - b * a.nodes;
    const int vocab = (int)a.vocab, v0 = rank * p.slice, n = max(0, min(p.slice, vocab - v0));
    const L* logits = reinterpret_cast<const L*>(a.logits) + b * a.logits_stride[0] + node * a.logits_stride[1] + v0;
    cluster_arrive();
    grid_wait();
    // (what is computed in 64 bits is computed by one thread: the unit for it is slow)
    const double temp = a.temperature ? (double)a.temperature[b] : a.temperature_all;
    const int64_t top_k = a.top_k ? (int64_t)a.top_k[b] : a.top_k_all;
    const double top_p = a.top_p ? (double)a.top_p[b] : a.top_p_all, min_p = a.min_p ? (double)a.min_p[b] : a.min_p_all;
    bool by_k = top_k > 0 && top_k < vocab, by_p = top_p < 1;
    if (tid == 0) {
        const double t = fmin(fmax(temp, 1e-30), 1e30);
        s.per_temp = 1.0 / t;
        // (a cut by count has nothing to do with the temperature)
        s.bins = (float)((kBins - 1) / (by_k ? fmax(32 * t, 32.0) : 32 * t));
        // e >= min_p, where exp's argument is (l - M) / T
        s.reach = min_p > 0 ? -fmin(log(min_p), 0.0) * t : INFINITY;
    }
    const float* noise = a.token ? a.noise + b * a.noise_stride + v0 : nullptr;
    if (noise && !by_k && !by_p && !(min_p > 0) && temp > 0 && tid == 0) to_l2(noise, (int64_t)n * 4);

    // the slice, in vectors that lie as they do in memory: `head` entries of the first one belong to another slice, or row
    const int head = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(L)), vectors = n ? (head + n + N - 1) / N : 0;
    uint4* const vec = reinterpret_cast<uint4*>(raw);
    const uint4* const from = reinterpret_cast<const uint4*>(logits - head);
    float most[kGroups];      // the largest of this thread's vectors, every fourth of them
#pragma unroll
    for (int k = 0; k < kGroups; ++k) most[k] = -INFINITY;
    for (int i0 = tid; i0 < vectors; i0 += kGroups * kThreads) {
        V x[kGroups];
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
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
        for (int k = 0; k < kGroups; ++k) {
            const int i = i0 + k * kThreads;
            if (i >= vectors) continue;
            vec[i] = x[k].raw;
            const float m = x[k].largest();
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(most[k]) : "f"(m));
        }
    }
    Slice<L> x{reinterpret_cast<const L*>(raw) + head, v0, n, nullptr, 0, 0, head};
    __syncwarp();
    cluster_wait();      // every CTA of the cluster has started: its shared memory may be written
    int step = 0;
    Note best{-INFINITY, 0, 0};
#pragma unroll
    for (int k = 0; k < kGroups; ++k) best.a = fmaxf(best.a, most[k]), best.b += most[k] == most[k] ? 0 : 1;
    best = join_all(s, step, best);
    Row r;
    r.top = best.a;
    const bool none_here = best.b != 0 || !(best.a > -INFINITY && best.a < INFINITY) || !(temp >= 0);
    const bool greedy = !none_here && temp == 0;
    r.per_temp = s.per_temp, r.bins = s.bins;
    const float per2 = (float)(r.per_temp * 1.4426950408889634);   // (exponents of 2)
    by_k = by_k && !none_here && !greedy, by_p = by_p && !none_here && !greedy;
    float limit = -INFINITY;      // what stays: above this, or equal with an index up to `last`
    int last = 0x7fffffff;
    if (greedy) {
        Note first = none();
        x.each([&](float f, int index) {
            if (f == r.top) add(first, f, index);
        });
        limit = r.top, last = join_all(s, step, first).i;
    } else if (by_k || by_p) {
        // the bin by which there are enough entries, from the groups' largest
        for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0;
        if (tid == 0) s.listed[0] = s.listed[1] = s.pairs = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            const int bin = bin_of(r, most[k]);
            if (bin < kBins - 1) atomicAdd(&s.count[bin], 1u);
        }
        add_bins(s, false);
        unsigned enough = (unsigned)top_k, more = 0;
        if (!by_k) {
            // Groups of m entries each, of which a share of 1 - (1 - q)^m has one of the largest q.  A thirtieth, and if that has less mass
            // than stays as many as the lists hold (some rows in 64 of 32,000, whose call took 53 us without, 19 otherwise).
            const float groups = fminf((float)(cs * kGroups * kThreads), (float)vocab / N), m = (float)vocab / groups;
            const float most_listed = fminf(0.75f * kList * cs / (float)vocab, 0.25f);
            enough = max(64u, (unsigned)(groups * (1.f - __expf(-0.0339f * m))));
            more = max(enough, (unsigned)(groups * (1.f - __expf(m * __logf(1.f - most_listed)))));
        }
        find_count(s, enough, more);
        const bool reached = !by_k || s.found.bin >= 0;
        // what has a bin up to that one (and, by the rounding of the edge, perhaps some more)
        // (-inf, which fills the vectors' ends too, is never among them: below the lowest number there is no edge)
        auto edge_of = [&](int bin) {
            return fmaxf(__fsub_rd(r.top, __fmul_ru(__fdiv_ru((float)((bin >= 0 ? bin : kBins - 2) + 1), r.bins), 1.00001f)), -FLT_MAX);
        };
        const float edge = edge_of(s.found.bin), further = edge_of(s.further);
        unsigned groups = 0;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) groups |= reached && !(by_k && most[k] < edge) ? 1u << k : 0u;
        const Listed l = list_from(s, x, r, vec, vectors, groups, !by_k, per2, edge);
        bool done = false;
        const unsigned k = by_k ? (unsigned)top_k : 0;
        if (by_k) {
            done = reached && l.fits;
            if (done && l.total <= kPairs) solve(s, r, k, 0ull, top_p, 0.0, 0, 0);
            else if (done) cut_all(s, step, x, r, k, top_p, 0ull, false, l.total, vocab);
        } else if (l.fits) {
            done = cut_by_mass(s, step, x, r, l, top_p, vocab, edge);
            if (!done && further < edge) {
                __syncthreads();
                if (tid == 0) s.listed[0] = s.listed[1] = s.pairs = 0;
                cluster_sync();
                const Listed all = list_from(s, x, r, vec, vectors, (1u << kGroups) - 1, true, per2, further);
                done = all.fits && cut_by_mass(s, step, x, r, all, top_p, vocab, further);
            }
        }
        if (!done) {
            x.list = nullptr;
            unsigned long long target = 0;
            __syncthreads();
            if (!by_k) {
                histogram(s, x, r, Range{0, 0, 0, 0, 0, 0}, true);
                target = share_of(top_p, (double)mass_of_bins(s));
            }
            cut_all(s, step, x, r, k, top_p, target, !by_k, vocab, vocab);
        }
        limit = value_of(s.cut.key), last = s.cut.index;
    }
    if (min_p > 0 && !none_here && !greedy) {
        const float least = fminf(__double2float_ru((double)r.top - s.reach), r.top);
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
        // (e to 2^-22 and 3 2^-24 |z|, the quotient to 2 units more; a list's order is the atomics', so its sum is in integers)
        got.a = 0.f;
        if (x.list) {
            x.each([&](float f, int index) {
                if (!stays(f, index)) return;
                const float q = exp2_of((f - r.top) * per2), chance = __fdividef(q, noise[index - v0]);
                got.b += __float2ull_rn(q * 0x1p44f);
                if (chance > got.a || (chance == got.a && index < got.i)) got.a = chance, got.i = index;
            });
        } else {
            constexpr int kAhead = 8;
            const bool all = limit == -INFINITY;
            // Multiples of 2^-44, as a list's (a conversion of each to 64 bits takes longer): those of 2^-22 are the mantissa beside 2,
            // those of the rest beside 3.
            static_assert(kRowBytes / 2 / kThreads + kAhead < 1024, "a thread's multiples of 2^-22 fit 32 bits");
            unsigned whole = 0, rest = 0, terms = 0;
            for (int i0 = tid; i0 < n; i0 += kAhead * kThreads) {
                float f[kAhead], e[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int i = i0 + k * kThreads;
                    f[k] = i < n ? (float)x.v[i] : -INFINITY;
                    if (!all && !stays(f[k], v0 + i)) f[k] = -INFINITY;
                    e[k] = f[k] > -INFINITY ? noise[i] : 1.f;
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const float q = f[k] = exp2_of((f[k] - r.top) * per2), chance = __fdividef(q, e[k]);
                    if (chance > got.a) got.a = chance, got.i = v0 + i0 + k * kThreads;
                }
                if (!a.logprob) continue;
                terms += kAhead;
#pragma unroll
                for (int k = 0; k < kAhead; k += 2) {
                    const Two q = two(f[k], f[k + 1]), near = add(q, two(2.f, 2.f)), far = fma(add(near, two(-2.f, -2.f)), two(-1.f, -1.f), q);
                    add_bits(whole, near), add_bits(rest, fma(far, two(0x1p22f, 0x1p22f), two(3.f, 3.f)));
                }
            }
            whole -= terms * 0x40000000u, rest -= terms * 0x40400000u;
            got.b = ((unsigned long long)whole << 22) + (long long)(int)rest;
        }
        got = join_all(s, step, got);
        if (got.i < 0) {
            // no chance above 0 (variates of infinity): all that stay tie
            Note first = none();
            x.each([&](float f, int index) {
                if (f > -INFINITY && stays(f, index)) add(first, 0.f, index);
            });
            got.i = join_all(s, step, first).i;
        }
    } else if (greedy) {
        got.i = last;
    }
    // the owner of the token knows its logit
    if (a.logprob && !none_here && !greedy && got.i >= v0 && got.i < v0 + n && tid == 0)
        a.logprob[b] = (float)(((double)(float)x.v[got.i - v0] - (double)r.top) * r.per_temp) - logf((float)((double)got.b * 0x1p-44));
    if (rank == 0 && tid == 0) {
        a.token[b] = got.i;
        if (a.logprob && (got.i < 0 || greedy)) a.logprob[b] = got.i < 0 ? NAN : 0.f;
    }
}


inline int64_t slice_of(int64_t vocab, int cs) { return ((vocab + cs - 1) / cs + 15) / 16 * 16; }

template <typename L, int CTAS>
int launch(const Params& p, int64_t rows, int cs, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(k_sample<L, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowBytes + 16);
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
    e = cudaLaunchKernelEx(&cfg, k_sample<L, CTAS>, p);
    if (e != cudaSuccess) return set_error((int)e, "spark_sample: launch failed: %s", cudaGetErrorString(e));
    return check_launch("spark_sample");
}
template <typename L>
int launch(Params& p, int64_t rows, int sms, cudaStream_t s) {
    // A CTA takes a row, a cluster one that does not fit, or a long one where SMs are left over.  Measured, us a call of sample without
    // a cut / with top_k 50 / with top_p 0.95:
    //   one row of 90,000 in bf16, by 1 / 4 / 8 CTAs: 18.6, 14.0, 30; 8.5, 11.8, 20; 6.3, 11.2, 18.  Of 32,000 by 1 / 8: 8.6, 9.4, 17;
    //   4.9, 10.8, 17.  36 of 50,000 in fp32 by 1 / 4 / 8 (more CTAs than SMs): 14.1, 14.5, 27; 10.4, 13.5, 25; 12.8, 23.7, 41.
    //   300 of 151,936 in bf16 by 2 / 4, which share an SM with others: 130, 83, 178; 99, 80, 163.  64 of 65,000 by 1 / 4: 14.7, 12.4,
    //   24; 10.8, 13.3, 39.
    // Clusters of 4 take long rows as long as all are there at once, two CTAs an SM: up to seven eighths of the SMs' places (they do not find
    // all); shorter ones up to half of that.  64 rows of 100,003 in bf16 by 1 / 4: 21.1, 14.4, 35 (85 with a border left open); 14.8, 14.8,
    // 32 (48).  65 of them the same; 80: 21.6, 13.9, 35; 22.4, 27.9, 51 (the last clusters come second); 148: 32.3, 14.4, 37; 40.7, 41.2, 80.
    int cs = slice_of(p.a.vocab, 1) * sizeof(L) <= kRowBytes ? 1 : slice_of(p.a.vocab, 4) * sizeof(L) <= kRowBytes ? 4 : 8;
    const int64_t bytes_row = p.a.vocab * (int64_t)sizeof(L);
    if (bytes_row >= kLongBytes) cs = 16 * rows <= sms ? 8 : (bytes_row >= 160 * 1024 ? 16 : 32) * rows <= 7 * sms ? std::max(cs, 4) : cs;
    p.slice = (int)slice_of(p.a.vocab, cs);
    // Two CTAs share an SM (64 registers a thread) where there are more than SMs and both fit, else one has it alone (128): 256 rows of
    // 32,000 in bf16 27.4 / 29.0 us, 8 of them in fp32 17.2 / 15.7, 64 of 100,003 34.8 / 33.4.  Clusters do not find all SMs: 36 rows
    // of 90,000 by 4 with an SM each 39.9 us, sharing SMs 30.0; 30 of 151,936 27.2 and 36.7.
    const size_t bytes = sizeof(Shared) + p.slice * sizeof(L) + 16 + 1024;
    const bool more = cs > 1 ? 8 * rows * cs > 7 * sms : rows > sms;
    return more && 2 * bytes <= kSmemSm ? launch<L, 2>(p, rows, cs, s) : launch<L, 1>(p, rows, cs, s);
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
        auto rows = [&](const void* at, const int64_t* stride) {
            return Rows{at, a->dtype == SPARK_DTYPE_F32 ? 4 : 2, a->vocab, 2, {a->batch, a->nodes}, {stride[0], stride[1]}};
        };
        const Rows out = rows(a->out, a->out_stride), in = rows(a->logits, a->logits_stride);
        bool same = true;
        for (int i = 0; i < 2; ++i) same = same && (out.extent[i] == 1 || out.stride[i] == in.stride[i]);
        SPARK_REQUIRE(rows_apart(out), SPARK_ERR_INVALID, "spark_sample: output rows in one place");
        SPARK_REQUIRE(a->out != a->logits || same, SPARK_ERR_INVALID, "spark_sample: in place needs equal strides");
        SPARK_REQUIRE(a->out == a->logits || !rows_meet(out, in), SPARK_ERR_INVALID, "spark_sample: the output overlaps the logits");
    }
    Params p;
    p.a = *a;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return set_error((int)e, "spark_sample: %s", cudaGetErrorString(e));
    const int64_t rows = a->batch * a->nodes;
    const int sms = tc::sm_count_cached(dev);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == SPARK_DTYPE_BF16) return launch<__nv_bfloat16>(p, rows, sms, st);
    if (a->dtype == SPARK_DTYPE_F16) return launch<__half>(p, rows, sms, st);
    return launch<float>(p, rows, sms, st);
}

}  // extern "C"
