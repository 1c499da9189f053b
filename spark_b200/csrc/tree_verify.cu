// tree_verify.cu -- verification of a drafted tree by rejection sampling.
//
// At node cur the target's distribution is r = softmax(logits[cur] / T).  A
// child drafted with probability q(x) is accepted when u q(x) < r(x); else
// r <- max(r - q, 0) / sum max(r - q, 0), which makes the accepted tokens
// samples of the target.  The last token is argmax_v r(v) / e(v): with
// exponential variates e(v) the index of the smallest e(v) / r(v) is v with
// probability proportional to r(v).
//
// One thread-block cluster of 8 CTAs (fewer where there are many sequences) per
// sequence, each CTA a contiguous slice of the
// vocabulary that it keeps in shared memory, so that a row is read from memory
// once.  The walk is a chain of row passes, its bound their latency (about 2 us
// each): one reduction in the CTA, one exchange of partial sums through
// distributed shared memory with one cluster barrier; all CTAs add them in rank
// order and so take the same decisions.  r at a single token needs no exchange:
// every CTA computes it from the token's logit and the sums.  Without draft
// probabilities a rejection needs no pass either, it takes one exponential out
// of the sum, unless a sixteenth or less is left of that.  Rows of nodes that the
// walk does not reach are not read, but for the row of the first child, which is
// brought into L2 while its parent's is worked on, as the noise is from the start.
// Measured: a chain of 8 nodes over
// 32000 entries 15 us (3.4 us a node: 1.2 the row's loads, 1.2 the join, 0.3 the
// exponentials), 64 trees of 16 nodes over 100003 entries 45 us
// (47 without the next entries' loads during the work on the last).  256 or 1024
// threads a CTA were 5 to 40% slower; three or four CTAs to an SM, which takes
// spilled registers, 7 to 35% for few sequences and no faster for many.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace spark {
namespace tc {
int sm_count_cached(int dev);
}

namespace tv {

constexpr int kThreads = 512;
constexpr int kMaxCluster = 8;
constexpr int kMaxNodes = 1024;
constexpr int kSliceMax = 52 * 1024;   // values in a CTA's shared memory (208 KB)
constexpr int kBatch = 8;              // loads of a thread on the way together

constexpr int kSmemSm = 228 * 1024;    // shared memory of an SM

// Vocabulary entries of each of cs CTAs.
inline int64_t slice_of(int64_t vocab, int cs) { return ((vocab + cs - 1) / cs + 7) / 8 * 8; }

struct Params {
    SparkTreeVerify a;
    int slice;   // vocabulary entries of a CTA
    int* err;
};

// What a CTA tells the others after a pass.
struct Note {
    float a, b;
    int i, pad;
};

struct Shared {
    Note note[2][kMaxCluster];
    Note red[kThreads / 32];
    float mass[kMaxNodes];   // sums of what was left after each rejection at this node, 0 where nothing was
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
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
// Asks for bytes [p, p + n) in L2.
__device__ __forceinline__ void to_l2(const void* p, int64_t n) {
    const uintptr_t a = (reinterpret_cast<uintptr_t>(p) + 15) & ~uintptr_t(15);
    const int64_t m = (reinterpret_cast<intptr_t>(p) + n - (intptr_t)a) & ~int64_t(15);
    if (m > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a), "r"((uint32_t)m) : "memory");
}

// Integers in the order of the floats (no NaN), and back.
__device__ __forceinline__ int ordered(float x) {
    const int i = __float_as_int(x);
    return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
__device__ __forceinline__ float max_of_warp(float x) { return unordered(__reduce_max_sync(0xffffffffu, ordered(x))); }
// (both lanes of a pair compute the same: an addition commutes)
__device__ __forceinline__ float sum_of_warp(float x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// How the notes of a warp's lanes become one.
// Largest value a with its lowest index i (-1 where there is none); b: any.
struct Best {
    static __device__ Note none() { return Note{-INFINITY, 0.f, -1, 0}; }
    static __device__ Note warp(Note v) {
        const float top = max_of_warp(v.i < 0 ? -INFINITY : v.a);
        const uint32_t first = __reduce_min_sync(0xffffffffu, v.i >= 0 && v.a == top ? (uint32_t)v.i : 0xffffffffu);
        return Note{top, __any_sync(0xffffffffu, v.b != 0.f) ? 1.f : 0.f, (int)first, 0};
    }
    static __device__ void add(Note& v, float a, int i) {
        if (v.i < 0 || a > v.a) v.a = a, v.i = i;     // indexes come in increasing order
    }
};
// Maximum a and the sum b of exponentials over it.
struct Softmax {
    static __device__ Note none() { return Note{-INFINITY, 0.f, 0, 0}; }
    static __device__ Note warp(Note v) {
        const float top = max_of_warp(v.a);
        return Note{top, sum_of_warp(v.b * expf(v.a - (top == -INFINITY ? 0.f : top))), 0, 0};
    }
};
struct Sum {
    static __device__ Note none() { return Note{0.f, 0.f, 0, 0}; }
    static __device__ Note warp(Note v) { return Note{sum_of_warp(v.a), 0.f, 0, 0}; }
};

// Joins the notes of all threads of the cluster; every thread gets the result.
// The order is fixed: by lanes, warps and CTAs.
template <typename J>
__device__ __forceinline__ Note join_all(Shared& s, int& step, Note v) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = (int)cluster_size();
    v = J::warp(v);
    if (lane == 0) s.red[warp] = v;
    __syncthreads();
    Note* slot = s.note[step & 1];
    if (step == 0) cluster_wait();     // every CTA of the cluster has started: its shared memory may be written
    ++step;
    if (warp == 0) {
        v = J::warp(lane < kThreads / 32 ? s.red[lane] : J::none());
        if (lane < n) {
            const uint32_t local = (uint32_t)__cvta_generic_to_shared(&slot[cluster_rank()]);
            uint32_t remote;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(lane));
            asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "r"(__float_as_uint(v.a)),
                         "r"(__float_as_uint(v.b)), "r"(v.i), "r"(0)
                         : "memory");
        }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    return J::warp(lane < n ? slot[lane] : J::none());
}

template <typename L, typename D>   // types of logits and draft probabilities
__global__ void __launch_bounds__(kThreads, 2) k_tree_verify(const __grid_constant__ Params p) {
    extern __shared__ float raw[];   // logits over T, after a rejection with draft probabilities r; below zero: nothing is left of -raw
    __shared__ Shared s;
    const SparkTreeVerify& a = p.a;
    const uint32_t rank = cluster_rank();
    const int64_t b = blockIdx.x / cluster_size();
    const int nodes = (int)a.nodes, tid = threadIdx.x, lane = tid & 31;
    const int64_t v0 = (int64_t)rank * p.slice;
    const int n = (int)max((int64_t)0, min((int64_t)p.slice, a.vocab - v0));
    // the tree, in shared memory after the slice: from here on a child costs no round trip but for its logit
    int* parents = reinterpret_cast<int*>(raw + p.slice);
    int* tokens = parents + nodes;        // -1: outside the vocabulary
    float* uniforms = reinterpret_cast<float*>(tokens + nodes);
    const float* noise = a.noise + b * a.noise_stride + v0;
    const L* logits = reinterpret_cast<const L*>(a.logits) + b * a.logits_stride[0];
    const D* draft = a.draft ? reinterpret_cast<const D*>(a.draft) + b * a.draft_stride[0] : nullptr;
    grid_wait();
    const float temp = a.temperature ? a.temperature[b] : 1.f;
    // Logits are multiplied by 1 / T: half a unit in the last place more than a division, which took a fifth of the time
    // (64 trees over 100003 entries 58 us).  1 / T stays between 2^-126 and 2^100: an infinite T gives equal chances to
    // all entries above -inf, a T that is all but 0 the argmax, and logits up to 2^27 do not overflow.
    const float per_temp = temp != temp ? temp : copysignf(fminf(fmaxf(1.f / fabsf(temp), FLT_MIN), 0x1p100f), temp);
    const bool lead = rank == 0 && tid == 0;
    int step = 0, cur = 0, accepted = 1;
    int64_t last = -1;
    cluster_arrive();
    if (lead) a.path[b * nodes] = 0;
    if (tid == 0 && temp != 0.f) to_l2(noise, (int64_t)n * 4);
    if (tid == 0) to_l2(logits + v0, (int64_t)n * sizeof(L));
    for (int i = tid; i < nodes; i += kThreads) {
        const int64_t x = a.tokens[b * a.tokens_stride + i];
        parents[i] = a.parents[b * a.parents_stride + i];
        tokens[i] = x >= 0 && x < a.vocab ? (int)x : -1;
        uniforms[i] = a.uniforms[b * a.uniforms_stride + i];
    }
    __syncthreads();

    while (true) {
        const L* row = logits + cur * a.logits_stride[1];
        const D* q_row = draft ? draft + cur * a.draft_stride[1] : nullptr;
        // The children in index order.  A lane has one of 32 nodes: logits and draft probabilities of all children among
        // them are on their way together, and during the pass.
        int base = cur + 1, child = -1, x = -1, xl;
        unsigned waiting;
        float lx = 0.f, qx = 1.f, lxl, qxl;
        auto gather = [&]() {
            const int c = base + lane;
            const bool is = c < nodes && parents[c] == cur;
            xl = is ? tokens[c] : -1;
            lxl = xl >= 0 ? (float)row[xl] : 0.f, qxl = xl >= 0 && draft ? (float)q_row[xl] : 1.f;
            waiting = __ballot_sync(0xffffffffu, is);
        };
        auto next = [&]() {
            while (!waiting) {
                base += 32;
                if (base >= nodes) {
                    child = -1;
                    return;
                }
                gather();
            }
            const int at = __ffs(waiting) - 1;
            waiting &= waiting - 1;
            child = base + at;
            x = __shfl_sync(0xffffffffu, xl, at), lx = __shfl_sync(0xffffffffu, lxl, at), qx = __shfl_sync(0xffffffffu, qxl, at);
        };
        gather();
        next();
        if (child >= 0 && tid == 0) to_l2(logits + child * a.logits_stride[1] + v0, (int64_t)n * sizeof(L));
        if (child >= 0 && draft && tid == 32) to_l2(q_row + v0, (int64_t)n * sizeof(D));
        // one pass: running maximum m and sum z of exponentials over it (a NaN stays in z), or the argmax
        float m = -INFINITY, z = 0.f;
        int at = -1;
        bool nan = false;
        const L none(temp < 0.f ? INFINITY : -INFINITY);   // over T -inf
        L ahead[kBatch];      // the next entries, on their way during the work on these
        auto load = [&](int i0) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int i = i0 + k * kThreads;
                ahead[k] = i < n ? row[v0 + i] : none;
            }
        };
        load(tid);
        for (int i0 = tid; i0 < n; i0 += kBatch * kThreads) {
            float l[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) l[k] = (float)ahead[k];
            load(i0 + kBatch * kThreads);
            if (temp == 0.f) {
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    nan |= l[k] != l[k];
                    if (l[k] > m) m = l[k], at = i0 + k * kThreads + (int)v0;
                }
                continue;
            }
            float most = m;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int i = i0 + k * kThreads;
                // (rounded alike wherever it is used: not fused with a subtraction)
                l[k] = __fmul_rn(l[k], per_temp);
                if (i < n) raw[i] = l[k];
                most = fmaxf(most, l[k]);
            }
            const float ref = most == -INFINITY ? 0.f : most;
            // (__expf(x) is off by up to 2 + 1.2 |x| units in its last place, the rounding of a scaled logit l makes
            // |l| / 2 of them in any case)
            z *= __expf(m - ref);
#pragma unroll
            for (int k = 0; k < kBatch; ++k) z += __expf(l[k] - ref);
            m = most;
        }
        if (temp == 0.f) {
            const Note got = join_all<Best>(s, step, Note{m, nan ? 1.f : 0.f, at, 0});
            if (got.b != 0.f || got.i < 0 || got.a == INFINITY) break;   // no distribution here
            while (child >= 0 && x != got.i) {
                if (x < 0 && lead) report_device_error(p.err, 11);
                next();
            }
            if (child < 0) {
                last = got.i;
                break;
            }
        } else {
            const Note got = join_all<Softmax>(s, step, Note{m, z, 0, 0});
            const float top = got.a;
            float sum = got.b, added = got.b;    // added: the sum as last added up, sum: that without the rejected ones
            if (!(sum > 0.f && sum < INFINITY)) break;   // no distribution here
            int rejected = 0;          // children whose rejection changed r; with draft probabilities raw is r then
            float f = 1.f;             // r = raw f
            // the children in turn
            while (child >= 0) {
                const bool valid = x >= 0;
                if (!valid && lead) report_device_error(p.err, 11);
                bool known = false;    // rejected already under another number
                if (valid && !draft) {
                    known = __any_sync(0xffffffffu, base + lane < child && xl == x);
                    for (int c = cur + 1 + lane; c - lane < base; c += 32)
                        known |= __any_sync(0xffffffffu, parents[c] == cur && tokens[c] == x);
                }
                if (valid && !known) {
                    const float e = expf(__fmul_rn(lx, per_temp) - top);
                    float rx = e / sum;
                    for (int k = 0; k < rejected && draft; ++k)
                        if (s.mass[k] > 0.f) rx = fmaxf(rx - qx, 0.f) / s.mass[k];
                    if (uniforms[child] * qx < rx) break;
                    if (!draft) {
                        // without x: its exponential leaves the sum, its owner forgets it.  The difference is as good as
                        // 2^-24 of what was added up: where a sixteenth of that or less is left, it is added up anew.
                        const int64_t i = (int64_t)x - v0;
                        const bool owner = i >= 0 && i < n && i % kThreads == tid;
                        if (owner) raw[i] = -INFINITY;
                        float rest = sum - e;
                        if (rest <= added * 0.0625f) {
                            rest = 0.f;
                            for (int k = tid; k < n; k += kThreads) rest += expf(raw[k] - top);
                            rest = join_all<Sum>(s, step, Note{rest, 0.f, 0, 0}).a;
                            if (rest > 0.f) added = rest;
                        }
                        if (rest > 0.f) sum = rest;
                        else if (owner) raw[i] = __fmul_rn(lx, per_temp);    // nothing is left: it stays what it was
                    } else {
                        float left = 0.f;
                        for (int i0 = tid; i0 < n; i0 += kBatch * kThreads) {
                            float q[kBatch];
#pragma unroll
                            for (int k = 0; k < kBatch; ++k) {
                                const int i = i0 + k * kThreads;
                                q[k] = i < n ? (float)q_row[v0 + i] : 0.f;
                            }
#pragma unroll
                            for (int k = 0; k < kBatch; ++k) {
                                const int i = i0 + k * kThreads;
                                if (i >= n) break;
                                const float old = rejected ? fmaxf(raw[i], 0.f) * f : expf(raw[i] - top) / sum;
                                const float t = fmaxf(old - q[k], 0.f);
                                raw[i] = t > 0.f ? t : -old;
                                left += t;
                            }
                        }
                        const float mass = join_all<Sum>(s, step, Note{left, 0.f, 0, 0}).a;
                        if (mass > 0.f) {
                            f = 1.f / mass;
                        } else {
                            // nothing is left: the distribution stays what it was
                            for (int i = tid; i < n; i += kThreads) raw[i] = -raw[i];
                            f = 1.f;
                        }
                        if (tid == 0) s.mass[rejected] = mass;
                        __syncthreads();
                        ++rejected;
                    }
                }
                next();
            }
            if (child < 0) {
                Note best = Best::none();
                for (int i0 = tid; i0 < n; i0 += kBatch * kThreads) {
                    float e[kBatch];
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        const int i = i0 + k * kThreads;
                        e[k] = i < n ? noise[i] : 1.f;
                    }
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        const int i = i0 + k * kThreads;
                        if (i >= n) break;
                        // (a common factor of r does not change which quotient is the largest; the quotient is good
                        // to two units in its last place)
                        const float r = rejected ? raw[i] : __expf(raw[i] - top);
                        if (r > 0.f) Best::add(best, __fdividef(r, e[k]), i + (int)v0);
                    }
                }
                last = join_all<Best>(s, step, best).i;
                break;
            }
        }
        if (lead) a.path[b * nodes + accepted] = child;
        ++accepted;
        cur = child;
    }
    if (rank == 0) {
        for (int i = accepted + tid; i < nodes; i += kThreads) a.path[b * nodes + i] = -1;
        if (tid == 0) a.accepted[b] = accepted, a.next[b] = last;
    }
}

template <typename L, typename D>
int launch(const Params& p, int64_t batch, int cs, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(k_tree_verify<L, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)((kSliceMax + 3 * kMaxNodes) * sizeof(float)));
    if (e != cudaSuccess) return set_error((int)e, "spark_tree_verify: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(batch * cs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = ((size_t)p.slice + 3 * (size_t)p.a.nodes) * sizeof(float);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, k_tree_verify<L, D>, p);
    if (e != cudaSuccess) return set_error((int)e, "spark_tree_verify: launch failed: %s", cudaGetErrorString(e));
    return check_launch("spark_tree_verify");
}

template <typename L>
int launch(const Params& p, int64_t batch, int cs, cudaStream_t s) {
    if (p.a.draft && p.a.draft_dtype == SPARK_DTYPE_BF16) return launch<L, __nv_bfloat16>(p, batch, cs, s);
    if (p.a.draft && p.a.draft_dtype == SPARK_DTYPE_F16) return launch<L, __half>(p, batch, cs, s);
    return launch<L, float>(p, batch, cs, s);
}

// CTAs of a cluster.  When the sequences' clusters do not fit the GPU at once they run one after another; smaller
// clusters then have more at work, each with longer rows, fewer barriers and less waiting.  The time goes with (sequences
// at a time, at least one filling) x (a pass's fixed part + a thread's share of the row), the fixed part worth 8 entries a
// thread.  Measured with 8 / 4 / 2 / 1 CTAs, sampled drafts: 32 trees of 8 nodes over 32000 entries 19 / 24 / 33 / 52 us, 64
// 36 / 29 / 40 / 60, 128 64 / 47 / 49 / 67, 512 225 / 144 / 117 / 155; over 100003 entries (2 at least) 64 64 / 64 / 89, 128
// 112 / 107 / 143, 512 387 / 303 / 390; over 1000 entries 128 47 / 26 / 16 / 15, 512 169 / 84 / 47 / 28.
int cluster_ctas(int64_t batch, int64_t vocab, int64_t nodes, int sms) {
    int best = kMaxCluster;
    double least = 0;
    for (int cs = kMaxCluster; cs >= 1; cs /= 2) {
        const int64_t slice = slice_of(vocab, cs);
        if (slice > kSliceMax) break;
        const size_t bytes = sizeof(Shared) + (slice + 3 * nodes) * sizeof(float) + 1024;
        const double at_once = (double)sms * (2 * bytes <= kSmemSm ? 2 : 1) / cs;
        const double time = std::max(1.0, batch / at_once) * (8 * kThreads + slice);
        if (cs == kMaxCluster || time < least) best = cs, least = time;
    }
    return best;
}

}  // namespace tv
}  // namespace spark

extern "C" {

int spark_tree_verify(const SparkTreeVerify* a, int* err, void* stream) {
    using namespace spark;
    using namespace spark::tv;
    SPARK_REQUIRE(a, SPARK_ERR_INVALID, "spark_tree_verify: null pointer");
    SPARK_REQUIRE(a->batch >= 0 && a->batch < (1 << 24) && a->nodes >= 1 &&  a->vocab >= 1,
                  SPARK_ERR_INVALID, "spark_tree_verify: bad size");
    SPARK_REQUIRE(a->nodes <= kMaxNodes, SPARK_ERR_UNSUPPORTED, "spark_tree_verify: %lld nodes, at most %d",
                  (long long)a->nodes, kMaxNodes);
    SPARK_REQUIRE(a->logits_dtype >= 0 && a->logits_dtype <= 2 && (!a->draft || (a->draft_dtype >= 0 && a->draft_dtype <= 2)),
                  SPARK_ERR_INVALID, "spark_tree_verify: bad dtype");
    SPARK_REQUIRE(a->vocab <= (int64_t)kMaxCluster * kSliceMax, SPARK_ERR_UNSUPPORTED,
                  "spark_tree_verify: a vocabulary of %lld entries is above %d", (long long)a->vocab,
                  kMaxCluster * kSliceMax);
    if (a->batch == 0) return SPARK_OK;
    SPARK_REQUIRE(a->logits && a->tokens && a->parents && a->uniforms && a->noise && a->path && a->accepted && a->next,
                  SPARK_ERR_INVALID, "spark_tree_verify: null pointer");
    Params p;
    p.a = *a;
    p.err = err;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return set_error((int)e, "spark_tree_verify: %s", cudaGetErrorString(e));
    const int cs = cluster_ctas(a->batch, a->vocab, a->nodes, tc::sm_count_cached(dev));
    p.slice = (int)slice_of(a->vocab, cs);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->logits_dtype == SPARK_DTYPE_BF16) return launch<__nv_bfloat16>(p, a->batch, cs, st);
    if (a->logits_dtype == SPARK_DTYPE_F16) return launch<__half>(p, a->batch, cs, st);
    return launch<float>(p, a->batch, cs, st);
}

}  // extern "C"
