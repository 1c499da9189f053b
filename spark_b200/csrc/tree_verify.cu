// tree_verify.cu -- verification of a drafted tree by rejection sampling.
//
// At node cur the target's distribution is r = softmax(logits[cur] / T).  A
// child drafted with probability q(x) is accepted when u q(x) < r(x); else
// r <- max(r - q, 0) / sum max(r - q, 0), which makes the accepted tokens
// samples of the target.  The last token is argmax_v r(v) / e(v): with
// exponential variates e(v) the index of the smallest e(v) / r(v) is v with
// probability proportional to r(v).
//
// One thread-block cluster per sequence, each CTA a contiguous slice of the
// vocabulary whose r stays in shared memory, so that a row of logits is read
// once.  The walk is a chain of row passes; after each the CTAs exchange their
// partial sums through distributed shared memory (one cluster barrier) and add
// them in rank order, so all of them take the same decisions.  Rows of nodes
// that the walk does not reach are not read.
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace spark {
namespace tv {

constexpr int kThreads = 512;
constexpr int kMaxCluster = 8;
constexpr int kSliceMax = 52 * 1024;   // values of r in a CTA's shared memory (208 KB)

struct Params {
    SparkTreeVerify a;
    int slice;   // vocabulary entries of a CTA
    int* err;
};

// What a CTA tells the others after a pass.
struct Note {
    float a, b, c;
    int i;
};

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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

struct Shared {
    Note note[2][kMaxCluster];
    float red[kThreads / 32], red2[kThreads / 32];
    int redi[kThreads / 32];
    float x, x2;   // r at the next token tried, written by the thread that holds it
};

// Sends (a, b, c, i) to every CTA of the cluster and waits for theirs.
__device__ __forceinline__ const Note* exchange(Shared& s, int& step, Note mine) {
    Note* slot = s.note[step & 1];
    ++step;
    const uint32_t n = cluster_size();
    if (threadIdx.x < n) {
        uint32_t local = (uint32_t)__cvta_generic_to_shared(&slot[cluster_rank()]), remote;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(threadIdx.x));
        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "r"(__float_as_uint(mine.a)),
                     "r"(__float_as_uint(mine.b)), "r"(__float_as_uint(mine.c)), "r"(mine.i)
                     : "memory");
    }
    cluster_barrier();
    return slot;
}

__device__ __forceinline__ float block_sum(Shared& s, float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) t += s.red[w];
    return t;
}
__device__ __forceinline__ float block_max(Shared& s, float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = s.red[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) t = fmaxf(t, s.red[w]);
    return t;
}
// The largest value and its lowest index (-1 where there is none).
__device__ __forceinline__ void better(float& v, int& i, float v2, int i2) {
    if (i2 >= 0 && (i < 0 || v2 > v || (v2 == v && i2 < i))) v = v2, i = i2;
}
__device__ __forceinline__ void block_best(Shared& s, float& v, int& i) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float v2 = __shfl_xor_sync(0xffffffffu, v, o);
        const int i2 = __shfl_xor_sync(0xffffffffu, i, o);
        better(v, i, v2, i2);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red2[threadIdx.x >> 5] = v, s.redi[threadIdx.x >> 5] = i;
    __syncthreads();
    v = s.red2[0], i = s.redi[0];
    for (int w = 1; w < kThreads / 32; ++w) better(v, i, s.red2[w], s.redi[w]);
}

// The first child of `cur` after node `from`, or -1.
__device__ __forceinline__ int next_child(const int* parents, int nodes, int cur, int from) {
    const int lane = threadIdx.x & 31;
    for (int base = from + 1; base < nodes; base += 32) {
        const int c = base + lane;
        const unsigned hit = __ballot_sync(0xffffffffu, c < nodes && parents[c] == cur);
        if (hit) return base + __ffs(hit) - 1;
    }
    return -1;
}

__global__ void __launch_bounds__(kThreads) k_tree_verify(const __grid_constant__ Params p) {
    extern __shared__ float raw[];   // r of this slice up to the factor `f`; below zero: nothing left of -raw
    __shared__ Shared s;
    const SparkTreeVerify& a = p.a;
    const uint32_t rank = cluster_rank(), csize = cluster_size();
    const int64_t b = blockIdx.x / csize;
    const int nodes = (int)a.nodes, tid = threadIdx.x;
    const int64_t v0 = (int64_t)rank * p.slice;
    const int n = (int)max((int64_t)0, min((int64_t)p.slice, a.vocab - v0));
    const int* parents = a.parents + b * a.parents_stride;
    const int64_t* tokens = a.tokens + b * a.tokens_stride;
    const float* noise = a.noise + b * a.noise_stride + v0;
    const float temp = a.temperature ? a.temperature[b] : 1.f;
    const bool lead = rank == 0 && tid == 0;
    int step = 0, cur = 0, accepted = 1;
    int64_t last = -1;
    cluster_barrier();   // every CTA of the cluster has started: its shared memory may be written
    if (lead) a.path[b * nodes] = 0;

    while (true) {
        const int64_t row = b * a.logits_stride[0] + cur * a.logits_stride[1] + v0;
        int child = next_child(parents, nodes, cur, cur);
        if (temp == 0.f) {
            float best = -INFINITY;
            int at = -1;
            bool nan = false;
            for (int i = tid; i < n; i += kThreads) {
                const float x = load_as_float(a.logits, (int)a.logits_dtype, row + i);
                nan |= x != x;
                if (x > best) best = x, at = i + (int)v0;
            }
            nan = __syncthreads_or(nan);
            block_best(s, best, at);
            const Note* got = exchange(s, step, Note{best, nan ? 1.f : 0.f, 0.f, at});
            best = -INFINITY, at = -1;
            for (uint32_t r = 0; r < csize; ++r) better(best, at, got[r].a, got[r].i), nan |= got[r].b != 0.f;
            if (nan || at < 0 || best == INFINITY) break;
            while (child >= 0 && tokens[child] != at) child = next_child(parents, nodes, cur, child);
            if (child < 0) {
                last = at;
                break;
            }
        } else {
            // r(v) = raw(v) f: the maximum, then exponentials and their sum
            int64_t x = child >= 0 ? tokens[child] : -1;
            if (tid == 0) s.x = 0.f, s.x2 = 0.f;
            float m = -INFINITY, z = 0.f;
            for (int i = tid; i < n; i += kThreads) {
                const float v = load_as_float(a.logits, (int)a.logits_dtype, row + i) / temp;
                raw[i] = v;
                m = fmaxf(m, v);
            }
            m = block_max(s, m);
            for (int i = tid; i < n; i += kThreads) {
                const float e = m == -INFINITY && raw[i] == m ? 0.f : expf(raw[i] - m);
                raw[i] = e;
                z += e;
                if (v0 + i == x) s.x = e;
            }
            z = block_sum(s, z);
            const Note* got = exchange(s, step, Note{m, z, s.x, 0});
            float top = -INFINITY, sum = 0.f, rx = 0.f;
            for (uint32_t r = 0; r < csize; ++r) top = fmaxf(top, got[r].a);
            for (uint32_t r = 0; r < csize; ++r) {
                const float g = got[r].b == 0.f ? 0.f : expf(got[r].a - top);
                sum += got[r].b * g;
                rx += got[r].c * g;
            }
            if (!(sum > 0.f && sum < INFINITY)) break;   // no distribution here
            float f = m == -INFINITY ? 0.f : expf(m - top) / sum;
            rx /= sum;
            // the children in turn
            while (child >= 0) {
                const bool valid = x >= 0 && x < a.vocab;
                if (!valid && lead) report_device_error(p.err, 11);
                const int64_t dr = b * a.draft_stride[0] + cur * a.draft_stride[1];
                const float qx = !valid ? 0.f : a.draft ? load_as_float(a.draft, (int)a.draft_dtype, dr + x) : 1.f;
                if (valid && a.uniforms[b * a.uniforms_stride + child] * qx < rx) break;
                child = next_child(parents, nodes, cur, child);
                const int64_t x2 = child >= 0 ? tokens[child] : -1;
                __syncthreads();
                if (tid == 0) s.x = 0.f, s.x2 = 0.f;
                __syncthreads();
                float left = 0.f;
                for (int i = tid; i < n; i += kThreads) {
                    const float old = fmaxf(raw[i], 0.f) * f;
                    float t = old;
                    if (!valid) t = old;
                    else if (a.draft) t = fmaxf(old - load_as_float(a.draft, (int)a.draft_dtype, dr + v0 + i), 0.f);
                    else if (v0 + i == x) t = 0.f;
                    raw[i] = t > 0.f ? t : -old;
                    left += t;
                    if (v0 + i == x2) s.x = t, s.x2 = old;
                }
                left = block_sum(s, left);
                got = exchange(s, step, Note{left, s.x, s.x2, 0});
                float mass = 0.f, rn = 0.f, ro = 0.f;
                for (uint32_t r = 0; r < csize; ++r) mass += got[r].a, rn += got[r].b, ro += got[r].c;
                if (mass > 0.f) {
                    f = 1.f / mass;
                    rx = rn / mass;
                } else {
                    // nothing is left: the distribution stays what it was
                    for (int i = tid; i < n; i += kThreads) raw[i] = -raw[i];
                    f = 1.f;
                    rx = ro;
                }
                x = x2;
            }
            if (child < 0) {
                float best = -INFINITY;
                int at = -1;
                for (int i = tid; i < n; i += kThreads) {
                    const float r = fmaxf(raw[i], 0.f) * f;
                    if (r > 0.f) better(best, at, r / noise[i], i + (int)v0);
                }
                block_best(s, best, at);
                got = exchange(s, step, Note{best, 0.f, 0.f, at});
                best = -INFINITY, at = -1;
                for (uint32_t r = 0; r < csize; ++r) better(best, at, got[r].a, got[r].i);
                last = at;
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

}  // namespace tv
}  // namespace spark

extern "C" {

int spark_tree_verify(const SparkTreeVerify* a, int* err, void* stream) {
    using namespace spark;
    using namespace spark::tv;
    SPARK_REQUIRE(a, SPARK_ERR_INVALID, "spark_tree_verify: null pointer");
    SPARK_REQUIRE(a->batch >= 0 && a->batch < (1 << 24) && a->nodes >= 1 && a->nodes < (1 << 20) && a->vocab >= 1,
                  SPARK_ERR_INVALID, "spark_tree_verify: bad size");
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
    const int cs = kMaxCluster;
    p.slice = (int)((a->vocab + cs - 1) / cs + 7) / 8 * 8;
    const size_t smem = (size_t)p.slice * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(k_tree_verify, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(kSliceMax * sizeof(float)));
    if (e != cudaSuccess) return set_error((int)e, "spark_tree_verify: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a->batch * cs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, k_tree_verify, p);
    if (e != cudaSuccess) return set_error((int)e, "spark_tree_verify: launch failed: %s", cudaGetErrorString(e));
    return check_launch("spark_tree_verify");
}

}  // extern "C"
