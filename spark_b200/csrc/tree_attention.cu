// tree_attention.cu -- attention of a tree of drafted tokens over a paged K/V
// cache and over the tree itself.
//
// Node t sees the context (all lens[b] tokens of the cache), itself and its
// ancestors.  One pass over the keys with the running maximum m and sum l of
// the softmax: a new score s changes them to m' = max(m, s),
// l' = l e^(m - m') + e^(s - m'), and the accumulator likewise.  Scores, sums
// and accumulators are fp32.
#include <math.h>

#include "common.cuh"

namespace spark {
int check_cache(const SparkPagedCache* c, const char* who);

namespace ta {

constexpr int kWarps = 4;
constexpr int kPerLane = 8;   // head_dim <= 256

struct Params {
    SparkTreeAttention a;
    int* err;
};

// The node's ancestors and itself as a bit mask, 0 where the node is unused.
__device__ __forceinline__ uint64_t ancestors(const int* parents, int t) {
    uint64_t mask = 0;
    int n = t;
    while (true) {
        mask |= 1ull << n;
        const int up = parents[n];
        if (up == -1) return mask;
        if (up < 0 || up >= n) return 0;
        n = up;
    }
}

// One CTA per (sequence, node, query head); each warp takes every fourth key.
__global__ void __launch_bounds__(kWarps * 32) k_tree_attention(const __grid_constant__ Params p) {
    const SparkTreeAttention& a = p.a;
    const SparkPagedCache& c = a.cache;
    const int h = blockIdx.x, t = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t b = blockIdx.z;
    const int kvh = h / (int)(a.q_heads / c.kv_heads), dim = (int)c.head_dim, dt = (int)c.dtype;
    __shared__ float s_m[kWarps], s_l[kWarps], s_acc[kWarps][kPerLane * 32];
    const uint64_t mask = ancestors(a.parents + b * a.parents_stride, t);
    int64_t len = c.lens[b];
    const int64_t room = c.max_pages * c.page_size;
    bool bad = len < 0 || len > room;
    len = len < 0 ? 0 : (len > room ? room : len);
    if (mask == 0) len = 0;
    float q[kPerLane], acc[kPerLane], m = -INFINITY, l = 0.f;
    const int64_t qo = b * a.q_stride[0] + t * a.q_stride[1] + h * a.q_stride[2];
    const float scale = (float)(a.scale * 1.4426950408889634);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const int d = lane + 32 * i;
        q[i] = d < dim ? load_as_float(a.q, dt, qo + d) * scale : 0.f;
        acc[i] = 0.f;
    }
    for (int64_t n = warp; n < len + a.nodes; n += kWarps) {
        const void *kp, *vp;
        int64_t ko, vo;
        if (n < len) {
            const int64_t page = c.page_table[b * c.page_table_stride + n / c.page_size], r = n % c.page_size;
            if (page < 0 || page >= c.pages) {
                bad = true;
                continue;
            }
            kp = c.k, vp = c.v;
            ko = page * c.k_stride[0] + r * c.k_stride[1] + kvh * c.k_stride[2];
            vo = page * c.v_stride[0] + r * c.v_stride[1] + kvh * c.v_stride[2];
        } else {
            const int j = (int)(n - len);
            if (!((mask >> j) & 1)) continue;
            kp = a.k, vp = a.v;
            ko = b * a.kn_stride[0] + j * a.kn_stride[1] + kvh * a.kn_stride[2];
            vo = b * a.vn_stride[0] + j * a.vn_stride[1] + kvh * a.vn_stride[2];
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int d = lane + 32 * i;
            if (d < dim) s += q[i] * load_as_float(kp, dt, ko + d);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const float m2 = fmaxf(m, s), f = m == m2 ? 1.f : exp2f(m - m2), e = exp2f(s - m2);
        l = l * f + e;
        m = m2;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int d = lane + 32 * i;
            if (d < dim) acc[i] = acc[i] * f + e * load_as_float(vp, dt, vo + d);
        }
    }
    if (bad && lane == 0) report_device_error(p.err, 9);
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) s_acc[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
    for (int w = 0; w < kWarps; ++w) sum += s_l[w] == 0.f ? 0.f : s_l[w] * exp2f(s_m[w] - top);
    for (int d = threadIdx.x; d < dim; d += kWarps * 32) {
        float o = 0.f;
        for (int w = 0; w < kWarps; ++w) o += s_l[w] == 0.f ? 0.f : s_acc[w][d] * exp2f(s_m[w] - top);
        store_from_float(a.out, dt, b * a.out_stride[0] + t * a.out_stride[1] + h * a.out_stride[2] + d,
                         sum == 0.f ? 0.f : o / sum);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[(b * a.nodes + t) * a.q_heads + h] = sum == 0.f ? -INFINITY : (log2f(sum) + top) * 0.6931471805599453f;
}

int check(const SparkTreeAttention* a) {
    SPARK_REQUIRE(a, SPARK_ERR_INVALID, "spark_tree_attention: null pointer");
    const int rc = check_cache(&a->cache, "spark_tree_attention");
    if (rc) return rc;
    SPARK_REQUIRE(a->batch >= 0 && a->batch < 65536, SPARK_ERR_INVALID, "spark_tree_attention: at most 65535 sequences");
    SPARK_REQUIRE(a->nodes >= 1 && a->nodes <= SPARK_MAX_TREE_NODES, SPARK_ERR_INVALID,
                  "spark_tree_attention: 1 to %d nodes (got %lld)", SPARK_MAX_TREE_NODES, (long long)a->nodes);
    SPARK_REQUIRE(a->q_heads >= 1 && a->q_heads < (1 << 16) && a->q_heads % a->cache.kv_heads == 0, SPARK_ERR_INVALID,
                  "spark_tree_attention: %lld query heads are no multiple of %lld kv heads", (long long)a->q_heads,
                  (long long)a->cache.kv_heads);
    SPARK_REQUIRE(a->cache.dtype == SPARK_DTYPE_BF16 || a->cache.dtype == SPARK_DTYPE_F16, SPARK_ERR_UNSUPPORTED,
                  "spark_tree_attention: bf16 or f16");
    SPARK_REQUIRE(a->cache.head_dim % 8 == 0 && a->cache.head_dim <= 256, SPARK_ERR_UNSUPPORTED,
                  "spark_tree_attention: head_dim %lld is no multiple of 8 up to 256", (long long)a->cache.head_dim);
    return SPARK_OK;
}

}  // namespace ta
}  // namespace spark

extern "C" {

size_t spark_tree_attention_workspace_size(const SparkTreeAttention* a) {
    return spark::ta::check(a) == SPARK_OK ? 256 : 0;
}

int spark_tree_attention(const SparkTreeAttention* a, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace spark;
    using namespace spark::ta;
    const int rc = check(a);
    if (rc) return rc;
    if (a->batch == 0) return SPARK_OK;
    SPARK_REQUIRE(a->q && a->k && a->v && a->out && a->parents && a->cache.k && a->cache.v && a->cache.lens &&
                      (a->cache.page_table || a->cache.max_pages == 0),
                  SPARK_ERR_INVALID, "spark_tree_attention: null pointer");
    SPARK_REQUIRE(workspace && workspace_bytes >= 256, SPARK_ERR_WORKSPACE, "spark_tree_attention: workspace too small");
    Params p;
    p.a = *a;
    p.err = reinterpret_cast<int*>(workspace);
    k_tree_attention<<<dim3((unsigned)a->q_heads, (unsigned)a->nodes, (unsigned)a->batch), kWarps * 32, 0,
                       reinterpret_cast<cudaStream_t>(stream)>>>(p);
    return check_launch("spark_tree_attention");
}

}  // extern "C"
