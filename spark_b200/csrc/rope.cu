// rope.cu -- rotary positions of q and k.
//
// For pair i of a head at position p, with c = table[p, i] and
// s = table[p, r / 2 + i]:  (a, b) -> (a c - b s, b c + a s), the rotation of
// (a, b) by the pair's angle; its transpose, the backward pass, is s -> -s.
// Arithmetic is fp32, rounded once to the tensors' type.
//
// Its bound is HBM: every value is read and written once (6 flop a pair).  A
// thread of k_rope_vec turns the same 16 bytes (half layout: and their partners
// half a rotation away) of four heads of a token: cosines and sines are loaded
// once for them, and eight loads are on the way together.
#include <algorithm>

#include "common.cuh"

namespace spark {
namespace rope {

struct Part {
    const void* x;
    void* y;
    int heads;
    int64_t xs[3], ys[3];
};
struct Params {
    Part part[2];
    int64_t tokens, n_tokens;   // per sequence, in all
    int dim, rot, dtype, interleaved, inverse, pos_bytes;
    const void* positions;
    const float* table;
    int64_t table_rows;
    int* err;
};

// (a, b) turned; written with explicit roundings, so that the kernels agree bit by bit
__device__ __forceinline__ void turn(float a, float b, float c, float s, float& ya, float& yb) {
    ya = __fmaf_rn(a, c, -__fmul_rn(b, s));
    yb = __fmaf_rn(b, c, __fmul_rn(a, s));
}

constexpr int kHeads = 4;   // of one token, by one thread

// 16 bytes of values as floats and back
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int n = 4;
    static __device__ void get(const uint4& v, float* f) {
        f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
    static __device__ uint4 put(const float* f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int n = 8;
    static __device__ void get(const uint4& v, float* f) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    static __device__ uint4 put(const float* f) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct Vec<__half> {
    static constexpr int n = 8;
    static __device__ void get(const uint4& v, float* f) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = t.x, f[2 * i + 1] = t.y;
        }
    }
    static __device__ uint4 put(const float* f) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// units: places in a head that a thread may take -- the vectors of the turned part
// (half layout: of its first half), then those that are copied (none in place).
template <typename T, bool INTER>
__global__ void __launch_bounds__(256) k_rope_vec(const __grid_constant__ Params p, int units, int turned) {
    constexpr int N = Vec<T>::n, PAIRS = INTER ? N / 2 : N;
    const int heads = p.part[0].heads + p.part[1].heads, groups = (heads + kHeads - 1) / kHeads;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t rest = i / units, tok = rest / groups;
    if (tok >= p.n_tokens) return;
    const int unit = (int)(i - rest * units), h0 = (int)(rest - tok * groups) * kHeads;
    const int64_t b = tok / p.tokens, t = tok - b * p.tokens;
    const bool copy = unit >= turned;
    const int half = p.rot / 2, d = copy ? p.rot + (unit - turned) * N : unit * N;
    const int64_t pos = p.pos_bytes == 8 ? reinterpret_cast<const int64_t*>(p.positions)[tok]
                                         : reinterpret_cast<const int*>(p.positions)[tok];
    uint4 va[kHeads], vb[kHeads];
    T* y[kHeads];
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
        int h = h0 + k;
        y[k] = nullptr;
        if (h >= heads) continue;
        const int which = h >= p.part[0].heads;
        const Part& s = p.part[which];
        if (which) h -= p.part[0].heads;
        const T* x = reinterpret_cast<const T*>(s.x) + b * s.xs[0] + t * s.xs[1] + h * s.xs[2] + d;
        y[k] = reinterpret_cast<T*>(s.y) + b * s.ys[0] + t * s.ys[1] + h * s.ys[2] + d;
        va[k] = *reinterpret_cast<const uint4*>(x);
        if (!INTER && !copy) vb[k] = *reinterpret_cast<const uint4*>(x + half);
    }
    const bool good = pos >= 0 && pos < p.table_rows;
    if (!good && unit == 0 && h0 == 0) report_device_error(p.err, 8);
    float c[PAIRS], sn[PAIRS];
    if (!copy) {
        const float* row = p.table + (good ? pos : 0) * p.rot + (INTER ? d / 2 : d);
#pragma unroll
        for (int k = 0; k < PAIRS; k += 2) {
            const float2 cc = *reinterpret_cast<const float2*>(row + k), ss = *reinterpret_cast<const float2*>(row + half + k);
            c[k] = cc.x, c[k + 1] = cc.y;
            sn[k] = p.inverse ? -ss.x : ss.x, sn[k + 1] = p.inverse ? -ss.y : ss.y;
        }
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
        if (!y[k]) continue;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        if (copy) {
            *reinterpret_cast<uint4*>(y[k]) = good ? va[k] : zero;
            continue;
        }
        float u[N], w[N];
        Vec<T>::get(va[k], u);
        if (INTER) {
#pragma unroll
            for (int e = 0; e < N; e += 2) turn(u[e], u[e + 1], c[e / 2], sn[e / 2], w[e], w[e + 1]);
            *reinterpret_cast<uint4*>(y[k]) = good ? Vec<T>::put(w) : zero;
        } else {
            float v[N], z[N];
            Vec<T>::get(vb[k], v);
#pragma unroll
            for (int e = 0; e < N; ++e) turn(u[e], v[e], c[e % PAIRS], sn[e % PAIRS], w[e], z[e]);
            *reinterpret_cast<uint4*>(y[k]) = good ? Vec<T>::put(w) : zero;
            *reinterpret_cast<uint4*>(y[k] + half) = good ? Vec<T>::put(z) : zero;
        }
    }
}

// Heads whose size, address or strides no 16-byte access fits: a thread a pair.
__global__ void __launch_bounds__(256) k_rope(const __grid_constant__ Params p) {
    const int half = p.rot / 2, items = half + (p.dim - p.rot);   // pairs, then copied values
    const int heads = p.part[0].heads + p.part[1].heads;
    const int64_t n = p.n_tokens * heads * items;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int it = (int)(i % items);
        const int64_t th = i / items, tok = th / heads;
        int h = (int)(th % heads);
        const int which = h >= p.part[0].heads;
        if (which) h -= p.part[0].heads;
        const Part& t = p.part[which];
        const int64_t b = tok / p.tokens, s = tok % p.tokens;
        const int64_t xo = b * t.xs[0] + s * t.xs[1] + h * t.xs[2], yo = b * t.ys[0] + s * t.ys[1] + h * t.ys[2];
        const int64_t pos = p.pos_bytes == 8 ? reinterpret_cast<const int64_t*>(p.positions)[tok]
                                             : reinterpret_cast<const int*>(p.positions)[tok];
        const bool good = pos >= 0 && pos < p.table_rows;
        if (!good) report_device_error(p.err, 8);
        if (it >= half) {
            const int d = p.rot + it - half;
            store_from_float(t.y, p.dtype, yo + d, good ? load_as_float(t.x, p.dtype, xo + d) : 0.f);
            continue;
        }
        const int da = p.interleaved ? 2 * it : it, db = p.interleaved ? da + 1 : half + it;
        float c = 0.f, sn = 0.f;
        if (good) c = p.table[pos * p.rot + it], sn = p.table[pos * p.rot + half + it];
        if (p.inverse) sn = -sn;
        const float va = load_as_float(t.x, p.dtype, xo + da), vb = load_as_float(t.x, p.dtype, xo + db);
        float ya, yb;
        turn(va, vb, c, sn, ya, yb);
        store_from_float(t.y, p.dtype, yo + da, good ? ya : 0.f);
        store_from_float(t.y, p.dtype, yo + db, good ? yb : 0.f);
    }
}

}  // namespace rope
}  // namespace spark

extern "C" {

int spark_rope(const SparkRopeHeads* q, const SparkRopeHeads* k, int dtype, int64_t batch, int64_t tokens, int head_dim,
               int rot_dim, int interleaved, int inverse, const void* positions, int position_bytes,
               const float* table, int64_t table_rows, int* err, void* stream) {
    using namespace spark;
    using namespace spark::rope;
    SPARK_REQUIRE(q, SPARK_ERR_INVALID, "spark_rope: null pointer");
    SPARK_REQUIRE(dtype >= 0 && dtype <= 2, SPARK_ERR_INVALID, "spark_rope: bad dtype %d", dtype);
    SPARK_REQUIRE(position_bytes == 4 || position_bytes == 8, SPARK_ERR_INVALID,
                  "spark_rope: positions are 4- or 8-byte integers");
    SPARK_REQUIRE(batch >= 0 && tokens >= 0 && head_dim >= 1 && table_rows >= 1, SPARK_ERR_INVALID,
                  "spark_rope: bad size");
    SPARK_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= head_dim && head_dim <= (1 << 16), SPARK_ERR_INVALID,
                  "spark_rope: rot_dim %d is not an even number of 2..head_dim (%d)", rot_dim, head_dim);
    if (batch == 0 || tokens == 0) return SPARK_OK;
    SPARK_REQUIRE(positions && table, SPARK_ERR_INVALID, "spark_rope: null pointer");
    Params p;
    for (int w = 0; w < 2; ++w) {
        const SparkRopeHeads* s = w ? k : q;
        Part& t = p.part[w];
        t = Part{};
        if (!s || s->heads == 0) continue;
        SPARK_REQUIRE(s->x && s->y && s->heads >= 0 && s->heads < (1 << 24), SPARK_ERR_INVALID, "spark_rope: heads");
        bool same = true;
        for (int i = 0; i < 3; ++i) same = same && s->xs[i] == s->ys[i];
        SPARK_REQUIRE(s->x != s->y || same, SPARK_ERR_INVALID, "spark_rope: in place needs equal strides");
        t.x = s->x, t.y = s->y, t.heads = (int)s->heads;
        for (int i = 0; i < 3; ++i) t.xs[i] = s->xs[i], t.ys[i] = s->ys[i];
    }
    p.tokens = tokens, p.n_tokens = batch * tokens;
    p.dim = head_dim, p.rot = rot_dim, p.dtype = dtype, p.interleaved = interleaved, p.inverse = inverse;
    p.pos_bytes = position_bytes, p.positions = positions, p.table = table, p.table_rows = table_rows, p.err = err;
    const int64_t heads = p.part[0].heads + p.part[1].heads;
    if (heads == 0) return SPARK_OK;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int vec = dtype == SPARK_DTYPE_F32 ? 4 : 8;
    bool fits = head_dim % vec == 0 && (interleaved ? rot_dim : rot_dim / 2) % vec == 0 && aligned(table, 8);
    bool in_place = true;
    for (const Part& t : p.part) {
        if (t.heads == 0) continue;
        fits = fits && aligned(t.x, 16) && aligned(t.y, 16);
        for (int i = 0; i < 3; ++i) fits = fits && t.xs[i] % vec == 0 && t.ys[i] % vec == 0;
        in_place = in_place && t.x == t.y;
    }
    if (fits) {
        const int turned = (interleaved ? rot_dim : rot_dim / 2) / vec, units = turned + (in_place ? 0 : (head_dim - rot_dim) / vec);
        const int64_t blocks = (p.n_tokens * ((heads + kHeads - 1) / kHeads) * units + 255) / 256;
        SPARK_REQUIRE(blocks < (1ll << 31), SPARK_ERR_UNSUPPORTED, "spark_rope: too many values for one call");
        const unsigned g = (unsigned)blocks;
        if (dtype == SPARK_DTYPE_F32)
            interleaved ? k_rope_vec<float, true><<<g, 256, 0, s>>>(p, units, turned)
                        : k_rope_vec<float, false><<<g, 256, 0, s>>>(p, units, turned);
        else if (dtype == SPARK_DTYPE_BF16)
            interleaved ? k_rope_vec<__nv_bfloat16, true><<<g, 256, 0, s>>>(p, units, turned)
                        : k_rope_vec<__nv_bfloat16, false><<<g, 256, 0, s>>>(p, units, turned);
        else
            interleaved ? k_rope_vec<__half, true><<<g, 256, 0, s>>>(p, units, turned)
                        : k_rope_vec<__half, false><<<g, 256, 0, s>>>(p, units, turned);
        return check_launch("spark_rope");
    }
    const int64_t n = p.n_tokens * heads * (rot_dim / 2 + head_dim - rot_dim);
    const int grid = (int)std::min<int64_t>((n + 255) / 256, 148 * 16);
    k_rope<<<grid, 256, 0, s>>>(p);
    return check_launch("spark_rope");
}

}  // extern "C"
