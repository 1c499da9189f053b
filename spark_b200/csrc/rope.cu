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
// once for them, and eight loads are on the way together.  Where rotation, head,
// address or strides are no multiple of 16 bytes, the vectors are as long as they
// let them be (8, 4 or 2 bytes; a warp's accesses stay contiguous).  Measured:
// 32768 tokens of 40 heads of 128, forward and backward, 230 us (5.9 TB/s); 2048
// tokens of 64 heads of 128, 12.7 us (5.4 TB/s); eight heads a thread 17 us, two
// 15 us.
#include <string.h>

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

// N values in one access, as floats and back.
template <int BYTES>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };
__device__ __forceinline__ void put_one(float& to, float v) { to = v; }
__device__ __forceinline__ void put_one(__nv_bfloat16& to, float v) { to = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put_one(__half& to, float v) { to = __float2half_rn(v); }
template <typename T, int N>
struct Vec {
    using type = typename Raw<N * (int)sizeof(T)>::type;
    static __device__ void get(const type& v, float* f) {
        T t[N];
        memcpy(t, &v, sizeof(type));
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = (float)t[i];
    }
    static __device__ type put(const float* f) {
        T t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) put_one(t[i], f[i]);
        type v;
        memcpy(&v, t, sizeof(type));
        return v;
    }
    static __device__ type zero() {
        type v;
        memset(&v, 0, sizeof(type));
        return v;
    }
};

// units: places in a head that a thread may take -- the vectors of the turned part
// (half layout: of its first half), then those that are copied (none in place, where
// the first unit clears them if the position is bad).
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(256) k_rope_vec(const __grid_constant__ Params p, int units, int turned) {
    using V = Vec<T, N>;
    using R = typename V::type;
    constexpr int PAIRS = INTER ? N / 2 : N;
    grid_wait();
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
    R va[kHeads], vb[kHeads];
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
        va[k] = *reinterpret_cast<const R*>(x);
        if (!INTER && !copy) vb[k] = *reinterpret_cast<const R*>(x + half);
    }
    const bool good = pos >= 0 && pos < p.table_rows;
    if (!good && unit == 0) {
        if (h0 == 0) report_device_error(p.err, 8);
#pragma unroll
        for (int k = 0; k < kHeads; ++k)
            for (int e = p.rot; units == turned && y[k] && e < p.dim; e += N) *reinterpret_cast<R*>(y[k] + e) = V::zero();
    }
    float c[PAIRS], sn[PAIRS];
    if (!copy) {
        const float* row = p.table + (good ? pos : 0) * p.rot + (INTER ? d / 2 : d);
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) c[k] = row[k], sn[k] = p.inverse ? -row[half + k] : row[half + k];
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
        if (!y[k]) continue;
        const R zero = V::zero();
        if (copy) {
            *reinterpret_cast<R*>(y[k]) = good ? va[k] : zero;
            continue;
        }
        float u[N], w[N];
        V::get(va[k], u);
        if (INTER) {
#pragma unroll
            for (int e = 0; e < N; e += 2) turn(u[e], u[e + 1], c[e / 2], sn[e / 2], w[e], w[e + 1]);
            *reinterpret_cast<R*>(y[k]) = good ? V::put(w) : zero;
        } else {
            float v[N], z[N];
            V::get(vb[k], v);
#pragma unroll
            for (int e = 0; e < N; ++e) turn(u[e], v[e], c[e % PAIRS], sn[e % PAIRS], w[e], z[e]);
            *reinterpret_cast<R*>(y[k]) = good ? V::put(w) : zero;
            *reinterpret_cast<R*>(y[k] + half) = good ? V::put(z) : zero;
        }
    }
}

// What not even a pair's access fits (interleaved pairs at an odd address): a thread a pair.
__global__ void __launch_bounds__(256) k_rope(const __grid_constant__ Params p) {
    grid_wait();
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

template <typename T, int N>
void launch(const Params& p, unsigned grid, int units, int turned, cudaStream_t s) {
    if constexpr (N > 1) {
        if (p.interleaved) {
            launch_overlapped(k_rope_vec<T, N, true>, grid, 256, 0, s, p, units, turned);
            return;
        }
    }
    launch_overlapped(k_rope_vec<T, N, false>, grid, 256, 0, s, p, units, turned);
}
template <typename T>
void launch(const Params& p, int vec, unsigned grid, int units, int turned, cudaStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (vec == 8) return launch<T, 8>(p, grid, units, turned, s);
    if (vec == 4) return launch<T, 4>(p, grid, units, turned, s);
    if (vec == 2) return launch<T, 2>(p, grid, units, turned, s);
    launch<T, 1>(p, grid, units, turned, s);
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
        const int64_t extent[3] = {batch, tokens, s->heads};
        for (int i = 0; i < 3; ++i)
            SPARK_REQUIRE(extent[i] == 1 || s->ys[i] != 0, SPARK_ERR_INVALID, "spark_rope: output rows in one place");
        t.x = s->x, t.y = s->y, t.heads = (int)s->heads;
        for (int i = 0; i < 3; ++i) t.xs[i] = s->xs[i], t.ys[i] = s->ys[i];
    }
    p.tokens = tokens, p.n_tokens = batch * tokens;
    p.dim = head_dim, p.rot = rot_dim, p.dtype = dtype, p.interleaved = interleaved, p.inverse = inverse;
    p.pos_bytes = position_bytes, p.positions = positions, p.table = table, p.table_rows = table_rows, p.err = err;
    if (p.part[0].heads && p.part[1].heads)
        SPARK_REQUIRE(p.part[0].y != p.part[1].x && p.part[1].y != p.part[0].x && p.part[0].y != p.part[1].y, SPARK_ERR_INVALID,
                      "spark_rope: the output of one part is the other's input or output");
    const int64_t heads = p.part[0].heads + p.part[1].heads;
    if (heads == 0) return SPARK_OK;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    // the longest vectors that fit everything
    const int es = dtype == SPARK_DTYPE_F32 ? 4 : 2;
    int vec = 16 / es;
    bool in_place = true;
    auto fits = [&](int64_t v) { return v % vec == 0; };
    for (; vec > 1; vec /= 2) {
        bool ok = fits(head_dim) && fits(interleaved ? rot_dim : rot_dim / 2);
        for (const Part& t : p.part) {
            if (t.heads == 0) continue;
            ok = ok && aligned(t.x, (size_t)vec * es) && aligned(t.y, (size_t)vec * es);
            for (int i = 0; i < 3; ++i) ok = ok && fits(t.xs[i]) && fits(t.ys[i]);
        }
        if (ok) break;
    }
    for (const Part& t : p.part) in_place = in_place && (t.heads == 0 || t.x == t.y);
    if (vec > 1 || !interleaved) {
        const int turned = (interleaved ? rot_dim : rot_dim / 2) / vec, units = turned + (in_place ? 0 : (head_dim - rot_dim) / vec);
        const int64_t blocks = (p.n_tokens * ((heads + kHeads - 1) / kHeads) * units + 255) / 256;
        SPARK_REQUIRE(blocks < (1ll << 31), SPARK_ERR_UNSUPPORTED, "spark_rope: too many values for one call");
        const unsigned g = (unsigned)blocks;
        if (dtype == SPARK_DTYPE_F32) launch<float>(p, vec, g, units, turned, s);
        else if (dtype == SPARK_DTYPE_BF16) launch<__nv_bfloat16>(p, vec, g, units, turned, s);
        else launch<__half>(p, vec, g, units, turned, s);
        return check_launch("spark_rope");
    }
    const int64_t n = p.n_tokens * heads * (rot_dim / 2 + head_dim - rot_dim);
    const int grid = (int)std::min<int64_t>((n + 255) / 256, 148 * 16);
    launch_overlapped(k_rope, grid, 256, 0, s, p);
    return check_launch("spark_rope");
}

}  // extern "C"
