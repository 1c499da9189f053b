// norm_rope.cu -- RMS norms of q and k for each head, with the rotary positions in
// the same pass, and its backward pass.
//
// For a head x of D values at position p, with the rotation R(p) of rope.cu:
//     s = (sum x^2 / D + eps)^-1/2,   y = R(p) (s x w).
// Backward, with d = R(p)^T dy:
//     dw = sum over tokens and heads of s x d,
//     dx = s (w d - x s^2 (sum w d x) / D).
// Both sums of a head are over what its lanes hold, so that x and dy are read once;
// s is computed anew in the backward pass, which costs less than reading it.  All in
// fp32, rounded once to the tensors' type.
//
// Its bound is HBM.  A head belongs to a group of lanes (a power of two), a lane has
// one vector of its turned part and the partners half a rotation away, so that sums
// go over a few shuffles and the rotation needs none.  What is not turned comes in
// pairs of vectors too.  A thread has four heads of a token (two in the backward
// pass, which holds dy too): cosines, sines and weights are loaded once for them,
// and eight loads are on the way together.
#include <string.h>

#include <algorithm>

#include "common.cuh"

namespace spark {
namespace tc {
int sm_count_cached(int dev);
}

namespace nr {
#ifndef FH
#define FH 4
#define FB 2
#define BH 2
#define BB 2
#endif

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 256;

struct Part {
    const void *x, *g;   // g: the gradient of y
    void* y;             // y, or the gradient of x
    const void* w;       // NULL: ones
    int heads, w_dtype, w_wide;   // w_wide: vectors of w lie as those of x do; fp32 on 16 bytes
    int64_t xs[3], gs[3], ys[3];
};
struct Params {
    Part part[2];
    int64_t tokens, n_tokens;        // per sequence, in all
    int dim, rot;
    int pos_bytes, wide_table;       // wide_table: rows of the table on 16 bytes
    float eps;
    const void* positions;
    const float* table;
    int64_t table_rows;
    float* partial;                  // [grid, 2, dim]: sums of the weights' gradients, or NULL
    int* err;
};

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
    static __device__ __forceinline__ void get(const type& v, float* f) {
        T t[N];
        memcpy(t, &v, sizeof(type));
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = (float)t[i];
    }
    static __device__ __forceinline__ type put(const float* f) {
        T t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) put_one(t[i], f[i]);
        type v;
        memcpy(&v, t, sizeof(type));
        return v;
    }
    static __device__ __forceinline__ type zero() {
        type v;
        memset(&v, 0, sizeof(type));
        return v;
    }
};

// Where a lane's two vectors of unit u begin (-1: there is none), and whether each is turned.
struct Place {
    int a, b;
    bool turn_a, turn_b;
};
template <int N, bool INTER>
__device__ __forceinline__ Place place(int u, int dim, int rot) {
    Place p;
    if (INTER) {
        const int n = dim / N, half = (n + 1) / 2;
        p.a = u < half ? u * N : -1;
        p.b = u < half && half + u < n ? (half + u) * N : -1;
        p.turn_a = p.a >= 0 && p.a < rot, p.turn_b = p.b >= 0 && p.b < rot;
    } else {
        const int turned = rot / 2 / N, n = (dim - rot) / N, half = (n + 1) / 2;
        p.turn_a = p.turn_b = u < turned;
        if (u < turned) {
            p.a = u * N, p.b = rot / 2 + u * N;
        } else {
            const int c = u - turned;
            p.a = c < half ? rot + c * N : -1;
            p.b = c < half && half + c < n ? rot + (half + c) * N : -1;
        }
    }
    return p;
}
// Units of a head: what `place` counts.
inline int units_of(int dim, int rot, int n, bool inter) {
    return inter ? (dim / n + 1) / 2 : rot / 2 / n + ((dim - rot) / n + 1) / 2;
}

// Cosines and sines of a lane's pairs: half layout, N of them; interleaved, N / 2 of each vector.
template <int N, bool INTER>
__device__ __forceinline__ void load_turn(const Params& p, const Place& at, int64_t pos, float* c, float* s) {
    const float* row = p.table + pos * p.rot;
    const int half = p.rot / 2;
    constexpr int M = INTER ? N / 2 : N;   // pairs of one run
    auto run = [&](int i, float* to_c, float* to_s) {
        if constexpr (M % 4 == 0) {
            if (p.wide_table) {
#pragma unroll
                for (int k = 0; k < M; k += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(row + i + k), y = *reinterpret_cast<const float4*>(row + half + i + k);
                    to_c[k] = x.x, to_c[k + 1] = x.y, to_c[k + 2] = x.z, to_c[k + 3] = x.w;
                    to_s[k] = y.x, to_s[k + 1] = y.y, to_s[k + 2] = y.z, to_s[k + 3] = y.w;
                }
                return;
            }
        }
#pragma unroll
        for (int k = 0; k < M; ++k) to_c[k] = row[i + k], to_s[k] = row[half + i + k];
    };
    if constexpr (INTER) {
        if (at.a >= 0 && at.turn_a) run(at.a / 2, c, s);
        if (at.b >= 0 && at.turn_b) run(at.b / 2, c + M, s + M);
    } else {
        if (at.turn_a) run(at.a, c, s);
    }
}

// (written with explicit roundings, so that all variants agree bit by bit)
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x = __fmaf_rn(a, c, -__fmul_rn(b, s));
    b = __fmaf_rn(b, c, __fmul_rn(a, s));
    a = x;
}
// Turns a lane's two vectors by the angles, or back.
template <int N, bool INTER>
__device__ __forceinline__ void turn_both(float* a, float* b, const Place& at, const float* c, const float* s, bool back) {
    if constexpr (INTER) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            if (at.turn_a) turn(a[k], a[k + 1], c[k / 2], back ? -s[k / 2] : s[k / 2]);
            if (at.turn_b) turn(b[k], b[k + 1], c[N / 2 + k / 2], back ? -s[N / 2 + k / 2] : s[N / 2 + k / 2]);
        }
    } else {
        if (at.turn_a) {
#pragma unroll
            for (int k = 0; k < N; ++k) turn(a[k], b[k], c[k], back ? -s[k] : s[k]);
        }
    }
}

template <typename T, int N>
__device__ __forceinline__ void load_weight(const Part& part, int at, float* w) {
    if (part.w_wide && at >= 0) {
        if (part.w_dtype == SPARK_DTYPE_F32) {
            if constexpr (N % 4 == 0) {
#pragma unroll
                for (int k = 0; k < N; k += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(part.w) + at + k);
                    w[k] = x.x, w[k + 1] = x.y, w[k + 2] = x.z, w[k + 3] = x.w;
                }
                return;
            }
        } else {
            Vec<T, N>::get(*reinterpret_cast<const typename Vec<T, N>::type*>(reinterpret_cast<const T*>(part.w) + at), w);
            return;
        }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = at >= 0 && part.w ? load_as_float(part.w, part.w_dtype, at + k) : 1.f;
}

__device__ __forceinline__ float sum_of_group(float x, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
__device__ __forceinline__ int64_t position(const Params& p, int64_t token) {
    return p.pos_bytes == 8 ? reinterpret_cast<const int64_t*>(p.positions)[token]
                            : (int64_t)reinterpret_cast<const int*>(p.positions)[token];
}
__device__ __forceinline__ float rstd_of(float squares, const Params& p) { return __frsqrt_rn(squares / (float)p.dim + p.eps); }

template <int N>
constexpr int kUnits = N >= 4 ? 1 : 4 / N;   // of a lane: kMaxDim / 2 / N over 32 lanes

// A group of `lanes` lanes takes HEADS heads of one token, of q or of k.
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(kThreads, FB) k_norm_rope(const __grid_constant__ Params p, int lanes) {
    using V = Vec<T, N>;
    using R = typename V::type;
    constexpr int U = kUnits<N>, HEADS = (FH / (U > 2 ? 2 : U) > 0 ? FH / (U > 2 ? 2 : U) : 1);
    grid_wait();
    const int groups_q = (p.part[0].heads + HEADS - 1) / HEADS, groups = groups_q + (p.part[1].heads + HEADS - 1) / HEADS;
    const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / lanes;
    const int64_t tok = i / groups;
    const bool in = tok < p.n_tokens;    // (the other lanes take part in the shuffles)
    int g = (int)(i - tok * groups);
    const int which = g >= groups_q;
    const Part& part = p.part[which];
    if (which) g -= groups_q;
    const int lane = threadIdx.x & (lanes - 1), heads = in ? min(HEADS, part.heads - g * HEADS) : 0;
    const int64_t b = in ? tok / p.tokens : 0, t = in ? tok - b * p.tokens : 0;
    const T* x = reinterpret_cast<const T*>(part.x) + b * part.xs[0] + t * part.xs[1] + (int64_t)g * HEADS * part.xs[2];
    Place at[U];
    R va[U][HEADS], vb[U][HEADS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        at[u] = place<N, INTER>(lane + u * lanes, p.dim, p.rot);
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            va[u][h] = h < heads && at[u].a >= 0 ? *reinterpret_cast<const R*>(x + h * part.xs[2] + at[u].a) : V::zero();
            vb[u][h] = h < heads && at[u].b >= 0 ? *reinterpret_cast<const R*>(x + h * part.xs[2] + at[u].b) : V::zero();
        }
    }
    const int64_t pos = in ? position(p, tok) : 0;
    const bool good = pos >= 0 && pos < p.table_rows;
    if (in && !good && lane == 0) report_device_error(p.err, 8);
    float c[U][N], s[U][N], wa[U][N], wb[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        load_turn<N, INTER>(p, at[u], good ? pos : 0, c[u], s[u]);
        load_weight<T, N>(part, at[u].a, wa[u]);
        load_weight<T, N>(part, at[u].b, wb[u]);
    }
    float rstd[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        float squares = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[N];
            V::get(va[u][h], f);
#pragma unroll
            for (int k = 0; k < N; ++k) squares = fmaf(f[k], f[k], squares);
            V::get(vb[u][h], f);
#pragma unroll
            for (int k = 0; k < N; ++k) squares = fmaf(f[k], f[k], squares);
        }
        rstd[h] = rstd_of(sum_of_group(squares, lanes), p);
    }
    T* y = reinterpret_cast<T*>(part.y) + b * part.ys[0] + t * part.ys[1] + (int64_t)g * HEADS * part.ys[2];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (h >= heads) break;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float fa[N], fb[N];
            V::get(va[u][h], fa);
            V::get(vb[u][h], fb);
#pragma unroll
            for (int k = 0; k < N; ++k) fa[k] = __fmul_rn(__fmul_rn(fa[k], rstd[h]), wa[u][k]), fb[k] = __fmul_rn(__fmul_rn(fb[k], rstd[h]), wb[u][k]);
            turn_both<N, INTER>(fa, fb, at[u], c[u], s[u], false);
            if (at[u].a >= 0) *reinterpret_cast<R*>(y + h * part.ys[2] + at[u].a) = good ? V::put(fa) : V::zero();
            if (at[u].b >= 0) *reinterpret_cast<R*>(y + h * part.ys[2] + at[u].b) = good ? V::put(fb) : V::zero();
        }
    }
}

// Backward.  The items (HEADS heads of a token) of q come first, then those of k; the groups of a warp take items side by
// side, of q or of k at once, so that a lane's sums of the weights' gradients are of one part and are put away when the
// other begins.  The order of the additions depends on the sizes alone.
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(kThreads, BB) k_norm_rope_backward(const __grid_constant__ Params p, int lanes) {
    using V = Vec<T, N>;
    using R = typename V::type;
    constexpr int U = kUnits<N>, HEADS = U > 2 ? 1 : BH;
    extern __shared__ float sums[];   // [2, kWarps, dim]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 31) / lanes, a_warp = 32 / lanes;
    for (int k = threadIdx.x; p.partial && k < 2 * kWarps * p.dim; k += kThreads) sums[k] = 0.f;
    __syncthreads();
    grid_wait();
    Place at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = place<N, INTER>(lane + u * lanes, p.dim, p.rot);
    const int64_t stride = (int64_t)gridDim.x * kWarps;
    int64_t w = (int64_t)blockIdx.x * kWarps + warp;
    for (int which = 0; which < 2; ++which) {
        const Part& part = p.part[which];
        const int groups = (part.heads + HEADS - 1) / HEADS;
        const int64_t items = p.n_tokens * groups, warps = (items + a_warp - 1) / a_warp;
        float wa[U][N], wb[U][N], da[U][N], db[U][N];
        if (w < warps) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                load_weight<T, N>(part, at[u].a, wa[u]);
                load_weight<T, N>(part, at[u].b, wb[u]);
#pragma unroll
                for (int k = 0; k < N; ++k) da[u][k] = db[u][k] = 0.f;
            }
            for (; w < warps; w += stride) {
                const int64_t i = w * a_warp + group, tok = i / groups;
                const bool in = i < items;
                const int g = in ? (int)(i - tok * groups) : 0, heads = in ? min(HEADS, part.heads - g * HEADS) : 0;
                const int64_t b = in ? tok / p.tokens : 0, t = in ? tok - b * p.tokens : 0;
                const T* x = reinterpret_cast<const T*>(part.x) + b * part.xs[0] + t * part.xs[1] + (int64_t)g * HEADS * part.xs[2];
                const T* gy = reinterpret_cast<const T*>(part.g) + b * part.gs[0] + t * part.gs[1] + (int64_t)g * HEADS * part.gs[2];
                R xa[U][HEADS], xb[U][HEADS], ga[U][HEADS], gb[U][HEADS];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) {
                        const bool ha = h < heads && at[u].a >= 0, hb = h < heads && at[u].b >= 0;
                        xa[u][h] = ha ? *reinterpret_cast<const R*>(x + h * part.xs[2] + at[u].a) : V::zero();
                        xb[u][h] = hb ? *reinterpret_cast<const R*>(x + h * part.xs[2] + at[u].b) : V::zero();
                        ga[u][h] = ha ? *reinterpret_cast<const R*>(gy + h * part.gs[2] + at[u].a) : V::zero();
                        gb[u][h] = hb ? *reinterpret_cast<const R*>(gy + h * part.gs[2] + at[u].b) : V::zero();
                    }
                const int64_t pos = in ? position(p, tok) : 0;
                const bool good = pos >= 0 && pos < p.table_rows;
                if (in && !good && lane == 0) report_device_error(p.err, 8);
                float c[U][N], s[U][N];
#pragma unroll
                for (int u = 0; u < U; ++u) load_turn<N, INTER>(p, at[u], good ? pos : 0, c[u], s[u]);
                T* dx = reinterpret_cast<T*>(part.y) + b * part.ys[0] + t * part.ys[1] + (int64_t)g * HEADS * part.ys[2];
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    float squares = 0.f, dots = 0.f;
                    float fa[U][N], fb[U][N], ea[U][N], eb[U][N];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        V::get(xa[u][h], fa[u]);
                        V::get(xb[u][h], fb[u]);
                        V::get(ga[u][h], ea[u]);
                        V::get(gb[u][h], eb[u]);
                        turn_both<N, INTER>(ea[u], eb[u], at[u], c[u], s[u], true);
#pragma unroll
                        for (int k = 0; k < N; ++k) {
                            squares = fmaf(fa[u][k], fa[u][k], squares);
                            squares = fmaf(fb[u][k], fb[u][k], squares);
                            dots = fmaf(ea[u][k] * wa[u][k], fa[u][k], dots);
                            dots = fmaf(eb[u][k] * wb[u][k], fb[u][k], dots);
                        }
                    }
                    squares = sum_of_group(squares, lanes);
                    dots = sum_of_group(dots, lanes);
                    if (h >= heads) continue;
                    const float r = rstd_of(squares, p), mean = dots * r / (float)p.dim;   // of w d times the unit row
#pragma unroll
                    for (int u = 0; u < U; ++u) {
#pragma unroll
                        for (int k = 0; k < N; ++k) {
                            const float na = fa[u][k] * r, nb = fb[u][k] * r;
                            if (good) da[u][k] = fmaf(ea[u][k], na, da[u][k]), db[u][k] = fmaf(eb[u][k], nb, db[u][k]);
                            ea[u][k] = r * fmaf(-na, mean, ea[u][k] * wa[u][k]);
                            eb[u][k] = r * fmaf(-nb, mean, eb[u][k] * wb[u][k]);
                        }
                        if (at[u].a >= 0) *reinterpret_cast<R*>(dx + h * part.ys[2] + at[u].a) = good ? V::put(ea[u]) : V::zero();
                        if (at[u].b >= 0) *reinterpret_cast<R*>(dx + h * part.ys[2] + at[u].b) = good ? V::put(eb[u]) : V::zero();
                    }
                }
            }
            if (p.partial) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        for (int o = lanes; o < 32; o <<= 1) {
                            da[u][k] += __shfl_xor_sync(0xffffffffu, da[u][k], o);
                            db[u][k] += __shfl_xor_sync(0xffffffffu, db[u][k], o);
                        }
                        float* to = sums + (which * kWarps + warp) * p.dim;
                        if (group == 0 && at[u].a >= 0) to[at[u].a + k] = da[u][k];
                        if (group == 0 && at[u].b >= 0) to[at[u].b + k] = db[u][k];
                    }
            }
        }
        w -= warps;   // the walk goes on in the other part
    }
    if (!p.partial) return;
    __syncthreads();
    for (int k = threadIdx.x; k < 2 * p.dim; k += kThreads) {
        const int which = k / p.dim, col = k - which * p.dim;
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) sum += sums[(which * kWarps + v) * p.dim + col];
        p.partial[(int64_t)blockIdx.x * 2 * p.dim + k] = sum;
    }
}

// dw of q and of k: the blocks' sums, added by 8 threads a column, then those.
struct Weights {
    void* to[2];
    int dtype[2];
};
__global__ void __launch_bounds__(256) k_norm_weights(const float* partial, int blocks, int dim, Weights out) {
    __shared__ float part[8][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, col = blockIdx.x * 32 + x;
    grid_wait();
    float sum = 0.f;
    if (col < 2 * dim)
        for (int i = y; i < blocks; i += 8) sum += partial[(int64_t)i * 2 * dim + col];
    part[y][x] = sum;
    __syncthreads();
    if (y == 0 && col < 2 * dim) {
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) all += part[i][x];
        const int which = col >= dim;
        if (out.to[which]) store_from_float(out.to[which], out.dtype[which], col - which * dim, all);
    }
}

template <typename T, int N, bool INTER>
cudaError_t launch(const Params& p, int lanes, bool backward, int grid, cudaStream_t s) {
    if (!backward) return launch_overlapped(k_norm_rope<T, N, INTER>, grid, kThreads, 0, s, p, lanes);
    return launch_overlapped(k_norm_rope_backward<T, N, INTER>, grid, kThreads, p.partial ? 2 * kWarps * p.dim * sizeof(float) : 0, s,
                             p, lanes);
}
template <typename T, int N>
cudaError_t launch(const Params& p, int lanes, bool inter, bool backward, int grid, cudaStream_t s) {
    if constexpr (N > 1)
        if (inter) return launch<T, N, true>(p, lanes, backward, grid, s);
    return launch<T, N, false>(p, lanes, backward, grid, s);
}
template <typename T>
cudaError_t launch(const Params& p, int vec, int lanes, bool inter, bool backward, int grid, cudaStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (vec == 8) return launch<T, 8>(p, lanes, inter, backward, grid, s);
    if (vec == 4) return launch<T, 4>(p, lanes, inter, backward, grid, s);
    if (vec == 2) return launch<T, 2>(p, lanes, inter, backward, grid, s);
    return launch<T, 1>(p, lanes, inter, backward, grid, s);
}

// Blocks of the backward pass: as many as are resident at two an SM.
int backward_blocks() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    return BB * tc::sm_count_cached(dev);
}

int run(const SparkNormRope* a, bool backward, void* workspace, size_t workspace_bytes, int* err, cudaStream_t s, const char* name) {
    SPARK_REQUIRE(a, SPARK_ERR_INVALID, "%s: null pointer", name);
    SPARK_REQUIRE(a->dtype >= 0 && a->dtype <= 2, SPARK_ERR_INVALID, "%s: bad dtype %d", name, (int)a->dtype);
    SPARK_REQUIRE(a->position_bytes == 4 || a->position_bytes == 8, SPARK_ERR_INVALID, "%s: positions are 4- or 8-byte integers", name);
    SPARK_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->table_rows >= 1, SPARK_ERR_INVALID, "%s: bad size", name);
    SPARK_REQUIRE(a->batch < (1ll << 31) && a->tokens < (1ll << 31), SPARK_ERR_UNSUPPORTED, "%s: bad size", name);
    SPARK_REQUIRE(a->head_dim >= 2 && a->head_dim % 2 == 0 && a->head_dim <= kMaxDim, SPARK_ERR_UNSUPPORTED,
                  "%s: head_dim %lld is not an even number of 2..%d", name, (long long)a->head_dim, kMaxDim);
    SPARK_REQUIRE(a->rot_dim >= 2 && a->rot_dim % 2 == 0 && a->rot_dim <= a->head_dim, SPARK_ERR_INVALID,
                  "%s: rot_dim %lld is not an even number of 2..head_dim (%lld)", name, (long long)a->rot_dim, (long long)a->head_dim);
    SPARK_REQUIRE(a->eps >= 0 && a->eps <= 1e30, SPARK_ERR_INVALID, "%s: eps must be 0 or above, got %g", name, a->eps);
    Params p{};
    const bool empty = a->batch == 0 || a->tokens == 0;
    bool weights = false;
    int64_t heads = 0;
    for (int w = 0; w < 2; ++w) {
        const SparkNormRopeHeads& h = a->part[w];
        Part& t = p.part[w];
        SPARK_REQUIRE(h.heads >= 0 && h.heads < (1 << 20), SPARK_ERR_INVALID, "%s: heads", name);
        SPARK_REQUIRE(!h.weight || (h.weight_dtype >= 0 && h.weight_dtype <= 2), SPARK_ERR_INVALID, "%s: bad dtype of a weight", name);
        SPARK_REQUIRE(!h.dweight || (backward && h.weight), SPARK_ERR_INVALID, "%s: the gradient of no weight", name);
        weights = weights || h.dweight;
        if (h.heads == 0 || empty) continue;
        SPARK_REQUIRE(h.x && h.y && (!backward || h.dy), SPARK_ERR_INVALID, "%s: null pointer", name);
        const int64_t extent[3] = {a->batch, a->tokens, h.heads};
        bool same = true;
        for (int i = 0; i < 3; ++i) {
            SPARK_REQUIRE(extent[i] == 1 || h.ys[i] != 0, SPARK_ERR_INVALID, "%s: output rows in one place", name);
            same = same && h.xs[i] == h.ys[i];
            // (a stride that no second row uses says nothing)
            t.xs[i] = extent[i] == 1 ? 0 : h.xs[i], t.ys[i] = extent[i] == 1 ? 0 : h.ys[i], t.gs[i] = extent[i] == 1 || !backward ? 0 : h.dys[i];
        }
        SPARK_REQUIRE(h.x != h.y || (same && !backward), SPARK_ERR_INVALID, "%s: in place needs equal strides, forward", name);
        t.x = h.x, t.y = h.y, t.g = h.dy, t.w = h.weight, t.w_dtype = (int)h.weight_dtype, t.heads = (int)h.heads;
        heads += h.heads;
    }
    if (p.part[0].heads && p.part[1].heads)
        SPARK_REQUIRE(p.part[0].y != p.part[1].x && p.part[1].y != p.part[0].x && p.part[0].y != p.part[1].y, SPARK_ERR_INVALID,
                      "%s: the output of one part is the other's input or output", name);
    if (empty || heads == 0) {
        // no token: the weights' gradients are zero
        for (const SparkNormRopeHeads& h : a->part) {
            if (!h.dweight) continue;
            const cudaError_t e = cudaMemsetAsync(h.dweight, 0, a->head_dim * (h.weight_dtype == SPARK_DTYPE_F32 ? 4 : 2), s);
            if (e != cudaSuccess) return set_error((int)e, "%s: %s", name, cudaGetErrorString(e));
        }
        return SPARK_OK;
    }
    SPARK_REQUIRE(a->positions && a->table, SPARK_ERR_INVALID, "%s: null pointer", name);
    p.tokens = a->tokens, p.n_tokens = a->batch * a->tokens;
    p.dim = (int)a->head_dim, p.rot = (int)a->rot_dim, p.eps = (float)a->eps;
    p.pos_bytes = (int)a->position_bytes, p.positions = a->positions, p.table = a->table, p.table_rows = a->table_rows, p.err = err;
    p.wide_table = aligned(a->table, 16) && a->rot_dim % 8 == 0;
    // the longest vectors that fit everything
    const bool inter = a->interleaved != 0;
    const int es = a->dtype == SPARK_DTYPE_F32 ? 4 : 2;
    int vec = 16 / es;
    for (; vec > 1; vec /= 2) {
        bool ok = inter ? p.dim % vec == 0 && p.rot % vec == 0 : p.rot / 2 % vec == 0 && (p.dim - p.rot) % vec == 0;
        for (const Part& t : p.part) {
            if (t.heads == 0) continue;
            ok = ok && aligned(t.x, (size_t)vec * es) && aligned(t.y, (size_t)vec * es) && aligned(t.g, (size_t)vec * es);
            for (int i = 0; i < 3; ++i) ok = ok && t.xs[i] % vec == 0 && t.ys[i] % vec == 0 && t.gs[i] % vec == 0;
        }
        if (ok) break;
    }
    SPARK_REQUIRE(vec > 1 || !inter, SPARK_ERR_ALIGNMENT, "%s: interleaved pairs lie on %d bytes, with even strides", name, 2 * es);
    for (Part& t : p.part)
        t.w_wide = t.w && (t.w_dtype == SPARK_DTYPE_F32 ? vec % 4 == 0 && aligned(t.w, 16)
                                                        : t.w_dtype == (int)a->dtype && aligned(t.w, (size_t)vec * es));
    const int units = units_of(p.dim, p.rot, vec, inter);
    int lanes = 1;
    while (lanes < units && lanes < 32) lanes *= 2;
    int64_t grid;
    const int u = vec >= 4 ? 1 : 4 / vec;   // kUnits
    if (!backward) {
        const int a_group = (FH / (u > 2 ? 2 : u) > 0 ? FH / (u > 2 ? 2 : u) : 1);
        const int64_t groups = (p.part[0].heads + a_group - 1) / a_group + (p.part[1].heads + a_group - 1) / a_group;
        const int64_t a_block = kThreads / lanes;
        grid = (p.n_tokens * groups + a_block - 1) / a_block;
    } else {
        const int a_group = u > 2 ? 1 : BH;
        const int64_t most = std::max((p.part[0].heads + a_group - 1) / a_group, (p.part[1].heads + a_group - 1) / a_group);
        const int64_t a_block = kThreads / lanes;
        const int blocks = backward_blocks();
        SPARK_REQUIRE(blocks > 0, SPARK_ERR_DEVICE, "%s: no device", name);
        grid = std::min<int64_t>((p.n_tokens * most + a_block - 1) / a_block, blocks);
        if (weights) {
            const size_t need = (size_t)blocks * 2 * p.dim * sizeof(float);
            SPARK_REQUIRE(workspace && workspace_bytes >= need && aligned(workspace, 16), SPARK_ERR_WORKSPACE,
                          "%s: workspace of %zu bytes on 16, %zu needed", name, workspace_bytes, need);
            p.partial = reinterpret_cast<float*>(workspace);
        }
    }
    SPARK_REQUIRE(grid < (1ll << 31), SPARK_ERR_UNSUPPORTED, "%s: too many values for one call", name);
    cudaError_t e;
    if (a->dtype == SPARK_DTYPE_F32) e = launch<float>(p, vec, lanes, inter, backward, (int)grid, s);
    else if (a->dtype == SPARK_DTYPE_BF16) e = launch<__nv_bfloat16>(p, vec, lanes, inter, backward, (int)grid, s);
    else e = launch<__half>(p, vec, lanes, inter, backward, (int)grid, s);
    if (e == cudaSuccess && p.partial) {
        Weights out;
        for (int w = 0; w < 2; ++w) out.to[w] = a->part[w].dweight, out.dtype[w] = (int)a->part[w].weight_dtype;
        e = launch_overlapped(k_norm_weights, (2 * p.dim + 31) / 32, 256, 0, s, (const float*)p.partial, (int)grid, p.dim, out);
    }
    if (e != cudaSuccess) return set_error((int)e, "%s: launch failed: %s", name, cudaGetErrorString(e));
    return check_launch(name);
}

}  // namespace nr
}  // namespace spark

extern "C" {

int spark_qk_norm_rope(const SparkNormRope* a, int* err, void* stream) {
    return spark::nr::run(a, false, nullptr, 0, err, reinterpret_cast<cudaStream_t>(stream), "spark_qk_norm_rope");
}

size_t spark_qk_norm_rope_backward_workspace_size(int64_t head_dim) {
    return head_dim > 0 ? (size_t)spark::nr::backward_blocks() * 2 * head_dim * sizeof(float) : 0;
}

int spark_qk_norm_rope_backward(const SparkNormRope* a, void* workspace, size_t workspace_bytes, int* err, void* stream) {
    return spark::nr::run(a, true, workspace, workspace_bytes, err, reinterpret_cast<cudaStream_t>(stream),
                          "spark_qk_norm_rope_backward");
}

}  // extern "C"
