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
    // how a warp's groups of lanes take it: 2^across of them side by side along the heads, the others along the tokens; an item is
    // such a tile of tokens with `span` steps along the heads, `chunks` of them for a token's heads
    int across, chunks, span, items;
};
struct Params {
    Part part[2];
    int tokens, n_tokens;            // per sequence, in all
    int dim, rot;
    int pos_bytes, wide_table;       // wide_table: rows of the table on 16 bytes
    float eps, per_dim;
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
__device__ __forceinline__ void put_two(float* to, float a, float b) { to[0] = a, to[1] = b; }
__device__ __forceinline__ void put_two(__nv_bfloat16* to, float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    memcpy(to, &v, 4);
}
__device__ __forceinline__ void put_two(__half* to, float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    memcpy(to, &v, 4);
}
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
        if constexpr (N == 1) {
            put_one(t[0], f[0]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) put_two(t + i, f[i], f[i + 1]);
        }
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

// Products and sums of N values, two an instruction.
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void untwo(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
template <int N>
__device__ __forceinline__ void mul(float (&d)[N], const float (&a)[N], const float (&b)[N]) {
    if constexpr (N == 1) {
        d[0] = __fmul_rn(a[0], b[0]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            uint64_t v;
            asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(two(a[i], a[i + 1])), "l"(two(b[i], b[i + 1])));
            untwo(v, d[i], d[i + 1]);
        }
    }
}
template <int N>
__device__ __forceinline__ void mul(float (&d)[N], const float (&a)[N], float b) {
    float bs[N];
#pragma unroll
    for (int i = 0; i < N; ++i) bs[i] = b;
    mul(d, a, bs);
}
// d = a b + c
template <int N>
__device__ __forceinline__ void fma(float (&d)[N], const float (&a)[N], const float (&b)[N], const float (&c)[N]) {
    if constexpr (N == 1) {
        d[0] = __fmaf_rn(a[0], b[0], c[0]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            uint64_t v;
            asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(two(a[i], a[i + 1])), "l"(two(b[i], b[i + 1])), "l"(two(c[i], c[i + 1])));
            untwo(v, d[i], d[i + 1]);
        }
    }
}
template <int N>
__device__ __forceinline__ void fma(float (&d)[N], const float (&a)[N], float b, const float (&c)[N]) {
    float bs[N];
#pragma unroll
    for (int i = 0; i < N; ++i) bs[i] = b;
    fma(d, a, bs, c);
}
// The two sums that a dot product of a and b runs in (one, where there is one value).
template <int N>
__device__ __forceinline__ void dot(float (&sum)[2], const float (&a)[N], const float (&b)[N]) {
    if constexpr (N == 1) {
        sum[0] = __fmaf_rn(a[0], b[0], sum[0]);
    } else {
        uint64_t v = two(sum[0], sum[1]);
#pragma unroll
        for (int i = 0; i < N; i += 2)
            asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(v) : "l"(two(a[i], a[i + 1])), "l"(two(b[i], b[i + 1])));
        untwo(v, sum[0], sum[1]);
    }
}

// A lane's part of the rotation: (a, b) -> (a pa + a' qa, b pb + b' qb), where a' and b' are, in the half layout, b and a;
// interleaved, a and b with the values of each pair exchanged.
template <int N, bool INTER>
struct Turn {
    float pa[N], qa[N], pb[N], qb[N];

    // the angles of a position, or of its inverse
    __device__ __forceinline__ void load(const Params& p, const Place& at, int64_t pos, bool back) {
        const float* row = p.table + pos * p.rot;
        const int half = p.rot / 2;
        constexpr int M = INTER ? N / 2 : N;   // pairs of one run
        auto run = [&](int i, float* c, float* s) {
            if constexpr (M % 4 == 0) {
                if (p.wide_table) {
#pragma unroll
                    for (int k = 0; k < M; k += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(row + i + k), y = *reinterpret_cast<const float4*>(row + half + i + k);
                        c[k] = x.x, c[k + 1] = x.y, c[k + 2] = x.z, c[k + 3] = x.w;
                        s[k] = y.x, s[k + 1] = y.y, s[k + 2] = y.z, s[k + 3] = y.w;
                    }
                    return;
                }
            }
#pragma unroll
            for (int k = 0; k < M; ++k) c[k] = row[i + k], s[k] = row[half + i + k];
        };
        float c[M], s[M];
        if constexpr (INTER) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (!(w ? at.turn_b : at.turn_a)) continue;
                run((w ? at.b : at.a) / 2, c, s);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    (w ? pb : pa)[k] = c[k / 2];
                    (w ? qb : qa)[k] = (k & 1) == back ? -s[k / 2] : s[k / 2];
                }
            }
        } else if (at.turn_a) {
            run(at.a, c, s);
#pragma unroll
            for (int k = 0; k < N; ++k) pa[k] = pb[k] = c[k], qa[k] = back ? s[k] : -s[k], qb[k] = back ? -s[k] : s[k];
        }
    }
    // with the weights of what is turned in it (where nothing is turned pa and pb are the weights)
    __device__ __forceinline__ void weigh(const Place& at, const float (&wa)[N], const float (&wb)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if constexpr (INTER) {
                pa[k] = at.turn_a ? wa[k] * pa[k] : wa[k], qa[k] *= wa[k ^ 1];
                pb[k] = at.turn_b ? wb[k] * pb[k] : wb[k], qb[k] *= wb[k ^ 1];
            } else {
                pa[k] = at.turn_a ? wa[k] * pa[k] : wa[k], qa[k] *= wb[k];
                pb[k] = at.turn_a ? wb[k] * pb[k] : wb[k], qb[k] *= wa[k];
            }
        }
    }
    // plain: what is not turned stays what it is; else it is multiplied too
    template <bool PLAIN>
    __device__ __forceinline__ void apply(const Place& at, float (&a)[N], float (&b)[N]) const {
        if constexpr (INTER) {
            one<PLAIN>(at.turn_a, pa, qa, a);
            one<PLAIN>(at.turn_b, pb, qb, b);
        } else {
            if (at.turn_a) {
                float x[N], y[N];
                mul(x, b, qa);
                mul(y, a, qb);
                fma(a, a, pa, x);
                fma(b, b, pb, y);
            } else if constexpr (!PLAIN) {
                mul(a, a, pa);
                mul(b, b, pb);
            }
        }
    }
    template <bool PLAIN>
    static __device__ __forceinline__ void one(bool turns, const float (&pp)[N], const float (&qq)[N], float (&a)[N]) {
        if (turns) {
            float x[N];
#pragma unroll
            for (int k = 0; k < N; ++k) x[k] = a[k ^ 1];
            mul(x, x, qq);
            fma(a, a, pp, x);
        } else if constexpr (!PLAIN) {
            mul(a, a, pp);
        }
    }
};

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

template <int N>
__device__ __forceinline__ void sum_of_group(float (&x)[N], int lanes) {
    for (int o = 1; o < lanes; o <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
}
// What a group of lanes does of an item.
struct Work {
    int token, head;    // the first head
    bool in;
    int64_t b, t;
};
template <int HEADS>
__device__ __forceinline__ Work work_of(const Params& p, const Part& part, int item, int group, int a_warp) {
    Work w;
    const int tile = part.chunks == 1 ? item : item / part.chunks, chunk = item - tile * part.chunks;
    w.token = tile * (a_warp >> part.across) + (group >> part.across);
    w.head = ((chunk * part.span << part.across) + (group & ((1 << part.across) - 1))) * HEADS;
    w.in = w.token < p.n_tokens;
    if (!w.in) w.token = 0;
    const int b = w.token / p.tokens;
    w.b = b, w.t = w.token - b * p.tokens;
    return w;
}
__device__ __forceinline__ int64_t position(const Params& p, int64_t token) {
    return p.pos_bytes == 8 ? reinterpret_cast<const int64_t*>(p.positions)[token]
                            : (int64_t)reinterpret_cast<const int*>(p.positions)[token];
}
// (the approximation's 2^-22, and a step of Newton's iteration, which leaves a rounding or two; 0 and infinity stay what it gives)
__device__ __forceinline__ float rstd_of(float squares, const Params& p) {
    const float x = __fmaf_rn(squares, p.per_dim, p.eps), r = rsqrtf(x), e = __fmaf_rn(-x * r, r, 1.f);
    return fabsf(e) < 1.f ? __fmaf_rn(0.5f * r, e, r) : r;
}

template <int N>
constexpr int kUnits = N >= 4 ? 1 : 4 / N;   // of a lane: kMaxDim / 2 / N over 32 lanes
template <int N>
constexpr int kHeads = N >= 4 ? FH : 2;      // of a step, forward
template <int N>
constexpr int kHeadsBack = N >= 2 ? BH : 1;  // backward

// A group of `lanes` lanes takes HEADS heads of one token at a step.
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(kThreads, FB) k_norm_rope(const __grid_constant__ Params p, int lanes) {
    using V = Vec<T, N>;
    using R = typename V::type;
    constexpr int U = kUnits<N>, HEADS = kHeads<N>;
    const int lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 31) / lanes, a_warp = 32 / lanes;
    grid_wait();
    Place at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = place<N, INTER>(lane + u * lanes, p.dim, p.rot);
    int item = blockIdx.x * kWarps + (threadIdx.x >> 5);
    for (int which = 0; which < 2; item -= p.part[which++].items) {
        const Part& part = p.part[which];
        if (item >= part.items) continue;
        for (; item < part.items; item += gridDim.x * kWarps) {
            const Work w = work_of<HEADS>(p, part, item, group, a_warp);
            const int64_t pos = position(p, w.token);
            const bool good = pos >= 0 && pos < p.table_rows;
            if (w.in && !good && lane == 0) report_device_error(p.err, 8);
            const T* x = reinterpret_cast<const T*>(part.x) + w.b * part.xs[0] + w.t * part.xs[1] + w.head * part.xs[2];
            T* y = reinterpret_cast<T*>(part.y) + w.b * part.ys[0] + w.t * part.ys[1] + w.head * part.ys[2];
            Turn<N, INTER> turn[U];
            for (int k = 0, left = w.in ? part.heads - w.head : 0; k < part.span; ++k) {
                R va[U][HEADS], vb[U][HEADS];
                // (lanes without a head take part in the shuffles)
#pragma unroll
                for (int h = 0; h < HEADS; ++h)
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        va[u][h] = h < left && at[u].a >= 0 ? *reinterpret_cast<const R*>(x + h * part.xs[2] + at[u].a) : V::zero();
                        vb[u][h] = h < left && at[u].b >= 0 ? *reinterpret_cast<const R*>(x + h * part.xs[2] + at[u].b) : V::zero();
                    }
                if (k == 0) {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float wa[N], wb[N];
                        turn[u].load(p, at[u], good ? pos : 0, false);
                        load_weight<T, N>(part, at[u].a, wa);
                        load_weight<T, N>(part, at[u].b, wb);
                        turn[u].weigh(at[u], wa, wb);
                    }
                }
                float squares[HEADS];
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    float both[2] = {0.f, 0.f};
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float f[N];
                        V::get(va[u][h], f);
                        dot(both, f, f);
                        V::get(vb[u][h], f);
                        dot(both, f, f);
                    }
                    squares[h] = both[0] + both[1];
                }
                sum_of_group(squares, lanes);
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    if (h >= left) break;
                    const float rstd = rstd_of(squares[h], p);
                    T* yh = y + h * part.ys[2];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float fa[N], fb[N];
                        V::get(va[u][h], fa);
                        V::get(vb[u][h], fb);
                        mul(fa, fa, rstd);
                        mul(fb, fb, rstd);
                        turn[u].template apply<false>(at[u], fa, fb);
                        va[u][h] = V::put(fa), vb[u][h] = V::put(fb);
                        if (!good) va[u][h] = vb[u][h] = V::zero();
                        if (at[u].a >= 0) *reinterpret_cast<R*>(yh + at[u].a) = va[u][h];
                        if (at[u].b >= 0) *reinterpret_cast<R*>(yh + at[u].b) = vb[u][h];
                    }
                }
                const int on = HEADS << part.across;
                x += on * part.xs[2], y += on * part.ys[2], left -= on;
            }
        }
    }
}

// Backward.  The items of q come first, then those of k, so that a lane's sums of the weights' gradients are of one part and are
// put away when the other begins.  The order of the additions depends on the sizes alone.
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(kThreads, BB) k_norm_rope_backward(const __grid_constant__ Params p, int lanes) {
    using V = Vec<T, N>;
    using R = typename V::type;
    constexpr int U = kUnits<N>, HEADS = kHeadsBack<N>;
    extern __shared__ float sums[];   // [2, kWarps, dim]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 31) / lanes, a_warp = 32 / lanes;
    for (int k = threadIdx.x; p.partial && k < 2 * kWarps * p.dim; k += kThreads) sums[k] = 0.f;
    __syncthreads();
    grid_wait();
    Place at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = place<N, INTER>(lane + u * lanes, p.dim, p.rot);
    int item = blockIdx.x * kWarps + warp;
    for (int which = 0; which < 2; item -= p.part[which++].items) {
        const Part& part = p.part[which];
        if (item >= part.items) continue;
        float wa[U][N], wb[U][N], da[U][N], db[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            load_weight<T, N>(part, at[u].a, wa[u]);
            load_weight<T, N>(part, at[u].b, wb[u]);
#pragma unroll
            for (int j = 0; j < N; ++j) da[u][j] = db[u][j] = 0.f;
        }
        for (; item < part.items; item += gridDim.x * kWarps) {
            const Work w = work_of<HEADS>(p, part, item, group, a_warp);
            const int64_t pos = position(p, w.token);
            const bool good = pos >= 0 && pos < p.table_rows;
            if (w.in && !good && lane == 0) report_device_error(p.err, 8);
            const T* x = reinterpret_cast<const T*>(part.x) + w.b * part.xs[0] + w.t * part.xs[1] + w.head * part.xs[2];
            const T* gy = reinterpret_cast<const T*>(part.g) + w.b * part.gs[0] + w.t * part.gs[1] + w.head * part.gs[2];
            T* dx = reinterpret_cast<T*>(part.y) + w.b * part.ys[0] + w.t * part.ys[1] + w.head * part.ys[2];
            Turn<N, INTER> turn[U];
            for (int k = 0, left = w.in ? part.heads - w.head : 0; k < part.span; ++k) {
                R xa[U][HEADS], xb[U][HEADS], ga[U][HEADS], gb[U][HEADS];
#pragma unroll
                for (int h = 0; h < HEADS; ++h)
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const bool ha = h < left && at[u].a >= 0, hb = h < left && at[u].b >= 0;
                        xa[u][h] = ha ? *reinterpret_cast<const R*>(x + h * part.xs[2] + at[u].a) : V::zero();
                        xb[u][h] = hb ? *reinterpret_cast<const R*>(x + h * part.xs[2] + at[u].b) : V::zero();
                        ga[u][h] = ha ? *reinterpret_cast<const R*>(gy + h * part.gs[2] + at[u].a) : V::zero();
                        gb[u][h] = hb ? *reinterpret_cast<const R*>(gy + h * part.gs[2] + at[u].b) : V::zero();
                    }
                if (k == 0) {
#pragma unroll
                    for (int u = 0; u < U; ++u) turn[u].load(p, at[u], good ? pos : 0, true);
                }
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    float squares[2] = {0.f, 0.f}, dots[2] = {0.f, 0.f};     // sums of squares and of w d x
                    float ea[U][N], eb[U][N];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float f[N], wd[N];
                        V::get(ga[u][h], ea[u]);
                        V::get(gb[u][h], eb[u]);
                        turn[u].template apply<true>(at[u], ea[u], eb[u]);
                        V::get(xa[u][h], f);
                        dot(squares, f, f);
                        mul(wd, ea[u], wa[u]);
                        dot(dots, wd, f);
                        V::get(xb[u][h], f);
                        dot(squares, f, f);
                        mul(wd, eb[u], wb[u]);
                        dot(dots, wd, f);
                    }
                    float sum[2] = {squares[0] + squares[1], dots[0] + dots[1]};
                    sum_of_group(sum, lanes);
                    if (h >= left) continue;   // (not further on: the others' shuffles take all lanes)
                    const float r = rstd_of(sum[0], p), mean = -(sum[1] * r) * p.per_dim;   // of w d times the unit row, negative
                    T* dh = dx + h * part.ys[2];
                    auto half = [&](const R& v, float (&e)[N], const float (&w)[N], float (&d)[N], int to) {
                        float n[N];
                        V::get(v, n);
                        mul(n, n, r);
                        if (good) fma(d, e, n, d);
                        mul(e, e, w);
                        fma(e, n, mean, e);
                        mul(e, e, r);
                        if (to >= 0) *reinterpret_cast<R*>(dh + to) = good ? V::put(e) : V::zero();
                    };
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        half(xa[u][h], ea[u], wa[u], da[u], at[u].a);
                        half(xb[u][h], eb[u], wb[u], db[u], at[u].b);
                    }
                }
                const int on = HEADS << part.across;
                x += on * part.xs[2], gy += on * part.gs[2], dx += on * part.ys[2], left -= on;
            }
        }
        if (!p.partial) continue;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                for (int o = lanes; o < 32; o <<= 1) {
                    da[u][j] += __shfl_xor_sync(0xffffffffu, da[u][j], o);
                    db[u][j] += __shfl_xor_sync(0xffffffffu, db[u][j], o);
                }
                float* to = sums + (which * kWarps + warp) * p.dim;
                if (group == 0 && at[u].a >= 0) to[at[u].a + j] = da[u][j];
                if (group == 0 && at[u].b >= 0) to[at[u].b + j] = db[u][j];
            }
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

int sm_count() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess ? tc::sm_count_cached(dev) : 0;
}

int run(const SparkNormRope* a, bool backward, void* workspace, size_t workspace_bytes, int* err, cudaStream_t s, const char* name) {
    SPARK_REQUIRE(a, SPARK_ERR_INVALID, "%s: null pointer", name);
    SPARK_REQUIRE(a->dtype >= 0 && a->dtype <= 2, SPARK_ERR_INVALID, "%s: bad dtype %d", name, (int)a->dtype);
    SPARK_REQUIRE(a->position_bytes == 4 || a->position_bytes == 8, SPARK_ERR_INVALID, "%s: positions are 4- or 8-byte integers", name);
    SPARK_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->table_rows >= 1, SPARK_ERR_INVALID, "%s: bad size", name);
    SPARK_REQUIRE(a->batch < (1ll << 30) && a->tokens < (1ll << 30) && a->batch * a->tokens < (1ll << 30), SPARK_ERR_UNSUPPORTED,
                  "%s: 2^30 tokens or more", name);
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
    p.tokens = (int)a->tokens, p.n_tokens = (int)(a->batch * a->tokens);
    p.dim = (int)a->head_dim, p.rot = (int)a->rot_dim, p.eps = (float)a->eps, p.per_dim = 1.f / (float)a->head_dim;
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
    const int blocks = (backward ? BB : FB) * sm_count();
    SPARK_REQUIRE(blocks > 0, SPARK_ERR_DEVICE, "%s: no device", name);
    const int step = backward ? (vec >= 2 ? BH : 1) : (vec >= 4 ? FH : 2);
    int64_t items = 0;
    for (Part& t : p.part) {
        if (t.heads == 0) continue;
        const int steps = (t.heads + step - 1) / step;     // of one group of lanes for a token's heads
        while ((1 << t.across) < 32 / lanes && (1 << t.across) < steps) ++t.across;
        const int64_t tiles = (p.n_tokens + (32 / lanes >> t.across) - 1) / (32 / lanes >> t.across);
        const int all = (steps + (1 << t.across) - 1) >> t.across;
        // as few items for a token as keep all warps at work, twice
        t.chunks = (int)std::min<int64_t>(all, std::max<int64_t>(1, 2 * (int64_t)blocks * kWarps / tiles));
        t.span = (all + t.chunks - 1) / t.chunks;
        SPARK_REQUIRE(tiles * t.chunks < (1ll << 30), SPARK_ERR_UNSUPPORTED, "%s: too many values for one call", name);
        t.items = (int)(tiles * t.chunks);
        items += t.items;
    }
    const int64_t grid = std::min<int64_t>((items + kWarps - 1) / kWarps, blocks);
    if (backward && weights) {
        const size_t need = (size_t)blocks * 2 * p.dim * sizeof(float);
        SPARK_REQUIRE(workspace && workspace_bytes >= need && aligned(workspace, 16), SPARK_ERR_WORKSPACE,
                      "%s: workspace of %zu bytes on 16, %zu needed", name, workspace_bytes, need);
        p.partial = reinterpret_cast<float*>(workspace);
    }
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
    return head_dim > 0 ? (size_t)BB * spark::nr::sm_count() * 2 * head_dim * sizeof(float) : 0;
}

int spark_qk_norm_rope_backward(const SparkNormRope* a, void* workspace, size_t workspace_bytes, int* err, void* stream) {
    return spark::nr::run(a, true, workspace, workspace_bytes, err, reinterpret_cast<cudaStream_t>(stream),
                          "spark_qk_norm_rope_backward");
}

}  // extern "C"
