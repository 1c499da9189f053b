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
// Its bound is HBM: 2 accesses a value forward, 3 backward, where 8 and 13 instructions a
// value take half to two thirds of that time.  A head belongs to a group of lanes (a
// power of two); a lane has one vector of its turned part and the partners half a
// rotation away, so that sums go over a few shuffles and the rotation needs none.  What
// is not turned comes in pairs of vectors too.  A group walks along the heads of a
// token, whose angles (with the weights in them, forward) stay in registers; vectors
// come three steps ahead by asynchronous copies.  Measured: 8 x 4096 tokens of 32 + 8
// heads of 128 in bf16, forward 126 us (5.3 TB/s), forward and backward 298 us (5.6
// TB/s); without the copies ahead 372 us, with one head's products in scalar
// instructions 454 us.  2048 tokens 13.4 us, of which half is the launch and the way
// from a position to its angles.
#include <string.h>

#include <algorithm>

#include "common.cuh"
#include "overlap.cuh"

namespace spark {
namespace tc {
int sm_count_cached(int dev);
}

namespace nr {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 256;
constexpr int kBlocks = 2;     // of an SM (128 registers a thread; 3 spill, and take 10 to 60% longer)
constexpr int kStages = 3;     // steps on their way (4 are no faster)

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
// The steps of a warp, in order: HEADS heads of a token at a time for each of its groups of lanes; the items of q first, then those
// of k.
template <typename T, int HEADS>
struct Steps {
    int which, item, k, left, token;    // left: heads from this step on (0 or fewer: none for this group)
    const T *x, *g;
    T* y;

    __device__ __forceinline__ bool done() const { return which == 2; }
    __device__ __forceinline__ void begin(const Params& p, int group, int a_warp) {
        which = 0, item = blockIdx.x * kWarps + (threadIdx.x >> 5);
        enter(p, group, a_warp);
    }
    __device__ __forceinline__ void enter(const Params& p, int group, int a_warp) {
        while (which < 2 && item >= p.part[which].items) item -= p.part[which++].items;
        if (which == 2) return;
        const Part& part = p.part[which];
        const int tile = part.chunks == 1 ? item : item / part.chunks, chunk = item - tile * part.chunks;
        const int head = ((chunk * part.span << part.across) + (group & ((1 << part.across) - 1))) * HEADS;
        token = tile * (a_warp >> part.across) + (group >> part.across);
        left = token < p.n_tokens ? part.heads - head : 0;
        if (token >= p.n_tokens) token = 0;
        const int b = token / p.tokens, t = token - b * p.tokens;
        k = 0;
        x = reinterpret_cast<const T*>(part.x) + b * part.xs[0] + t * part.xs[1] + head * part.xs[2];
        g = reinterpret_cast<const T*>(part.g) + b * part.gs[0] + t * part.gs[1] + head * part.gs[2];
        y = reinterpret_cast<T*>(part.y) + b * part.ys[0] + t * part.ys[1] + head * part.ys[2];
    }
    __device__ __forceinline__ void next(const Params& p, int group, int a_warp) {
        const Part& part = p.part[which];
        if (++k < part.span) {
            const int on = HEADS << part.across;
            x += on * part.xs[2], g += on * part.gs[2], y += on * part.ys[2], left -= on;
        } else {
            item += gridDim.x * kWarps;
            enter(p, group, a_warp);
        }
    }
};

// What a thread reads, kStages steps ahead: its vectors, in places of its own in shared memory, so that registers hold none on
// their way and no thread waits for another.  (Vectors of 2 bytes are below what can be copied so: they are loaded when needed.)
template <typename T, int N, int VECTORS>
struct Ring {
    using V = Vec<T, N>;
    using R = typename V::type;
    static constexpr int kBytes = sizeof(R);
    static constexpr bool kAsync = kBytes >= 4;
    R* mine;      // [kStages, VECTORS], kThreads apart

    __device__ __forceinline__ R* place(int stage, int v) const { return mine + (stage * VECTORS + v) * kThreads; }
    __device__ __forceinline__ void fetch(int stage, int v, const T* from, bool is) const {
        if constexpr (kAsync) {
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(place(stage, v));
            if constexpr (kBytes == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(is ? 16 : 0) : "memory");
            else
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(kBytes), "r"(is ? kBytes : 0) : "memory");
        }
    }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory"); }
    __device__ __forceinline__ R get(int stage, int v, const T* from, bool is) const {
        if constexpr (kAsync) return *place(stage, v);
        return is ? *reinterpret_cast<const R*>(from) : V::zero();
    }
};

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
constexpr int kHeads = 2;                    // of a step, forward (backward 1; more spill, or take as long)

// A group of `lanes` lanes takes HEADS heads of one token at a step.
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(kThreads, kBlocks) k_norm_rope(const __grid_constant__ Params p, int lanes) {
    using V = Vec<T, N>;
    using R = typename V::type;
    constexpr int U = kUnits<N>, HEADS = kHeads;
    extern __shared__ __align__(16) unsigned char raw[];
    const Ring<T, N, 2 * U * HEADS> ring{reinterpret_cast<R*>(raw) + threadIdx.x};
    const int lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 31) / lanes, a_warp = 32 / lanes;
    Place at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = place<N, INTER>(lane + u * lanes, p.dim, p.rot);
    Steps<T, HEADS> ahead, now;
    ahead.begin(p, group, a_warp);
    now = ahead;
    grid_wait();
    auto fetch = [&](int stage) {
        if (!ahead.done()) {
            const int64_t apart = p.part[ahead.which].xs[2];
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool is = h < ahead.left, ha = is && at[u].a >= 0, hb = is && at[u].b >= 0;
                    const T* x = ahead.x + (is ? h * apart : 0);
                    ring.fetch(stage, (h * U + u) * 2, ha ? x + at[u].a : ahead.x, ha);
                    ring.fetch(stage, (h * U + u) * 2 + 1, hb ? x + at[u].b : ahead.x, hb);
                }
            ahead.next(p, group, a_warp);
        }
        ring.commit();
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) fetch(i);
    Turn<N, INTER> turn[U];
    bool good = true;
    for (int stage = 0; !now.done(); stage = stage + 1 == kStages ? 0 : stage + 1) {
        const Part& part = p.part[now.which];
        if (now.k == 0) {
            const int64_t pos = position(p, now.token);
            good = pos >= 0 && pos < p.table_rows;
            if (now.left > 0 && !good && lane == 0) report_device_error(p.err, 8);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float wa[N], wb[N];
                turn[u].load(p, at[u], good ? pos : 0, false);
                load_weight<T, N>(part, at[u].a, wa);
                load_weight<T, N>(part, at[u].b, wb);
                turn[u].weigh(at[u], wa, wb);
            }
        }
        ring.wait();
        R va[U][HEADS], vb[U][HEADS];
        float squares[HEADS];
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            float both[2] = {0.f, 0.f};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool is = h < now.left;
                const T* x = now.x + h * part.xs[2];
                va[u][h] = ring.get(stage, (h * U + u) * 2, x + at[u].a, is && at[u].a >= 0);
                vb[u][h] = ring.get(stage, (h * U + u) * 2 + 1, x + at[u].b, is && at[u].b >= 0);
                float f[N];
                V::get(va[u][h], f);
                dot(both, f, f);
                V::get(vb[u][h], f);
                dot(both, f, f);
            }
            squares[h] = both[0] + both[1];
        }
        sum_of_group(squares, lanes);    // (lanes without a head take part)
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            if (h >= now.left) break;
            const float rstd = rstd_of(squares[h], p);
            T* yh = now.y + h * part.ys[2];
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
        fetch(stage);
        now.next(p, group, a_warp);
    }
}

// Backward.  A lane's sums of the weights' gradients are of one part, and are put away when the other begins.  The order of the
// additions depends on the sizes, the vectors' length (strides and alignment) and the number of SMs alone.
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(kThreads, kBlocks) k_norm_rope_backward(const __grid_constant__ Params p, int lanes) {
    using V = Vec<T, N>;
    using R = typename V::type;
    constexpr int U = kUnits<N>;
    extern __shared__ __align__(16) unsigned char raw[];
    float* sums = reinterpret_cast<float*>(raw);   // [2, kWarps, dim], when there are weights
    const Ring<T, N, 4 * U> ring{reinterpret_cast<R*>(raw + (p.partial ? 2 * kWarps * kMaxDim * sizeof(float) : 0)) + threadIdx.x};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 31) / lanes, a_warp = 32 / lanes;
    for (int k = threadIdx.x; p.partial && k < 2 * kWarps * p.dim; k += kThreads) sums[k] = 0.f;
    __syncthreads();
    Place at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = place<N, INTER>(lane + u * lanes, p.dim, p.rot);
    Steps<T, 1> ahead, now;
    ahead.begin(p, group, a_warp);
    now = ahead;
    grid_wait();
    auto fetch = [&](int stage) {
        if (!ahead.done()) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool ha = ahead.left > 0 && at[u].a >= 0, hb = ahead.left > 0 && at[u].b >= 0;
                ring.fetch(stage, u * 4, ha ? ahead.x + at[u].a : ahead.x, ha);
                ring.fetch(stage, u * 4 + 1, hb ? ahead.x + at[u].b : ahead.x, hb);
                ring.fetch(stage, u * 4 + 2, ha ? ahead.g + at[u].a : ahead.g, ha);
                ring.fetch(stage, u * 4 + 3, hb ? ahead.g + at[u].b : ahead.g, hb);
            }
            ahead.next(p, group, a_warp);
        }
        ring.commit();
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) fetch(i);
    Turn<N, INTER> turn[U];
    bool good = true;
    float wa[U][N], wb[U][N], da[U][N], db[U][N];
    for (int stage = 0, which = -1; ; stage = stage + 1 == kStages ? 0 : stage + 1) {
        if (now.which != which) {
            if (which >= 0 && p.partial) {
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
            if (now.done()) break;
            which = now.which;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                load_weight<T, N>(p.part[which], at[u].a, wa[u]);
                load_weight<T, N>(p.part[which], at[u].b, wb[u]);
#pragma unroll
                for (int j = 0; j < N; ++j) da[u][j] = db[u][j] = 0.f;
            }
        }
        if (now.k == 0) {
            const int64_t pos = position(p, now.token);
            good = pos >= 0 && pos < p.table_rows;
            if (now.left > 0 && !good && lane == 0) report_device_error(p.err, 8);
#pragma unroll
            for (int u = 0; u < U; ++u) turn[u].load(p, at[u], good ? pos : 0, true);
        }
        ring.wait();
        R xa[U], xb[U];
        float squares[2] = {0.f, 0.f}, dots[2] = {0.f, 0.f};     // sums of squares and of w d x
        float ea[U][N], eb[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool ha = now.left > 0 && at[u].a >= 0, hb = now.left > 0 && at[u].b >= 0;
            float f[N], wd[N];
            xa[u] = ring.get(stage, u * 4, now.x + at[u].a, ha), xb[u] = ring.get(stage, u * 4 + 1, now.x + at[u].b, hb);
            V::get(ring.get(stage, u * 4 + 2, now.g + at[u].a, ha), ea[u]);
            V::get(ring.get(stage, u * 4 + 3, now.g + at[u].b, hb), eb[u]);
            turn[u].template apply<true>(at[u], ea[u], eb[u]);
            V::get(xa[u], f);
            dot(squares, f, f);
            mul(wd, ea[u], wa[u]);
            dot(dots, wd, f);
            V::get(xb[u], f);
            dot(squares, f, f);
            mul(wd, eb[u], wb[u]);
            dot(dots, wd, f);
        }
        float sum[2] = {squares[0] + squares[1], dots[0] + dots[1]};
        sum_of_group(sum, lanes);
        if (now.left > 0) {
            const float r = rstd_of(sum[0], p), mean = -(sum[1] * r) * p.per_dim;   // of w d times the unit row, negative
            auto half = [&](const R& v, float (&e)[N], const float (&w)[N], float (&d)[N], int to) {
                float n[N];
                V::get(v, n);
                mul(n, n, r);
                if (good) fma(d, e, n, d);
                mul(e, e, w);
                fma(e, n, mean, e);
                mul(e, e, r);
                if (to >= 0) *reinterpret_cast<R*>(now.y + to) = good ? V::put(e) : V::zero();
            };
#pragma unroll
            for (int u = 0; u < U; ++u) {
                half(xa[u], ea[u], wa[u], da[u], at[u].a);
                half(xb[u], eb[u], wb[u], db[u], at[u].b);
            }
        }
        fetch(stage);
        now.next(p, group, a_warp);
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
    auto go = [&](void (*kernel)(const Params, int), int vectors, size_t more) {
        const size_t smem = (N * sizeof(T) >= 4 ? (size_t)kStages * vectors * kThreads * N * sizeof(T) : 0) + more;
        const cudaError_t e = smem > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : cudaSuccess;
        return e != cudaSuccess ? e : launch_overlapped(kernel, dim3(grid), dim3(kThreads), smem, s, p, lanes);
    };
    if (!backward) return go(k_norm_rope<T, N, INTER>, 2 * kUnits<N> * kHeads, 0);
    return go(k_norm_rope_backward<T, N, INTER>, 4 * kUnits<N>, p.partial ? 2 * kWarps * kMaxDim * sizeof(float) : 0);
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

// Divides the tokens and their heads into items of at most `most` steps each, for groups of lanes that take `step` heads a step;
// most is what costs least: a warp's share of all steps, each item's angles counting as one more, and at the end half an item that
// some warps have and others have not.  (Measured with 1 / 4 / 16 steps at most: 8 x 4096
// tokens 561 / 342 / 325 us, 2048 tokens 16.4 / 13.5 / 21.7 us, 16 tokens 3.9 / 5.9 / 13.7 us.)  Returns the number
// of items.
int64_t split(Params& p, int groups, int step, int64_t warps) {
    double least = 0;
    int64_t items = 0;
    Params best = p;
    for (int most = 1; most <= 32; most *= 2) {
        double work = 0, longest = 0;
        int64_t all = 0;
        for (Part& t : p.part) {
            if (t.heads == 0) continue;
            const int steps = (t.heads + step - 1) / step;
            t.across = 0;
            while ((1 << t.across) < groups && (steps + (1 << t.across) - 1) >> t.across > most) ++t.across;
            const int each = (steps + (1 << t.across) - 1) >> t.across, side = groups >> t.across;
            t.chunks = (each + most - 1) / most;
            t.span = (each + t.chunks - 1) / t.chunks;
            const int64_t n = (int64_t)((p.n_tokens + side - 1) / side) * t.chunks;
            t.items = (int)std::min<int64_t>(n, 1 << 30);
            all += n, work += (double)n * (t.span + 1), longest = std::max(longest, t.span + 1.0);
        }
        const double time = all <= warps ? longest : work / warps + longest / 2;
        if (most == 1 || time < least) least = time, best = p, items = all;
    }
    p = best;
    return items;
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
    Rows xs[2], ys[2], gs[2];
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
            same = same && h.xs[i] == h.ys[i];
            // (a stride that no second row uses says nothing)
            t.xs[i] = extent[i] == 1 ? 0 : h.xs[i], t.ys[i] = extent[i] == 1 ? 0 : h.ys[i], t.gs[i] = extent[i] == 1 || !backward ? 0 : h.dys[i];
        }
        SPARK_REQUIRE(h.x != h.y || (same && !backward), SPARK_ERR_INVALID, "%s: in place needs equal strides, forward", name);
        auto rows = [&](const void* at, const int64_t* stride) {
            return Rows{at, a->dtype == SPARK_DTYPE_F32 ? 4 : 2, a->head_dim, 3, {extent[0], extent[1], extent[2]}, {stride[0], stride[1], stride[2]}};
        };
        xs[w] = rows(h.x, h.xs), ys[w] = rows(h.y, h.ys), gs[w] = rows(backward ? h.dy : nullptr, h.dys);
        SPARK_REQUIRE(rows_apart(ys[w]), SPARK_ERR_INVALID, "%s: output rows in one place", name);
        SPARK_REQUIRE(h.x == h.y || !rows_meet(ys[w], xs[w]), SPARK_ERR_INVALID, "%s: the output overlaps the input", name);
        t.x = h.x, t.y = h.y, t.g = h.dy, t.w = h.weight, t.w_dtype = (int)h.weight_dtype, t.heads = (int)h.heads;
        heads += h.heads;
    }
    if (p.part[0].heads && p.part[1].heads)
        SPARK_REQUIRE(!rows_meet(ys[0], xs[1]) && !rows_meet(ys[1], xs[0]) && !rows_meet(ys[0], ys[1]), SPARK_ERR_INVALID,
                      "%s: the output of one part is the other's input or output", name);
    for (int i = 0; i < 4 && backward; ++i)
        SPARK_REQUIRE(!p.part[i / 2].heads || !p.part[i % 2].heads || !rows_meet(ys[i / 2], gs[i % 2]), SPARK_ERR_INVALID,
                      "%s: the output overlaps a gradient", name);
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
    const int blocks = kBlocks * sm_count();
    SPARK_REQUIRE(blocks > 0, SPARK_ERR_DEVICE, "%s: no device", name);
    const int step = backward ? 1 : kHeads;
    const int64_t items = split(p, 32 / lanes, step, (int64_t)blocks * kWarps);
    SPARK_REQUIRE(items < (1ll << 30), SPARK_ERR_UNSUPPORTED, "%s: too many values for one call", name);
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
    return head_dim > 0 ? (size_t)spark::nr::kBlocks * spark::nr::sm_count() * 2 * head_dim * sizeof(float) : 0;
}

int spark_qk_norm_rope_backward(const SparkNormRope* a, void* workspace, size_t workspace_bytes, int* err, void* stream) {
    return spark::nr::run(a, true, workspace, workspace_bytes, err, reinterpret_cast<cudaStream_t>(stream),
                          "spark_qk_norm_rope_backward");
}

}  // extern "C"
