// lora.cu -- low-rank adapters of many requests beside a shared projection:
//     out[t] = y[t] + scale[a] B[a] (A[a] x[t]),   a = the adapter of token t.
//
// Two launches: h = A x (fp32, split over the input's columns where there are few
// tokens), then B h on top of y.  Tokens are taken in tiles of consecutive rows; a
// tile's items are its distinct adapters: the product of all its rows with that
// adapter's weights, of which the rows that have the adapter are kept.  Tokens of a
// request lie together, so that a prompt's tile has one or two of them, and a decoding
// batch's sixteen cost no more than reading each adapter once: nothing is sorted, and
// nothing of an adapter reaches another one's rows.
//
// Bound by memory: x, y in and out, and the weights of the adapters once.  The second product
// has three forms:
//   k_lora_up_tc   many tokens: tcgen05, 128 tokens and columns a block, y by TMA in and
//                  out.  4096 tokens, rank 32, 2560 to 9728: 57 us in all (27 us more for 4096 more: 6
//                  TB/s; 11 us are the first product, 15 the beginning), five requests 66 us (f16 68.5).
//   k_lora_up      the tiles that have more adapters than that takes, fp32 y, rows off 16
//                  bytes: mma.sync from registers.  All tiles so: 79 and 93 us.
//   k_lora_up_few  few tokens, most with an adapter of their own: no tensor cores, where 15 of 16 rows
//                  would be computed for nothing.  48 requests 14 us, one token 6.7 us.
// The first product is mma.sync throughout: rank rows are too few for tcgen05's tiles,
// and at up to 2 x 256 flop a value of x the tensor cores are not what it waits for.
//
// Fragments come straight from memory: the order of a contraction's terms is free, so
// that a lane takes 8 consecutive values of a row (16 bytes) as its share of two
// steps, and in k_lora_up the columns of a lane are 8 consecutive ones of y.
//
// h is in fp32 and meets B in 16 bits on the tensor cores: it is split into two (y in 16 bits) or
// three (fp32) terms of B's type and of its own sign, so that what is infinite in B or h is what
// the formula says.  Two are good to 2^-16 of h in bf16 (8 bits, of which the first is cut: a rest
// below 2^-7 of its power of 2, rounded at 2^-16; from |h| = 2^-110 on, as a rest of 0 counts
// 2^-126) and 2^-22 in f16, three to 2^-24.  For f16, whose exponents are few, a row is brought to
// 2^15 by a power of 2 first: its smallest step, 2^-24, is 2^-39 of the row's largest h, and no
// component of that row is better than one or, of three terms, two of those.  (Rounded terms are
// good to 2^-17, but then a rest may have the other sign; finding the infinities in the loops
// instead took prompts of 4096 tokens 2 to 8% longer.)
#include <math.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "overlap.cuh"
#include "tc_common.cuh"

namespace spark {
namespace tc {
int sm_count_cached(int dev);
int get_encoder();
int encode_2d(CUtensorMap* map, CUtensorMapDataType dt, const void* base, uint64_t inner, uint64_t outer,
              uint64_t row_stride_bytes, uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle sw);
}

namespace lora {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRank = 256;
constexpr int kRanks = 32;     // of a CTA of the first product (64 leave an SM one CTA: 512 tokens of rank 128 28.6 us instead of 21.6)
constexpr int kColumns = 32;   // of y, by one warp at a time
// Tokens up to which tiles have 16 rows, and B h is computed without tensor cores (rank 16, 2560 to 9728, us without tensor cores / with:
// 16 tokens of 16 adapters 10.0 / 11.3, 48 of 48 15.1 / 24.8, 64 of 64 19.7 / 26.2, 96 of 96 31.5 / 36.2, 64 of one 9.0 / 8.7).  From there on
// it is the number of adapters that decides, which is on the device: 64 loses nothing to speak of where all have one.
constexpr int kFew = 64;
constexpr int kFewThreads = 128;
// B h on the tensor memory, for tiles of 128 tokens that are not crowded
constexpr int kMany = 256;     // tokens from which on, and values of y: below, its beginning takes longer than it saves (measured, us
constexpr int64_t kManyValues = 1 << 23;   // without / with: 1024 x 1024 11 / 20, 512 x 9728 22.6 / 23.5, 1024 x 9728 39 / 30, 4096 x 9728 79 / 57)
constexpr int kTcRows = 128, kTcCols = 128;
constexpr int kTcRank = 64;    // ranks up to which one 128-byte row of B holds them
constexpr int kTcIds = 2;      // adapters of a tile; more: the other kernel's
constexpr int kTcStages = 4;   // blocks of y: one worked on, two on their way in, one on its way in or out
constexpr int kTcThreads = 512;

struct Params {
    const void *x, *a, *b, *y;
    void* out;
    const int* adapter;
    const float* scale;
    float scale_all;
    int64_t tokens, ic, oc, ldx, ldy, ldo;
    int64_t adapters;
    int rank, repeat;            // tokens of an entry of `adapter`
    int splits, slots;           // of the input's columns; of a tile's items, worked on side by side
    int rank_blocks, columns, run;   // first product: blocks of ranks; second: column blocks of kWarps * kColumns in y, of an item
    int wide_y;                  // rows of y and out on 16 bytes
    int* crowded;                // their number, and the tiles that the tensor memory's kernel leaves; NULL: all are the other's
    float* h;                    // [splits, tokens, rank]
    int* err;
};

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
    static __device__ __forceinline__ void run(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ __nv_bfloat16 round(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ __nv_bfloat16 cut(float x) { return __float2bfloat16_rz(x); }
    static constexpr float kTiny = 0x1p-126f;
    static __device__ __forceinline__ void round2(__nv_bfloat16* to, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(a, b); }
};
template <>
struct Mma<__half> {
    static __device__ __forceinline__ void run(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ __half round(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ __half cut(float x) { return __float2half_rz(x); }
    static constexpr float kTiny = 0x1p-24f;
    static __device__ __forceinline__ void round2(__half* to, float a, float b) { *reinterpret_cast<__half2*>(to) = __floats2half2_rn(a, b); }
};

// f(q, term) for the terms of a value of h.  All have its sign and none is 0 (unless h is): times an infinity of B they are infinities of
// one sign, where a rest of the other sign, or of 0, would make a NaN.  So all but the last are cut, not rounded, an infinity's rest is
// the infinity, and nothing finite becomes one.
template <typename T, int TERMS, typename F>
__device__ __forceinline__ void terms_of(float h, F f) {
    float rest = h;
#pragma unroll
    for (int q = 0; q < TERMS; ++q) {
        T term = q + 1 < TERMS ? Mma<T>::cut(rest) : Mma<T>::round(rest);
        const float is = (float)term;
        if (fabsf(is) < INFINITY) rest -= is;
        if (is == 0.f && h != 0.f) term = Mma<T>::round(copysignf(Mma<T>::kTiny, h));
        f(q, term);
    }
}

// The power of 2 that brings a row of h whose largest value this is to 2^15 (the first term of what is above f16's largest value is that);
// an infinity's row is brought to where all that is finite in fp32 would be.
__device__ __forceinline__ int exponent_for(float most) {
    return most < INFINITY ? most > 0.f ? min(15 - ilogbf(most), 100) : 0 : -112;
}

// A matrix's first value and what comes behind its last.
template <typename T>
struct Span {
    const T *begin, *end;
};
// The 8 values that begin `off` values into the vectors a and b, those from the n-th on zero.
__device__ __forceinline__ uint4 part_of(const uint4& a, const uint4& b, int off, int64_t n) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 6; ++j) w[j] = off & 4 ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = off & 2 ? w[j + 1] : w[j];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        w[j] = __funnelshift_r(w[j], w[j + 1], (off & 1) * 16);
        w[j] &= 2 * j >= n ? 0u : 2 * j + 1 >= n ? 0xffffu : 0xffffffffu;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Values k..k + 7 of a row of n, zeros behind its end; VEC: rows on 16 bytes, n a multiple of 8.  Else out of the two 16-byte
// vectors that they are in, where these are within the matrix.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load8(const T* row, int64_t k, int64_t n, const Span<T>& all) {
    if (k >= n) return make_uint4(0, 0, 0, 0);
    if constexpr (VEC) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + k), from = at & ~uintptr_t(15);
    const int off = (int)(at - from) / 2;
    if (from >= reinterpret_cast<uintptr_t>(all.begin) && from + (off ? 32 : 16) <= reinterpret_cast<uintptr_t>(all.end)) {
        const uint4 a = *reinterpret_cast<const uint4*>(from);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        if (off) {
            const uint4 b = *reinterpret_cast<const uint4*>(from + 16);
            w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        }
        if (off & 4) {
#pragma unroll
            for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
        }
        if (off & 2) {
#pragma unroll
            for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
        }
        if (off & 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] &= k + 2 * j >= n ? 0u : k + 2 * j + 1 >= n ? 0xffffu : 0xffffffffu;
    } else {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = k + 2 * j < n ? p[k + 2 * j] : 0, hi = k + 2 * j + 1 < n ? p[k + 2 * j + 1] : 0;
            w[j] = lo | hi << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The same without a branch, so that loads go out together, for rows `inside` the matrix: behind a row's end its beginning is read, and
// none of it taken.
template <typename T>
__device__ __forceinline__ uint4 load8_inside(const T* row, int64_t k, int64_t n) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + (k < n ? k : 0)), from = at & ~uintptr_t(15);
    const int off = (int)(at - from) / 2;
    return part_of(*reinterpret_cast<const uint4*>(from), *reinterpret_cast<const uint4*>(from + (off ? 16 : 0)), off, n - k);
}
// Whether the 16-byte vectors that hold rows first..last, of n values at distance ld, are within a matrix of `rows` such rows: 7 values
// before the first row and 15 behind the last are.
__device__ __forceinline__ bool inside(int64_t first, int64_t last, int64_t n, int64_t ld, int64_t rows) {
    return first * ld >= 7 && last < rows && last * ld + n + 15 <= (rows - 1) * ld + n;
}

// A tile's adapters: ids[row] (-1: none, or no such token), and the distinct ones in order of their first rows.
template <int ROWS>
struct Tile {
    int ids[ROWS];
    int distinct[ROWS];
    int count;
};
template <int ROWS>
__device__ __forceinline__ void load_tile(Tile<ROWS>& s, const Params& p, int64_t t0, bool report) {
    static_assert(ROWS <= 32, "a lane has a row");
    const int i = threadIdx.x;
    if (i < 32) {
        const bool is = i < ROWS && t0 + i < p.tokens;
        int id = is ? p.adapter[p.repeat == 1 ? t0 + i : (t0 + i) / p.repeat] : -1;
        if (id >= p.adapters) {
            if (report) report_device_error(p.err, 12);
            id = -1;
        }
        if (id < 0) id = -1;
        const unsigned same = __match_any_sync(0xffffffffu, is ? id : -2);
        const unsigned leads = __ballot_sync(0xffffffffu, is && __ffs(same) - 1 == i);
        if (i < ROWS) s.ids[i] = id;
        if (leads >> i & 1) s.distinct[__popc(leads & ((1u << i) - 1))] = id;
        if (i == 0) s.count = __popc(leads);
    }
    __syncthreads();
}

// The same for 128 rows: of the distinct ones the first kTcIds and their number.
struct WideTile {
    int ids[kTcRows];
    int distinct[kTcIds];
    int count;
    unsigned leads[kTcRows / 32];
};
__device__ __forceinline__ void load_wide_tile(WideTile& s, const Params& p, int64_t t0) {
    const int i = threadIdx.x, warp = i >> 5, lane = i & 31;
    const bool is = i < kTcRows && t0 + i < p.tokens;
    int id = -1;
    if (is) id = p.adapter[p.repeat == 1 ? t0 + i : (t0 + i) / p.repeat];
    if (id < 0 || id >= p.adapters) id = -1;
    if (i < kTcRows) s.ids[i] = id;
    __syncthreads();
    if (__syncthreads_and(!is || id == s.ids[0])) {
        if (i == 0) s.count = id >= 0, s.distinct[0] = id;
    } else {
        if (i < kTcRows) {
            const unsigned same = __match_any_sync(0xffffffffu, id);
            bool lead = id >= 0 && __ffs(same) - 1 == lane;
            for (int j = 0; j < warp * 32; ++j) lead = lead && s.ids[j] != id;
            const unsigned leads = __ballot_sync(0xffffffffu, lead);
            if (lane == 0) s.leads[warp] = leads;
        }
        __syncthreads();
        if (i < kTcRows) {
            int before = 0;
            for (int w = 0; w < warp; ++w) before += __popc(s.leads[w]);
            const unsigned mine = s.leads[warp];
            before += __popc(mine & ((1u << lane) - 1));
            if ((mine >> lane & 1) && before < kTcIds) s.distinct[before] = id;
            if (i == kTcRows - 1) s.count = before + (int)(mine >> 31);
        }
    }
    __syncthreads();
}

// h[split, t, :] = A[a] x[t] over the split's columns.  The warps of a CTA take chunks of 32 columns in turn.
template <typename T, int MT, int NT, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) k_lora_down(const __grid_constant__ Params p) {
    constexpr int ROWS = 16 * MT, RANKS = 8 * NT;
    __shared__ Tile<ROWS> s;
    extern __shared__ float part[];   // [kWarps, ROWS, RANKS]
    // the next launch reads what was ready before this one: it may begin when this one may
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t t0 = (int64_t)blockIdx.x * ROWS;
    if (p.crowded && blockIdx.x + blockIdx.y + blockIdx.z + threadIdx.x == 0) *p.crowded = 0;
    const int split = blockIdx.y, r0 = (int)(blockIdx.z % p.rank_blocks) * RANKS, slot = blockIdx.z / p.rank_blocks;
    load_tile(s, p, t0, split == 0 && r0 == 0 && slot == 0);
    const T* x = reinterpret_cast<const T*>(p.x);
    for (int d = slot; d < s.count; d += p.slots) {
        const int id = s.distinct[d];
        if (id < 0) continue;
        const T* a = reinterpret_cast<const T*>(p.a) + (int64_t)id * p.rank * p.ic;
        float acc[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][n][j] = 0.f;
        const Span<T> ax{reinterpret_cast<const T*>(p.a), reinterpret_cast<const T*>(p.a) + p.adapters * p.rank * p.ic};
        const Span<T> xx{x, x + (p.tokens - 1) * p.ldx + p.ic};
        struct Part {
            uint4 u[MT][2], w[NT];
        };
        // (many rows off 16 bytes: without branches where all are inside; 3019 tokens of 4217 values 167 us without, 99 with)
        const bool whole = !VEC && MT > 1 && inside(t0, t0 + ROWS - 1, p.ic, p.ldx, p.tokens) &&
                           inside((int64_t)id * p.rank + r0, (int64_t)id * p.rank + min(r0 + RANKS, p.rank) - 1, p.ic, p.ic, p.adapters * p.rank);
        auto load = [&](Part& q, int64_t k) {
            if (!VEC && MT > 1 && whole) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int e = 0; e < 2; ++e) q.u[m][e] = load8_inside(x + (t0 + m * 16 + e * 8 + g) * p.ldx, k, p.ic);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int r = r0 + n * 8 + g;
                    // (a rank behind the last: one that is there, its products are not taken)
                    q.w[n] = load8_inside(a + (int64_t)min(r, p.rank - 1) * p.ic, k, p.ic);
                }
                return;
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int64_t row = t0 + m * 16 + e * 8 + g;
                    q.u[m][e] = load8<T, VEC>(x + (row < p.tokens ? row : 0) * p.ldx, k, row < p.tokens ? p.ic : 0, xx);
                }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int r = r0 + n * 8 + g;
                q.w[n] = load8<T, VEC>(a + (int64_t)(r < p.rank ? r : 0) * p.ic, k, r < p.rank ? p.ic : 0, ax);
            }
        };
        auto products = [&](const Part& q) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    Mma<T>::run(acc[m][n], q.u[m][0].x, q.u[m][1].x, q.u[m][0].y, q.u[m][1].y, q.w[n].x, q.w[n].y);
                    Mma<T>::run(acc[m][n], q.u[m][0].z, q.u[m][1].z, q.u[m][0].w, q.u[m][1].w, q.w[n].z, q.w[n].w);
                }
        };
        // (zeros behind the end: the loop may run one part further; two parts at once take the registers of a second CTA with more)
        const int64_t step = (int64_t)p.splits * kWarps * 32;
        int64_t k = ((int64_t)split * kWarps + warp) * 32 + 8 * t;
        if constexpr (MT * NT <= 4) {
            Part q0, q1;
            load(q0, k);
            for (; k - 8 * t < p.ic; k += 2 * step) {
                load(q1, k + step);
                products(q0);
                load(q0, k + 2 * step);
                products(q1);
            }
        } else {
            Part q;
#pragma unroll 2
            for (; k - 8 * t < p.ic; k += step) {
                load(q, k);
                products(q);
            }
        }
        float* mine = part + warp * ROWS * RANKS;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    *reinterpret_cast<float2*>(mine + (m * 16 + e * 8 + g) * RANKS + n * 8 + 2 * t) =
                        make_float2(acc[m][n][2 * e], acc[m][n][2 * e + 1]);
        __syncthreads();
        for (int i = threadIdx.x; i < ROWS * RANKS; i += kThreads) {
            const int row = i / RANKS, r = r0 + i % RANKS;
            if (s.ids[row] != id || r >= p.rank) continue;
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) sum += part[w * ROWS * RANKS + i];
            p.h[((int64_t)split * p.tokens + t0 + row) * p.rank + r] = sum;
        }
        __syncthreads();
    }
}

// f(row, rank, value) for the rows' h, summed over the splits; zeros behind the rank and where the row has no adapter (or is not in
// `rows`).  Four ranks a thread where they lie on 16 bytes; four such loads are on the way together.
template <int ROWS, int THREADS, typename F>
__device__ __forceinline__ void sum_h(const Params& p, const int* ids, int64_t t0, unsigned rows, int chunks, F f) {
    const int64_t apart = p.tokens * p.rank;
    auto sum = [&](auto one, int n, int wide) {
        using V = decltype(one);
        constexpr int W = sizeof(V) / 4;
        // four values of a thread at a time, or, where there are not that many, four splits of each
        const int across = n > THREADS ? 4 : 1, along = 4 / across;
        for (int i0 = threadIdx.x; i0 < n; i0 += across * THREADS) {
            float v[4][W];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < W; ++e) v[j][e] = 0.f;
            for (int k0 = 0; k0 < p.splits; k0 += along) {
                V u[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = i0 + (across > 1 ? j * THREADS : 0), k = k0 + (across > 1 ? 0 : j), row = i / wide, r = (i - row * wide) * W;
                    const bool is = i < n && k < p.splits && ids[i < n ? row : 0] >= 0 && (rows >> (row & 31) & 1) && r < p.rank;
                    u[j] = is ? *reinterpret_cast<const V*>(p.h + k * apart + (t0 + row) * p.rank + r) : V{};
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float e[W];
                    memcpy(e, &u[j], sizeof(V));
#pragma unroll
                    for (int w = 0; w < W; ++w) (across > 1 ? v[j][w] : v[0][w]) += e[w];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = i0 + j * THREADS, row = i / wide, r = (i - row * wide) * W;
                if (j >= across || i >= n) break;
#pragma unroll
                for (int w = 0; w < W; ++w) f(row, r + w, v[j][w]);
            }
        }
    };
    if (p.rank % 4 == 0) sum(float4{}, ROWS * chunks * 8, chunks * 8);
    else sum(float{}, ROWS * chunks * 32, chunks * 32);
}

// 8 values of a row of y as floats, and back.
template <typename Y>
struct Eight;
template <>
struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    __device__ __forceinline__ float get(int j) const { return v[j]; }
    static __device__ __forceinline__ void store(float* p, const float* f) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
};
template <typename Y>
struct Eight {
    union {
        uint4 raw;
        Y v[8];
    };
    __device__ __forceinline__ Eight() {}
    __device__ __forceinline__ void load(const Y* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ float get(int j) const { return (float)v[j]; }
    static __device__ __forceinline__ void store(Y* p, const float* f) {
        Eight e;
#pragma unroll
        for (int j = 0; j < 8; j += 2) Mma<Y>::round2(e.v + j, f[j], f[j + 1]);
        *reinterpret_cast<uint4*>(p) = e.raw;
    }
    // off 16 bytes: three words on 4 bytes and the two values beside them
    static __device__ __forceinline__ void store_off(Y* p, const float* f) {
        Eight e;
#pragma unroll
        for (int j = 0; j < 8; j += 2) Mma<Y>::round2(e.v + j, f[j], f[j + 1]);
        const uint32_t w[4] = {e.raw.x, e.raw.y, e.raw.z, e.raw.w};
        const int odd = (int)(reinterpret_cast<uintptr_t>(p) >> 1 & 1);
#pragma unroll
        for (int j = 0; j < 3; ++j) *reinterpret_cast<uint32_t*>(p + 2 * j + odd) = __funnelshift_r(w[j], w[j + 1], odd * 16);
        uint16_t* const h = reinterpret_cast<uint16_t*>(p);
        h[odd ? 0 : 6] = (uint16_t)(odd ? w[0] : w[3]);
        h[7] = (uint16_t)(w[3] >> 16);
    }
};
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
template <typename Y>
__device__ __forceinline__ void put(Y* p, float v) { *p = Mma<Y>::round(v); }

// out[t, :] = y[t, :] + scale B[a] h[t], for many tokens.  An item is a run of column blocks (kColumns for each warp) of a tile, with
// every slots-th adapter and its rows: y is read for all of them at once, and written for each adapter's.  Tiles with several
// adapters take longer: their runs go to different CTAs.
template <typename T, typename Y, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) k_lora_up(const __grid_constant__ Params p) {
    constexpr int MT = 2, ROWS = 16 * MT, TERMS = sizeof(Y) == 4 ? 3 : 2;
    constexpr bool kScaled = std::is_same<T, __half>::value;
    __shared__ Tile<ROWS> s;
    __shared__ float row_scale[ROWS];
    __shared__ int mine_ids[ROWS];
    extern __shared__ __align__(16) unsigned char raw[];
    asm volatile("griddepcontrol.launch_dependents;");
    const int chunks = (p.rank + 31) / 32, ranks = chunks * 32, width = ranks + 8;
    T* terms = reinterpret_cast<T*>(raw);                                             // [TERMS, ROWS, width]
    float* sums = reinterpret_cast<float*>(raw + (size_t)TERMS * ROWS * width * sizeof(T));   // [ROWS, ranks], where rows are scaled
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const Y* y = reinterpret_cast<const Y*>(p.y);
    Y* out = reinterpret_cast<Y*>(p.out);
    const Span<T> bb{reinterpret_cast<const T*>(p.b), reinterpret_cast<const T*>(p.b) + p.adapters * p.oc * p.rank};
    constexpr int kInWide = kTcRows / ROWS;
    const int runs = (p.columns + p.run - 1) / p.run;
    bool waited = false;
    if (p.crowded) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        waited = true;
    }
    const int64_t items = (p.crowded ? (int64_t)*p.crowded * kInWide : (p.tokens + ROWS - 1) / ROWS) * runs;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        int64_t tile = item / runs;
        if (p.crowded) tile = (int64_t)p.crowded[1 + tile / kInWide] * kInWide + tile % kInWide;
        const int64_t t0 = tile * ROWS;
        const int c0 = (int)(item % runs) * p.run, n_c = min(p.run, p.columns - c0);
        __syncthreads();      // (the last tile is done with)
        if (t0 >= p.tokens) continue;
        load_tile(s, p, t0, false);
        // this slot's adapters, and a lane's rows (g, g + 8, ...) with one of them (or none, which is copied)
        const int slot = blockIdx.y;
        unsigned rows = 0;
        int n_ids = 0;
        for (int d = slot; d < s.count; d += p.slots) {
            const int id = s.distinct[d];
            if (id < 0 && p.y == p.out) continue;
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) rows |= t0 + i * 8 + g < p.tokens && s.ids[i * 8 + g] == id ? 1u << i : 0u;
            if (id < 0) continue;
            if (threadIdx.x == 0) mine_ids[n_ids] = id;
            ++n_ids;
        }
        const bool any = __syncthreads_or(rows != 0);
        const int steps = n_ids * chunks;       // of a column block: an adapter's 32 ranks each
        const Y* y_row = y + (t0 + g) * p.ldy + 8 * t;
        Y* out_row = out + (t0 + g) * p.ldo + 8 * t;
        const bool y_inside = inside(t0, t0 + ROWS - 1, p.oc, p.ldy, p.tokens) && p.oc >= 8;
        auto load_old = [&](Eight<Y> (&old)[MT][2], int c) {
            const int64_t o0 = ((int64_t)(c0 + c) * kWarps + warp) * kColumns;
            if (c >= n_c) return;
            const Y* from = y_row + o0;
            if (sizeof(Y) == 2 && !p.wide_y && y_inside) {
                if constexpr (sizeof(Y) == 2) {
                    // (rows off 16 bytes out of two vectors, and written in words: 1636 tokens to 14,423 122 us, value by value 197)
                    // (a column behind the row: its first ones, of which none is taken)
                    const int64_t back = o0 + 8 * t < p.oc ? 0 : o0 + 8 * t;
#pragma unroll
                    for (int i = 0; i < 2 * MT; ++i, from += 8 * p.ldy) old[i / 2][i % 2].raw = load8_inside(from - back, 0, 8);
                }
                return;
            }
            if (!p.wide_y || o0 + 8 * t + 8 > p.oc) {
#pragma unroll
                for (int i = 0; i < 2 * MT; ++i, from += 8 * p.ldy)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if ((rows >> i & 1) && o0 + 8 * t + j < p.oc) old[i / 2][i % 2].v[j] = from[j];
                return;
            }
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i, from += 8 * p.ldy)
                if (rows >> i & 1) old[i / 2][i % 2].load(from);
        };
        // step j of block c; behind the last step comes the next block's first
        auto load_weights = [&](uint4 (&w)[4], int c, int j) {
            if (j >= steps) ++c, j = 0;
            if (c >= n_c || steps == 0) return;
            const int id = mine_ids[chunks == 1 ? j : j / chunks], k = chunks == 1 ? 0 : j % chunks;
            const int64_t o0 = ((int64_t)(c0 + c) * kWarps + warp) * kColumns;
            // column n of a step is one of lane g / 2's eight
            const int64_t o = o0 + 8 * (g >> 1) + (g & 1);
            const T* from = bb.begin + ((int64_t)id * p.oc + o) * p.rank;
            if (o0 + kColumns <= p.oc) {
#pragma unroll
                for (int n = 0; n < 4; ++n, from += 2 * p.rank) w[n] = load8<T, VEC>(from, k * 32 + 8 * t, p.rank, bb);
            } else {
#pragma unroll
                for (int n = 0; n < 4; ++n, from += 2 * p.rank)
                    w[n] = o + 2 * n < p.oc ? load8<T, VEC>(from, k * 32 + 8 * t, p.rank, bb) : make_uint4(0, 0, 0, 0);
            }
        };
        Eight<Y> old_a[MT][2], old_b[MT][2];
        uint4 w[4];
        load_old(old_a, 0);
        load_weights(w, 0, 0);
        if (!waited) {
            // (what was ready before the first product could be read before it ends)
            asm volatile("griddepcontrol.wait;" ::: "memory");
            waited = true;
        }
        if (!any) continue;
        // h of the rows, summed over the splits
        sum_h<ROWS, kThreads>(p, s.ids, t0, 0xffffffffu, chunks, [&](int row, int r, float v) {
            if constexpr (kScaled) {
                sums[row * ranks + r] = v;
            } else {
                terms_of<T, TERMS>(v, [&](int k, T q) { terms[(k * ROWS + row) * width + r] = q; });
            }
        });
        if (threadIdx.x < ROWS) {
            const int id = s.ids[threadIdx.x];
            row_scale[threadIdx.x] = id < 0 ? 0.f : p.scale ? p.scale[id] : p.scale_all;
        }
        __syncthreads();
        if constexpr (kScaled) {
            for (int row = warp; row < ROWS; row += kWarps) {
                float most = 0.f;
                for (int r = lane; r < ranks; r += 32) most = fmaxf(most, fabsf(sums[row * ranks + r]));
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const int e = exponent_for(most);
                const float up = ldexpf(1.f, e);
                if (lane == 0) row_scale[row] *= ldexpf(1.f, -e);
                for (int r = lane; r < ranks; r += 32)
                    terms_of<T, TERMS>(sums[row * ranks + r] * up, [&](int k, T q) { terms[(k * ROWS + row) * width + r] = q; });
            }
            __syncthreads();
        }
        auto work = [&](int c, Eight<Y> (&old)[MT][2], Eight<Y> (&coming)[MT][2]) {
            load_old(coming, c + 1);
            const int64_t o0 = ((int64_t)(c0 + c) * kWarps + warp) * kColumns;
            const bool whole = p.wide_y && o0 + 8 * t + 8 <= p.oc;
            for (int d = 0; d < max(n_ids, 1); ++d) {
                const int id = n_ids > 0 ? mine_ids[d] : -1;
                __syncwarp();      // (the last adapter's rows are done with)
                float acc[MT][4][4];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[m][n][j] = 0.f;
                for (int k = 0; k < chunks && n_ids > 0; ++k) {
                    const T* a = terms + g * width + k * 32 + 8 * t;
#pragma unroll
                    for (int q = 0; q < TERMS; ++q)
#pragma unroll
                        for (int m = 0; m < MT; ++m, a += 16 * width) {
                            const uint4 lo = *reinterpret_cast<const uint4*>(a), hi = *reinterpret_cast<const uint4*>(a + 8 * width);
#pragma unroll
                            for (int n = 0; n < 4; ++n) {
                                Mma<T>::run(acc[m][n], lo.x, hi.x, lo.y, hi.y, w[n].x, w[n].y);
                                Mma<T>::run(acc[m][n], lo.z, hi.z, lo.w, hi.w, w[n].z, w[n].w);
                            }
                        }
                    load_weights(w, c, d * chunks + k + 1);
                }
                Y* to = out_row + o0;
#pragma unroll
                for (int i = 0; i < 2 * MT; ++i, to += 8 * p.ldo) {
                    const int its = s.ids[i * 8 + g];
                    if (!(rows >> i & 1) || (its != id && (its >= 0 || d > 0))) continue;
                    const float f = row_scale[i * 8 + g];
                    const float(&v)[4][4] = acc[i / 2];
                    const int e = i % 2;
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = its < 0 ? old[i / 2][e].get(j) : fmaf(v[j >> 1][2 * e + (j & 1)], f, old[i / 2][e].get(j));
                    if (whole) {
                        Eight<Y>::store(to, x);
                    } else if (sizeof(Y) == 2 && o0 + 8 * t + 8 <= p.oc) {
                        if constexpr (sizeof(Y) == 2) Eight<Y>::store_off(to, x);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (o0 + 8 * t + j < p.oc) put(to + j, x[j]);
                    }
                }
            }
        };
        for (int c = 0; c < n_c; c += 2) {
            work(c, old_a, old_b);
            if (c + 1 < n_c) work(c + 1, old_b, old_a);
        }
    }
    // (the end of this launch is to be the end of those before it)
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The same on the tensor memory, for many tokens of few adapters a tile.  D [128 tokens, 128 columns] = A B^T with the rows of h in A
// (its two terms side by side along K) and 128 rows of B[a], both in shared memory in 128-byte rows, swizzled.  Blocks of y come two
// ahead by TMA, in the same layout; a lane, which has a row of D, adds to its row of the block, and the block leaves by TMA.
// Meanwhile the next step's B arrives and is multiplied, into another part of the tensor memory.  Of a tile's two adapters each has a
// D of all rows, from which a lane takes its own: an infinity in one adapter is nothing to the other's rows.  Rows without an adapter
// go out as they came in.  Bound by memory: the products take a tenth of the time.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kTcThreads) k_lora_up_tc(const __grid_constant__ CUtensorMap y_map, const __grid_constant__ CUtensorMap out_map,
                                                         const __grid_constant__ Params p) {
    using namespace tcx;
    constexpr int TERMS = 2;
    constexpr bool kScaled = std::is_same<T, __half>::value;
    constexpr uint32_t kTypes = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
    constexpr uint32_t kIdesc = (1u << 4) | kTypes | ((uint32_t)(kTcCols >> 3) << 17) | ((uint32_t)(kTcRows >> 4) << 24);
    constexpr int kPart = kTcRows * 128, kBlock = 2 * kPart;      // bytes of 128 rows of 64 values, of a block of y
    constexpr int kWeights = kTcCols * kTcRank * 2 / 16 / kTcThreads;
    extern __shared__ uint8_t smem_raw[];
    __shared__ WideTile s;
    __shared__ float row_scale[kTcRows];
    __shared__ __align__(8) uint64_t bars[2 + kTcStages];
    __shared__ uint32_t s_tmem;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int padded = (p.rank + 15) / 16 * 16;
    uint8_t* const y_smem = smem;                                // [kTcStages]
    uint8_t* const b_smem = y_smem + kTcStages * kBlock;         // [2, kTcIds]
    uint8_t* const a_smem = b_smem + 2 * kTcIds * kPart;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t product = smem_u32(&bars[0]), arrived = smem_u32(&bars[2]);
    asm volatile("griddepcontrol.launch_dependents;");
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 + kTcStages; ++i) mbar_init(product + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(2 * kTcIds * kTcCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const Span<T> bb{reinterpret_cast<const T*>(p.b), reinterpret_cast<const T*>(p.b) + p.adapters * p.oc * p.rank};
    const int64_t blocks = (p.tokens + kTcRows - 1) / kTcRows * p.columns;
    // a CTA's blocks: an equal share of them all, or of one of its tile's `run` shares
    int64_t lo = blocks * blockIdx.x / gridDim.x, hi = blocks * (blockIdx.x + 1) / gridDim.x;
    if (p.run > 0) {
        const int64_t tile = blockIdx.x / p.run, part = blockIdx.x % p.run;
        lo = tile * p.columns + p.columns * part / p.run, hi = tile * p.columns + p.columns * (part + 1) / p.run;
    }
    bool waited = false, ok = true;
    uint32_t block = 0, products = 0;      // blocks so far; parities of the products waited for
    for (int64_t at = lo; at < hi && ok;) {
        const int64_t tile = at / p.columns, t0 = tile * kTcRows;
        const int c0 = (int)(at - tile * p.columns), n_c = (int)min((int64_t)(p.columns - c0), hi - at);
        at += n_c;
        __syncthreads();      // (the last tile is done with)
        load_wide_tile(s, p, t0);
        const int n_ids = s.count;
        if (!waited && n_ids > kTcIds) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            waited = true;
        }
        if (n_ids > kTcIds && c0 == 0 && threadIdx.x == 0) p.crowded[1 + atomicAdd(p.crowded, 1)] = (int)tile;
        if (n_ids > kTcIds || (n_ids == 0 && p.y == p.out)) continue;
        // block c of the tile, number `to`, into its stage; what left that stage has been read: all copies out but the last one have
        auto fetch = [&](int c, uint32_t to) {
            const uint32_t stage = to % kTcStages, at_smem = smem_u32(y_smem) + stage * kBlock;
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            mbar_expect_tx(arrived + 8 * stage, kBlock);
            tma_load_2d(at_smem, &y_map, (c0 + c) * kTcCols, (int)t0, arrived + 8 * stage);
            tma_load_2d(at_smem + kPart, &y_map, (c0 + c) * kTcCols + 64, (int)t0, arrived + 8 * stage);
        };
        if (threadIdx.x == 0) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            for (int c = 0; c < kTcStages - 1 && c < n_c; ++c) fetch(c, block + c);
        }
        // this thread's part of a block's B: 16 bytes of a column
        using Weights = uint4[kTcIds][kWeights];
        auto load_b = [&](Weights& w, int c) {
            const int64_t o0 = (int64_t)(c0 + c) * kTcCols;
#pragma unroll
            for (int d = 0; d < kTcIds; ++d) {
                if (d >= n_ids || c >= n_c) break;
                const T* b = bb.begin + ((int64_t)s.distinct[d] * p.oc + o0) * p.rank;
#pragma unroll
                for (int j = 0; j < kWeights; ++j) {
                    const int i = j * kTcThreads + threadIdx.x, col = i >> 3, k = (i & 7) * 8;
                    w[d][j] = o0 + col < p.oc ? load8<T, VEC>(b + col * p.rank, k, p.rank, bb) : make_uint4(0, 0, 0, 0);
                }
            }
        };
        auto put_b = [&](const Weights& w, uint32_t to) {
#pragma unroll
            for (int d = 0; d < kTcIds; ++d) {
                if (d >= n_ids) break;
                uint8_t* const at_smem = b_smem + ((to & 1) * kTcIds + d) * kPart;
#pragma unroll
                for (int j = 0; j < kWeights; ++j) {
                    const int i = j * kTcThreads + threadIdx.x, col = i >> 3, k = i & 7;
                    if (k * 8 < padded) *reinterpret_cast<uint4*>(at_smem + col * 128 + ((k ^ (col & 7)) << 4)) = w[d][j];
                }
            }
        };
        Weights w, first;
        load_b(first, 0);
        load_b(w, 1);
        if (!waited) {
            // (y was ready before the first product, and could be read before that ends)
            asm volatile("griddepcontrol.wait;" ::: "memory");
            waited = true;
        }
        // A: value (row, k) of the terms, 16 bytes of a row exchanged by its number
        auto put_terms = [&](int row, int r, float v) {
            uint8_t* const to = a_smem + row * 128;
            terms_of<T, TERMS>(v, [&](int q, T x) {
                const int k = q * padded + r, in = k & 63;
                *reinterpret_cast<T*>(to + (k >> 6) * kPart + (((in >> 3) ^ (row & 7)) << 4) + (in & 7) * 2) = x;
            });
        };
        const int chunks = (p.rank + 31) / 32, ranks = chunks * 32;
        // (the stage that no block is on its way to holds the sums before they are scaled)
        float* const sums = reinterpret_cast<float*>(y_smem + (block + kTcStages - 1) % kTcStages * kBlock);
        if (kScaled) __syncthreads();
        if (n_ids > 0)
            sum_h<kTcRows, kTcThreads>(p, s.ids, t0, 0xffffffffu, chunks, [&](int row, int r, float v) {
                if (kScaled) sums[row * ranks + r] = v;
                else if (r < padded) put_terms(row, r, v);
            });
        if (threadIdx.x < kTcRows) {
            const int id = s.ids[threadIdx.x];
            row_scale[threadIdx.x] = id < 0 ? 0.f : p.scale ? p.scale[id] : p.scale_all;
        }
        if (kScaled && n_ids > 0) {
            __syncthreads();
            for (int row = warp; row < kTcRows; row += kTcThreads / 32) {
                float most = 0.f;
                for (int r = lane; r < ranks; r += 32) most = fmaxf(most, fabsf(sums[row * ranks + r]));
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const int e = exponent_for(most);
                const float up = ldexpf(1.f, e);
                if (lane == 0) row_scale[row] *= ldexpf(1.f, -e);
                for (int r = lane; r < padded; r += 32) put_terms(row, r, sums[row * ranks + r] * up);
            }
        }
        // block number `to`
        auto multiply = [&](uint32_t to) {
            tc_fence_after();
            for (int d = 0; d < n_ids; ++d) {
                const uint32_t part = (to & 1) * kTcIds + d, a = smem_u32(a_smem), b = smem_u32(b_smem) + part * kPart;
                for (int q = 0; q < TERMS; ++q)
                    for (int k = 0; k < padded; k += 16) {
                        const int ka = q * padded + k;
                        const uint64_t da = sdesc_sw128(a + (ka >> 6) * kPart + (ka & 63) * 2), db = sdesc_sw128(b + k * 2);
                        asm volatile(
                            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem + part * kTcCols),
                            "l"(da), "l"(db), "r"(kIdesc), "r"((uint32_t)(q + k > 0))
                            : "memory");
                    }
            }
            mma_commit(product + 8 * (to & 1));
        };
        // a block's product begins two blocks before it is read back, and its B comes through registers one more before
        put_b(first, block);
        put_b(w, block + 1);
        load_b(w, 2);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0 && n_ids > 0) {
            multiply(block);
            if (n_c > 1) multiply(block + 1);
        }
        // a lane's row: one of the 32 of its warp's quarter of the tensor memory; a quarter of a block's columns
        const int across = warp >> 2, row = (warp & 3) * 32 + lane, mine = s.ids[row];
        const bool second = n_ids > 1 && mine == s.distinct[1];
        const float f = row_scale[row];
        for (int c = 0; c < n_c; ++c, ++block) {
            const uint32_t stage = block % kTcStages;
            uint8_t* const here = y_smem + stage * kBlock + (across >> 1) * kPart + row * 128;
            ok = mbar_wait(arrived + 8 * stage, block / kTcStages & 1);
            if (n_ids > 0) {
                ok = mbar_wait(product + 8 * (block & 1), products >> (block & 1) & 1) && ok;
                products ^= 1u << (block & 1);
                tc_fence_after();
            }
            if (n_ids > 0 && __all_sync(0xffffffffu, ok)) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t from = tmem + (block & 1) * kTcIds * kTcCols + across * 32 + 16 * j + ((uint32_t)((warp & 3) * 32) << 16);
                    float v[16];
                    __syncwarp();      // (rows without an adapter are ahead)
                    tmem_ld16(from, v);
                    if (n_ids > 1) {
                        float u[16];
                        tmem_ld16(from + kTcCols, u);
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = second ? u[i] : v[i];
                    }
                    if (mine < 0) continue;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint4* const place = reinterpret_cast<uint4*>(here + ((((across & 1) * 4 + 2 * j + h) ^ (row & 7)) << 4));
                        Eight<T> old;
                        old.raw = *place;
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = fmaf(v[8 * h + i], f, old.get(i));
                        Eight<T>::store(reinterpret_cast<T*>(place), x);
                    }
                }
                tc_fence_before();
            }
            if (c + 2 < n_c) put_b(w, block + 2);     // (this block's product is done with its B)
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            ok = __syncthreads_and(ok);
            if (!ok) {
                // (given up: what is still on its way into this memory ends first, or gets as long again)
                for (int i = 0; threadIdx.x == 0 && i < kTcStages - 1 && c + i < n_c; ++i) {
                    mbar_wait(arrived + 8 * ((block + i) % kTcStages), (block + i) / kTcStages & 1);
                    if (n_ids > 0 && i < 2) mbar_wait(product + 8 * ((block + i) & 1), (products >> ((block + i) & 1) & 1) ^ (i == 0));
                }
                break;
            }
            if (threadIdx.x == 0) {
                const uint32_t from = smem_u32(y_smem) + stage * kBlock;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(&out_map),
                                 "r"((c0 + c) * kTcCols + 64 * h), "r"((int)t0), "r"(from + h * kPart)
                                 : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                if (n_ids > 0 && c + 2 < n_c) multiply(block + 2);
                if (c + kTcStages - 1 < n_c) fetch(c + kTcStages - 1, block + kTcStages - 1);
            }
            load_b(w, c + 3);
        }
    }
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (threadIdx.x == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (!ok) report_device_error(p.err, 10);
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kTcIds * kTcCols) : "memory");
    }
}

// The same for few tokens, most with an adapter of their own: a tensor core's 16 rows would be one row's work and 15 others'.  A lane
// has a column of y, a warp 32, and of a tile of 16 rows every slots-th adapter: of B 32 ranks at a time in registers, for as many
// rows as have that adapter; the next adapter's are on the way meanwhile.  fp32 throughout.
template <typename T, typename Y, bool VEC>
__global__ void __launch_bounds__(kFewThreads, 5) k_lora_up_few(const __grid_constant__ Params p) {
    constexpr int ROWS = 16;
    __shared__ Tile<ROWS> s;
    __shared__ float row_scale[ROWS];
    extern __shared__ __align__(16) float h[];   // [ROWS, chunks * 32]
    asm volatile("griddepcontrol.launch_dependents;");
    const int chunks = (p.rank + 31) / 32, ranks = chunks * 32, lane = threadIdx.x & 31, slot = blockIdx.z;
    const int64_t t0 = (int64_t)blockIdx.y * ROWS, o = (int64_t)blockIdx.x * kFewThreads + threadIdx.x;
    const bool in_place = p.y == p.out;
    const Span<T> bb{reinterpret_cast<const T*>(p.b), reinterpret_cast<const T*>(p.b) + p.adapters * p.oc * p.rank};
    load_tile(s, p, t0, false);
    if (slot >= s.count) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    unsigned rows = 0;      // those of this slot
    for (int d = slot; d < s.count; d += p.slots)
        rows |= __ballot_sync(0xffffffffu, lane < ROWS && t0 + lane < p.tokens && s.ids[lane & (ROWS - 1)] == s.distinct[d]);
    auto load = [&](uint4 (&w)[4], int d, int k) {
        if (d >= s.count) return;
        const int id = s.distinct[d];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = id >= 0 && o < p.oc ? load8<T, VEC>(bb.begin + ((int64_t)id * p.oc + o) * p.rank, k * 32 + 8 * j, p.rank, bb)
                                       : make_uint4(0, 0, 0, 0);
    };
    uint4 now[4], coming[4];
    load(now, slot, 0);
    const Y* y = reinterpret_cast<const Y*>(p.y) + t0 * p.ldy + o;
    Y* out = reinterpret_cast<Y*>(p.out) + t0 * p.ldo + o;
    Y old[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if ((rows >> r & 1) && o < p.oc) old[r] = y[r * p.ldy];
    // (what was ready before the first product could be read before it ends)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    sum_h<ROWS, kFewThreads>(p, s.ids, t0, rows, chunks, [&](int row, int r, float v) { h[row * ranks + r] = v; });
    if (threadIdx.x < ROWS) {
        const int id = s.ids[threadIdx.x];
        row_scale[threadIdx.x] = id < 0 ? 0.f : p.scale ? p.scale[id] : p.scale_all;
    }
    __syncthreads();
    for (int d = slot; d < s.count; d += p.slots) {
        const int id = s.distinct[d];
        const unsigned mine = __ballot_sync(0xffffffffu, lane < ROWS && t0 + lane < p.tokens && s.ids[lane & (ROWS - 1)] == id);
        float acc[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) acc[r] = 0.f;
        for (int k = 0; k < chunks; ++k) {
            if (k + 1 < chunks) load(coming, d, k + 1);
            else load(coming, d + p.slots, 0);
            if (id >= 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (k * 32 + 8 * j >= p.rank) break;
                    T v[8];
                    memcpy(v, &now[j], 16);
                    float b[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[i] = (float)v[i];
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        if (!(mine >> r & 1)) continue;
                        const float4* hr = reinterpret_cast<const float4*>(h + r * ranks + k * 32 + 8 * j);
                        const float4 c = hr[0], e = hr[1];
                        acc[r] = fmaf(c.x, b[0], acc[r]), acc[r] = fmaf(c.y, b[1], acc[r]), acc[r] = fmaf(c.z, b[2], acc[r]);
                        acc[r] = fmaf(c.w, b[3], acc[r]), acc[r] = fmaf(e.x, b[4], acc[r]), acc[r] = fmaf(e.y, b[5], acc[r]);
                        acc[r] = fmaf(e.z, b[6], acc[r]), acc[r] = fmaf(e.w, b[7], acc[r]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) now[j] = coming[j];
        }
        if (o >= p.oc || (id < 0 && in_place)) continue;
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            if (mine >> r & 1) put(out + r * p.ldo, id < 0 ? (float)old[r] : fmaf(acc[r], row_scale[r], (float)old[r]));
    }
}

// Splits of the input's columns: as many as give two CTAs an SM work, each at least a chunk of 32 columns a warp.
int splits_of(int64_t tokens, int64_t ic, int64_t rank, int sms) {
    const int64_t rows = tokens <= kFew ? 16 : 32, tiles = (tokens + rows - 1) / rows * ((rank + kRanks - 1) / kRanks);
    const int64_t most = std::max<int64_t>(1, ic / (32 * kWarps));
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(most, 16), 2 * sms / tiles));
}

// Fewer where few tokens may have many adapters, which are worked on side by side too: each costs a beginning and an end.  (At most
// two CTAs an SM if all of a tile's are different, but two splits at least.  us without / with / with one split at least: 64 tokens of
// 64 adapters of rank 64, 4096 to 4096, 40.6 / 26 / 26, of one adapter 20.5 / 17 / 17; 62 tokens, rank 128, 3054 to 938 54 / 35 / 47;
// 48 tokens, rank 16, 2560 to 9728 16.2 / 14.3 / 14.3.)
int splits_for(const SparkLora& a, int sms) {
    const int splits = splits_of(a.tokens, a.ic, a.rank, sms);
    if (a.tokens > kFew) return splits;
    const int64_t many = std::min(std::min<int64_t>(16, a.tokens), std::min<int64_t>(std::max<int64_t>(a.adapters, 1), (a.tokens + a.repeat - 1) / a.repeat));
    const int64_t parts = (a.tokens + 15) / 16 * ((a.rank + kRanks - 1) / kRanks) * many;
    return (int)std::min<int64_t>(splits, std::max<int64_t>(2, 2 * sms / parts));
}

// The workspace: h, then the crowded tiles.
size_t h_bytes(int64_t tokens, int64_t rank, int splits) { return ((size_t)splits * tokens * rank * sizeof(float) + 15) / 16 * 16; }
size_t workspace_bytes_of(int64_t tokens, int64_t rank, int splits) {
    return h_bytes(tokens, rank, splits) + (tokens >= kMany ? (1 + (tokens + kTcRows - 1) / kTcRows) * sizeof(int) : 0);
}

template <typename F>
cudaError_t start(F kernel, dim3 grid, size_t smem, cudaStream_t s, const Params& p) {
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    return launch_overlapped(kernel, grid, dim3(kThreads), smem, s, p);
}
template <typename T, int MT, int NT>
cudaError_t down(const Params& p, bool vec, dim3 grid, cudaStream_t s) {
    const size_t smem = (size_t)kWarps * 16 * MT * 8 * NT * sizeof(float);
    return vec ? start(k_lora_down<T, MT, NT, true>, grid, smem, s, p) : start(k_lora_down<T, MT, NT, false>, grid, smem, s, p);
}
template <typename T, int MT>
cudaError_t down(const Params& p, bool vec, dim3 grid, cudaStream_t s) {
    if (p.rank <= 16) return down<T, MT, 2>(p, vec, grid, s);
    return down<T, MT, 4>(p, vec, grid, s);
}
template <typename T, typename Y>
cudaError_t up(const Params& p, bool vec, dim3 grid, bool few, cudaStream_t s) {
    const size_t ranks = (p.rank + 31) / 32 * 32;
    if (few) {
        const size_t smem = 16 * ranks * sizeof(float);
        return vec ? launch_overlapped(k_lora_up_few<T, Y, true>, grid, dim3(kFewThreads), smem, s, p)
                   : launch_overlapped(k_lora_up_few<T, Y, false>, grid, dim3(kFewThreads), smem, s, p);
    }
    const size_t smem = (sizeof(Y) == 4 ? 3 : 2) * 32 * (ranks + 8) * sizeof(T) + (std::is_same<T, __half>::value ? 32 * ranks * 4 : 0);
    return vec ? start(k_lora_up<T, Y, true>, grid, smem, s, p) : start(k_lora_up<T, Y, false>, grid, smem, s, p);
}
template <typename T>
int up_tc(const Params& p, bool vec, int grid, cudaStream_t s, const char* name) {
    const int rc = tc::get_encoder();
    if (rc) return rc;
    CUtensorMap maps[2];
    for (int i = 0; i < 2; ++i) {
        const CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        const int e = tc::encode_2d(&maps[i], type, i ? p.out : p.y, (uint64_t)p.oc, (uint64_t)p.tokens, (uint64_t)(i ? p.ldo : p.ldy) * 2, 64,
                                    kTcRows, CU_TENSOR_MAP_SWIZZLE_128B);
        if (e) return e;
    }
    const int padded = (p.rank + 15) / 16 * 16, parts = (2 * padded + 63) / 64;
    const size_t smem = 1024 + (2 * kTcStages + 2 * kTcIds + parts) * (size_t)kTcRows * 128;
    auto kernel = vec ? k_lora_up_tc<T, true> : k_lora_up_tc<T, false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = launch_overlapped(kernel, dim3((unsigned)grid), dim3(kTcThreads), smem, s, maps[0], maps[1], p);
    return e == cudaSuccess ? SPARK_OK : set_error((int)e, "%s: %s", name, cudaGetErrorString(e));
}
template <typename T>
int run(Params& p, bool vec_down, bool vec_up, bool wide, int sms, cudaStream_t s, const char* name) {
    const bool few = p.tokens <= kFew;
    {
        const int64_t rows = few ? 16 : 32, tiles = (p.tokens + rows - 1) / rows;
        p.rank_blocks = (p.rank + kRanks - 1) / kRanks;
        // (few tokens: more CTAs than find room, most of which have no adapter; 8 tokens of rank 128, 9728 to 2560, 26.8 us with half)
        p.slots = (int)std::min<int64_t>(rows, std::max<int64_t>(1, (few ? 4 : 2) * sms / (tiles * p.splits * p.rank_blocks)));
        p.slots = (int)std::min<int64_t>(p.slots, p.tokens);
        const dim3 grid((unsigned)tiles, (unsigned)p.splits, (unsigned)(p.slots * p.rank_blocks));
        const cudaError_t e = few ? down<T, 1>(p, vec_down, grid, s) : down<T, 2>(p, vec_down, grid, s);
        if (e != cudaSuccess) return set_error((int)e, "%s: launch failed: %s", name, cudaGetErrorString(e));
    }
    // few tiles are divided by their adapters too
    const int64_t rows = few ? 16 : 32, tiles = (p.tokens + rows - 1) / rows;
    dim3 grid;
    if (p.crowded) {
        p.columns = (int)((p.oc + kTcCols - 1) / kTcCols);
        // Shares of the CTAs: equal ones go over a tile's end, whose new beginning takes as long as four blocks.
        const int64_t wide_tiles = (p.tokens + kTcRows - 1) / kTcRows, blocks = wide_tiles * p.columns, parts = std::min<int64_t>(sms / wide_tiles, p.columns);
        const bool whole = parts > 0 && (p.columns + parts - 1) / parts <= (blocks + sms - 1) / sms + 4;
        p.run = whole ? (int)parts : 0;
        const int rc = up_tc<T>(p, vec_up, (int)(whole ? wide_tiles * parts : std::min<int64_t>(blocks, sms)), s, name);
        if (rc) return rc;
    }
    if (few) {
        const int64_t columns = (p.oc + kFewThreads - 1) / kFewThreads;
        p.slots = (int)std::min<int64_t>(std::min<int64_t>(rows, p.tokens), std::max<int64_t>(1, 5 * sms / (tiles * columns)));
        grid = dim3((unsigned)columns, (unsigned)tiles, (unsigned)p.slots);
    } else {
        p.columns = (int)((p.oc + kWarps * kColumns - 1) / (kWarps * kColumns));
        p.run = (int)std::min<int64_t>(4, std::max<int64_t>(1, tiles * p.columns / (8 * sms)));
        const int64_t items = tiles * ((p.columns + p.run - 1) / p.run);
        p.slots = (int)std::min<int64_t>(rows, std::max<int64_t>(1, 2 * sms / items));
        grid = dim3((unsigned)std::min<int64_t>(items, std::max(1, 2 * sms / p.slots)), (unsigned)p.slots);
    }
    const cudaError_t e = wide ? up<T, float>(p, vec_up, grid, few, s) : up<T, T>(p, vec_up, grid, few, s);
    return e == cudaSuccess ? SPARK_OK : set_error((int)e, "%s: launch failed: %s", name, cudaGetErrorString(e));
}

}  // namespace lora
}  // namespace spark

extern "C" {

size_t spark_lora_workspace_size(int64_t tokens, int64_t ic, int64_t rank) {
    using namespace spark;
    int dev = 0;
    if (tokens <= 0 || ic <= 0 || rank <= 0 || cudaGetDevice(&dev) != cudaSuccess) return 0;
    return lora::workspace_bytes_of(tokens, rank, lora::splits_of(tokens, ic, rank, tc::sm_count_cached(dev)));
}

int spark_lora(const SparkLora* a, void* workspace, size_t workspace_bytes, int* err, void* stream) {
    using namespace spark;
    using namespace spark::lora;
    const char* name = "spark_lora";
    SPARK_REQUIRE(a, SPARK_ERR_INVALID, "%s: null pointer", name);
    SPARK_REQUIRE(a->dtype == SPARK_DTYPE_BF16 || a->dtype == SPARK_DTYPE_F16, SPARK_ERR_INVALID, "%s: bad dtype %d", name, (int)a->dtype);
    SPARK_REQUIRE(a->y_dtype == a->dtype || a->y_dtype == SPARK_DTYPE_F32, SPARK_ERR_INVALID, "%s: y is of dtype or fp32, got %d", name,
                  (int)a->y_dtype);
    SPARK_REQUIRE(a->tokens >= 0 && a->ic >= 1 && a->oc >= 0 && a->adapters >= 0 && a->repeat >= 1, SPARK_ERR_INVALID, "%s: bad size", name);
    SPARK_REQUIRE(a->rank >= 1 && a->rank <= kMaxRank, SPARK_ERR_UNSUPPORTED, "%s: rank %lld is not in 1..%d", name, (long long)a->rank, kMaxRank);
    SPARK_REQUIRE(a->tokens < (1 << 26) && a->ic < (1 << 26) && a->oc < (1 << 26) && a->adapters < (1ll << 31) && a->repeat < (1ll << 31),
                  SPARK_ERR_UNSUPPORTED, "%s: size", name);
    if (a->tokens == 0 || a->oc == 0) return SPARK_OK;
    SPARK_REQUIRE(a->x && a->y && a->out && a->adapter && ((a->a && a->b) || a->adapters == 0), SPARK_ERR_INVALID, "%s: null pointer", name);
    SPARK_REQUIRE(a->tokens == 1 || a->ldo >= a->oc, SPARK_ERR_INVALID, "%s: output rows in one place", name);
    SPARK_REQUIRE(a->out != a->y || a->ldo == a->ldy || a->tokens == 1, SPARK_ERR_INVALID, "%s: in place needs equal strides", name);
    const Rows out{a->out, a->y_dtype == SPARK_DTYPE_F32 ? 4 : 2, a->oc, 1, {a->tokens}, {a->ldo}};
    const Rows y{a->y, out.item, a->oc, 1, {a->tokens}, {a->ldy}}, x{a->x, 2, a->ic, 1, {a->tokens}, {a->ldx}};
    SPARK_REQUIRE(!rows_meet(out, x) && (a->out == a->y || !rows_meet(out, y)), SPARK_ERR_INVALID, "%s: the output overlaps an input", name);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return set_error((int)e, "%s: %s", name, cudaGetErrorString(e));
    const int sms = tc::sm_count_cached(dev);
    Params p{};
    p.splits = splits_for(*a, sms);
    const size_t need = spark_lora_workspace_size(a->tokens, a->ic, a->rank);
    SPARK_REQUIRE(workspace && workspace_bytes >= need && aligned(workspace, 16), SPARK_ERR_WORKSPACE,
                  "%s: workspace of %zu bytes on 16, %zu needed", name, workspace_bytes, need);
    p.x = a->x, p.a = a->a, p.b = a->b, p.y = a->y, p.out = a->out, p.adapter = a->adapter, p.scale = a->scale;
    p.scale_all = (float)a->scale_all;
    p.tokens = a->tokens, p.ic = a->ic, p.oc = a->oc, p.adapters = a->adapters;
    // (a stride that no second row uses says nothing)
    p.ldx = a->tokens == 1 ? 0 : a->ldx, p.ldy = a->tokens == 1 ? 0 : a->ldy, p.ldo = a->tokens == 1 ? 0 : a->ldo;
    p.rank = (int)a->rank, p.repeat = (int)a->repeat;
    p.h = reinterpret_cast<float*>(workspace), p.err = err;
    const int items = a->y_dtype == SPARK_DTYPE_F32 ? 4 : 8;   // of y, in 16 bytes
    p.wide_y = aligned(p.y, 16) && aligned(p.out, 16) && p.ldy % items == 0 && p.ldo % items == 0;
    const bool vec_down = p.ic % 8 == 0 && p.ldx % 8 == 0 && aligned(p.x, 16) && aligned(p.a, 16);
    const bool vec_up = p.rank % 8 == 0 && aligned(p.b, 16), wide = a->y_dtype == SPARK_DTYPE_F32;
    // (the tensor maps' rows are on 16 bytes, apart)
    if (p.tokens >= kMany && p.tokens * p.oc >= kManyValues && p.rank <= kTcRank && !wide && p.wide_y && p.ldy >= p.oc)
        p.crowded = reinterpret_cast<int*>(reinterpret_cast<char*>(workspace) + h_bytes(p.tokens, p.rank, p.splits));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int rc = a->dtype == SPARK_DTYPE_BF16 ? run<__nv_bfloat16>(p, vec_down, vec_up, wide, sms, st, name)
                                                : run<__half>(p, vec_down, vec_up, wide, sms, st, name);
    if (rc) return rc;
    return check_launch(name);
}

}  // extern "C"
