// tree_attention.cu -- attention of a tree of drafted tokens over a paged K/V
// cache and over the tree itself, on the 5th-generation tensor cores.
//
// Node t sees the context (all lens[b] tokens of the cache), itself and its
// ancestors.  The queries of one kv head (nodes x the heads that share it) are
// the rows of one matrix Q, so that a tile of keys is read once for all of
// them: S = Q K^T, then per row the running maximum m and sum l of the softmax
//     m' = max(m, max S), l' = l 2^(m - m') + sum 2^(S - m'),
//     O' = O 2^(m - m') + 2^(S - m') V          (S in units of log 2).
// Scores, m, l and O are fp32; the weights 2^(S - m) are rounded to the cache's
// type for the second product, as the tensor cores take them (their relative
// error, at most 2^-9 in bf16, is independent from weight to weight).  O is
// rescaled only when m grows by more than 2^8 -- weights up to 2^8 are as exact
// as those below 1 -- since a rescale is a round trip of O through registers.
// The tensor cores cut a product off at 2^-25 of the O that it is added to: next
// to one token, n others of 2^-25 of its weight lose up to n 2^-25 of the sum
// (two tokens and 262144 others of 2^-25.3 of them: half of the others' 0.3 % of
// the sum).
//
// Work: an item is (sequence, kv head, tile of rows), its tiles are the context
// in steps of 128 tokens (64 for heads above 128 wide) and last the tree.  All tiles of all items form one
// sequence cut into equal contiguous ranges, one per CTA (one CTA per SM), so
// that ragged batches and single long sequences fill the GPU alike without the
// host knowing the lengths.  Where a range cuts an item, the parts leave O, m
// and l in the workspace; once all parts of an item are there (the launch is
// cooperative, all CTAs run at the same time and end their ranges at about the
// same time) its CTAs add them, each a share of the values, in the CTAs' order:
// the result does not depend on timing.
//
// Roles (384 threads):
//   warps 0-3, 4-7  softmax: two groups (streams), a thread owns one row (TMEM
//                   lane).  Up to 128 rows (whole nodes): both groups have the same
//                   rows and take tiles in turn, each with its own m, l and O, added
//                   at the end of the item.  Above: group g has its own rows, the
//                   item's g-th 128, and takes every tile.  Heads above 128 wide leave room for
//                   one O only: group 0 works alone, on two score buffers in turn.
//                   The group writes its weights over the scores they came from (the
//                   A operand of the second product is read from TMEM).
//   warps 8, 9      load K and V tiles by TMA, page by page, each into a ring of
//                   slots of its own.
//   warp 11         loads Q, the next item's while the last one still ends.
//   warp 10         allocates TMEM and issues the MMAs.  It and the loaders run whole
//                   and elect a lane for each instruction, so that the operands stay
//                   in uniform registers: under a branch on the lane an MMA took 110
//                   cycles to issue and a load 500, more than they take to run.
// What bounds it.  A tile of 128 tokens x 128 values is 64 KB of K and V: 2670
// cycles of an SM's share of HBM at 1.8 GHz, against 1024 of tensor cores for a
// stream's 128 rows (an MMA of 128 x 128 x 16 takes 64, also with Q from shared
// memory; 128 x 64 from shared memory takes 48, so that tiles of 64 tokens cost
// more) and about 2100 of softmax (1024 of them the exponential unit's).  In turns
// two streams hide each other's chains and HBM bounds: 16 sequences of up to 32k
// tokens, 128 rows, 2430 cycles a tile, 290 us (5.7 TB/s).  By rows a tile is
// 2 x (1024 + 2100) cycles of work on two engines that wait for each other: 64
// nodes x 8 heads over 65k tokens, 3990 cycles a tile, 129-135 us (0.9 PFLOP/s), where
// neither is full.  Both run into the power cap when repeated (1000 W at 1.4 GHz:
// 331-341 us, 155-158 us).  Small calls are their start (5 us to the first scores: lengths,
// page numbers and the first tile are three round trips to memory) and their end
// (about 6 us: the parts' stores made visible, counted, read and added).  Many
// short contexts are a chain for each item (about 8500 cycles for 88 tokens and 8
// nodes: 700 to find it, 3500 of softmax, 2000 of products, 2000 to write O): 800
// items 44 us.
//
// Every wait is bounded (2 s); one that expires sets error 10 and all roles end.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>

#include <algorithm>
#include <mutex>

#include "common.cuh"
#include "tc_common.cuh"

namespace spark {
int check_cache(const SparkPagedCache* c, const char* who);
namespace tc {
int get_encoder();
int encode_4d(CUtensorMap* map, CUtensorMapDataType dt, const void* base, const uint64_t* dims,
              const uint64_t* stride_bytes, const uint32_t* box, CUtensorMapSwizzle sw);
int sm_count_cached(int dev);
}  // namespace tc

namespace ta {
using namespace tcx;

constexpr int kThreads = 384;
constexpr int kKWarp = 8, kVWarp = 9, kMmaWarp = 10, kQWarp = 11;
constexpr int kMaxSlots = 12;   // of one ring
constexpr int kHeader = 3 * 1024;   // barriers and the exchange of the two groups
constexpr uint32_t kTmemCols = 512;

// DP: head_dim padded to 64, 128 or 256.
template <int DP>
struct Cfg {
    static constexpr bool kOne = DP == 256;                // one O, one softmax group
    static constexpr int kTok = kOne ? 64 : 128;           // tokens of a tile
    static constexpr int kChunks = DP / 64;                // 128-byte columns of a tile
    static constexpr int kSlotBytes = kTok * DP * 2;       // 16 or 32 KB
    static constexpr int kQBytes = 128 * DP * 2;           // one 128-row Q tile
    static constexpr uint32_t kOCol = 256;                 // first column of O; before it two S buffers
};

struct Params {
    SparkTreeAttention a;
    int* err;
    float4* part;           // [2 * grid][DP / 4][rows] O of cut items
    float2* part_ml;        // [2 * grid][rows] their m, l
    int* count;             // [grid][2] warps that left their part of the item cut first in a CTA, that added it
    int rows_item, row_tiles, group, box_rows, by_rows, tok, per_seq;   // per_seq: items of a sequence
    int tile_nodes, item_nodes;   // nodes of a 128-row tile, of an item (two tiles by_rows)
    float inv_group, inv_rows;    // 1 / group, 1 / rows_item: (n + 0.5) times them is exact enough to divide n < 2^16
    int slots[2];           // of K, of V
    float scale;            // times log2 e
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

__device__ __forceinline__ int context_len(const Params& p, int64_t b) {
    const int64_t room = p.a.cache.max_pages * p.a.cache.page_size, len = p.a.cache.lens[b];
    return (int)(len < 0 ? 0 : (len > room ? room : len));
}

// Starting an item (loading Q, filling the pipeline, writing O) costs as much as
// this many tiles: the cut into ranges counts them in front of the item's own.
constexpr int kStart = 3;
// Places of an item of sequence b (all items' are below 2^31: the host checks it by the longest context the pages hold)
__device__ __forceinline__ int tiles_of(const Params& p, int b) {
    return b < (int)p.a.batch ? (context_len(p, b) + p.tok - 1) / p.tok + 1 + kStart : 0;
}
// Number of tiles of all items, by one warp.
__device__ __forceinline__ int count_tiles(const Params& p, int lane) {
    int total = 0;
    for (int b = lane; b < (int)p.a.batch; b += 32) total += tiles_of(p, b);
    return (int)__reduce_add_sync(0xffffffffu, (unsigned)total) * p.per_seq;
}
// The sequence and its item that hold place `pos` of all, and the place in the item, by one warp.
__device__ __forceinline__ void locate(const Params& p, int lane, int pos, int& b, int& item, int& off) {
    int at = 0;
    b = (int)p.a.batch, item = off = 0;
    for (int base = 0; base < (int)p.a.batch; base += 32) {
        const int places = tiles_of(p, base + lane), n = places * p.per_seq;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && pos < at + sum);
        if (hit) {
            const int l = __ffs(hit) - 1;
            b = base + l;
            off = pos - (at + __shfl_sync(0xffffffffu, sum - n, l));
            const int of_item = __shfl_sync(0xffffffffu, places, l);
            item = off / of_item;
            off -= item * of_item;
            return;
        }
        at += __shfl_sync(0xffffffffu, sum, 31);
    }
}

// A run of tiles of one item.
struct Segment {
    int b, head, rt, t0, t1, tiles, len;   // tiles t0..t1-1 of `tiles`; the last is the tree
    int lo;                                // place of tile 0 among all
};

// Walks `left` places from place `at` of an item of sequence b on; a run may be
// empty where the range ends in front of an item's own tiles.
struct Walker {
    const Params& p;
    int b, head, rt, at, left, pos;
    __device__ Walker(const Params& q, int b0, int item, int off, int n, int first)
        : p(q), b(b0), head(item / q.row_tiles), rt(item - head * q.row_tiles), at(off), left(n), pos(first) {}
    __device__ bool next(Segment& s) {
        while (left > 0 && b < (int)p.a.batch) {
            s.len = context_len(p, b);
            s.tiles = (s.len + p.tok - 1) / p.tok + 1;
            s.b = b, s.head = head, s.rt = rt;
            const int n = min(s.tiles + kStart - at, left);
            s.t0 = max(at - kStart, 0);
            s.t1 = at + n - kStart;
            s.lo = pos - at + kStart;
            pos += n;
            left -= n;
            at = 0;
            if (++rt == p.row_tiles) {
                rt = 0;
                if (++head == (int)p.a.cache.kv_heads) head = 0, ++b;
            }
            if (s.t1 > s.t0) return true;
        }
        return false;
    }
};

// A bounded wait that reads the clock only every 64 tries.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity) {
    uint64_t deadline = 0;
    for (int i = 1;; ++i) {
        if (mbar_try(bar, parity)) return true;
        if ((i & 63) == 0) {
            const uint64_t now = globaltimer_ns();
            if (deadline == 0) deadline = now + kWaitNs;
            if (now > deadline) return false;
        }
    }
}

// 64 consecutive entries of a sequence's page table in a warp's registers, the
// later half loaded ahead of its use: a load's page number costs no round trip
// to memory (that alone was 0.8 us per K or V tile).
struct Pages {
    const int* table;
    int n, base, cur, nxt;
    __device__ int entry(int i) const { return i < n ? table[i] : 0; }
    __device__ void start(const int* t, int entries, int first, int lane) {
        table = t, n = entries, base = first;
        cur = entry(base + lane), nxt = entry(base + 32 + lane);
    }
    // makes entries first .. first + 32 available
    __device__ void advance(int first, int lane) {
        while (first >= base + 32) base += 32, cur = nxt, nxt = entry(base + 32 + lane);
    }
    __device__ int at(int i) const {   // every lane of the warp, i within the window
        const int o = i - base, a = __shfl_sync(0xffffffffu, cur, o & 31), b = __shfl_sync(0xffffffffu, nxt, o & 31);
        return o < 32 ? a : b;
    }
};

// An item that this CTA has a part of, with CTAs c0 .. c0 + parts - 1.
struct Cut {
    Segment sg;
    int c0, parts;
};

struct Smem {
    uint64_t full[2][kMaxSlots], empty[2][kMaxSlots];   // [K, V]
    uint64_t q_full, q_free, s_full[2], p_full[2], pv_done, merge, done, ended, cuts_known;   // [score buffer]; pv_done: kOne
    uint32_t tmem;
    int cuts;                // items in parts: at most the range's first and its last
    Cut cut[2];
    int bad_v[2];            // the segment (one of each parity) whose tree values hold an infinity or NaN
    float2 ml[2][128];
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}
// D (+)= A B, both from shared memory; the descriptors' high halves are constant
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
// D (+)= A B, A from TMEM
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Halves of a shared-memory operand descriptor, 128-byte swizzle.  Low: address
// and leading offset; high: stride offset (groups of eight rows 1024 bytes apart),
// version and swizzle mode.  K-major (Q, K) does not use the leading offset; for
// N-major V it is the distance of the 64-column chunks.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t chunk_bytes) { return (addr >> 4) | (chunk_bytes >> 4) << 16; }
// 32 consecutive TMEM columns of this warp's 32 lanes; wait with tmem_wait_ld
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (BF)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ bool all_ok(bool ok) { return __all_sync(0xffffffffu, ok); }

__device__ __forceinline__ void add_release(int* p, int v) {
    asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
__device__ __forceinline__ int load_acquire(const int* p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// CTAs that get places (no more than there are), the first place of one, and the one that has place `pos`.
__device__ __forceinline__ int ctas(int total) { return min(total, (int)gridDim.x); }
__device__ __forceinline__ int first_tile(int total, int cta) { return (int)((uint64_t)total * cta / (unsigned)ctas(total)); }
__device__ __forceinline__ int cta_of(int total, int pos) {
    return (int)(((uint64_t)(pos + 1) * ctas(total) - 1) / (unsigned)total);
}

// Scores that a row does not see: of 64, those of the tree outside its mask, of the context from `valid` (> 0) on.
__device__ __forceinline__ void hide(float (&x)[64], bool tree, uint64_t mask, int valid) {
    const uint64_t sees = tree ? mask : (valid >= 64 ? ~0ull : (1ull << valid) - 1);   // (h < valid; the tree has one run of 64)
    const uint32_t lo = (uint32_t)sees, hi = (uint32_t)(sees >> 32);
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        if (!(lo & (1u << e))) x[e] = -INFINITY;
        if (!(hi & (1u << e))) x[e + 32] = -INFINITY;
    }
}

// The node and query head of a row of an item, -1 where it has none.
__device__ __forceinline__ int node_of(const Params& p, const Segment& sg, int row, int& head) {
    const int in = p.by_rows ? row & 127 : row, t = (int)((in + 0.5f) * p.inv_group);
    head = sg.head * p.group + in - t * p.group;
    const int node = sg.rt * p.item_nodes + (p.by_rows ? (row >> 7) * p.tile_nodes : 0) + t;
    return t < p.tile_nodes && node < (int)p.a.nodes ? node : -1;
}

// Waits until all parts of an item are there, and says that this warp knows.
// The last warp to know clears the counters for the next call.
__device__ __forceinline__ bool await_parts(int* count, int parts, int lane) {
    bool ok = true;
    if (lane == 0) {
        uint64_t deadline = 0;
        for (int i = 1; load_acquire(count) < 8 * parts && ok; ++i)
            if ((i & 63) == 0) {
                const uint64_t now = globaltimer_ns();
                if (deadline == 0) deadline = now + kWaitNs;
                ok = now <= deadline;
            }
        if (ok && atomicAdd(count + 1, 1) == 8 * parts - 1) count[0] = 0, count[1] = 0;
    }
    return all_ok(ok);
}

// This warp's share of the sum of an item's parts.  A lane adds U times four
// columns of a row, PU parts loaded together: the loads' latency is what this
// costs, about a microsecond a round.
template <int DP, bool BF, int U, int PU>
__device__ __forceinline__ void add_parts(const Params& p, const Segment& sg, int c0, int parts) {
    const SparkTreeAttention& a = p.a;
    const int rows = p.rows_item, n = rows * (int)((a.cache.head_dim + 3) / 4), step = parts * 256;
#pragma unroll 1
    for (int e0 = ((int)blockIdx.x - c0) * 256 + (int)threadIdx.x; e0 < n; e0 += U * step) {
        float top[U], sum[U];
        float4 o[U];
        int row[U], col[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            top[k] = -INFINITY, sum[k] = 0.f, o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            col[k] = (int)((e0 + k * step + 0.5f) * p.inv_rows);
            row[k] = e0 + k * step - col[k] * rows;
        }
#pragma unroll 1
        for (int q = 0; q < parts; q += PU) {
            float2 ml[PU][U];
            float4 v[PU][U];
#pragma unroll
            for (int i = 0; i < PU; ++i)
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    ml[i][k] = make_float2(-INFINITY, 0.f);
                    v[i][k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (q + i < parts && e0 + k * step < n) {
                        const int slot = 2 * (c0 + q + i) + (q + i == 0 ? 1 : 0);
                        ml[i][k] = __ldcg(p.part_ml + slot * rows + row[k]);
                        v[i][k] = __ldcg(p.part + (slot * (DP / 4) + col[k]) * rows + row[k]);
                    }
                }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                float m2 = top[k];
#pragma unroll
                for (int i = 0; i < PU; ++i) m2 = ml[i][k].y == 0.f ? m2 : fmaxf(m2, ml[i][k].x);
                const float f = sum[k] == 0.f ? 0.f : exp2_approx(top[k] - m2);
                top[k] = m2;
                sum[k] *= f;
                o[k].x *= f, o[k].y *= f, o[k].z *= f, o[k].w *= f;
#pragma unroll
                for (int i = 0; i < PU; ++i) {
                    const float g = ml[i][k].y == 0.f ? 0.f : exp2_approx(ml[i][k].x - m2);
                    sum[k] += ml[i][k].y * g;
                    if (g == 0.f) v[i][k] = make_float4(0.f, 0.f, 0.f, 0.f);   // (an infinity of no weight)
                    o[k].x += v[i][k].x * g, o[k].y += v[i][k].y * g, o[k].z += v[i][k].z * g, o[k].w += v[i][k].w * g;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            int head;
            const int node = e0 + k * step < n ? node_of(p, sg, row[k], head) : -1;
            if (node < 0) continue;
            const float norm = sum[k] == 0.f ? 0.f : __fdividef(1.f, sum[k]);
            uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)sg.b * a.out_stride[0] + node * a.out_stride[1] + head * a.out_stride[2];
            *reinterpret_cast<uint2*>(out + col[k] * 4) =
                make_uint2(pack2<BF>(o[k].x * norm, o[k].y * norm), pack2<BF>(o[k].z * norm, o[k].w * norm));
            if (a.lse && col[k] == 0)
                a.lse[((int64_t)sg.b * a.nodes + node) * a.q_heads + head] =
                    sum[k] == 0.f ? -INFINITY : (__log2f(sum[k]) + top[k]) * 0.6931471805599453f;
        }
    }
}

template <int DP, bool BF>
__global__ void __launch_bounds__(kThreads, 1)
    k_tree_attention(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ CUtensorMap ktmap, const __grid_constant__ CUtensorMap vtmap,
                     const __grid_constant__ Params p) {
    using C = Cfg<DP>;
    constexpr int kTok = C::kTok;
    extern __shared__ __align__(1024) uint8_t smem[];
    const bool by_rows = p.by_rows;
    uint8_t* q_smem = smem + (size_t)(p.slots[0] + p.slots[1]) * C::kSlotBytes;   // after the slots of K and of V
    Smem& sm = *reinterpret_cast<Smem*>(q_smem + (size_t)(by_rows ? 2 : 1) * C::kQBytes);
    const SparkTreeAttention& a = p.a;
    const SparkPagedCache& c = a.cache;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == kKWarp) {
        if (lane < kMaxSlots)
            for (int v = 0; v < 2; ++v) mbar_init(smem_u32(&sm.full[v][lane]), 1), mbar_init(smem_u32(&sm.empty[v][lane]), 1);
        if (lane == 0) {
            mbar_init(smem_u32(&sm.q_full), 1);
            mbar_init(smem_u32(&sm.q_free), 1);
            mbar_init(smem_u32(&sm.cuts_known), 1);
            mbar_init(smem_u32(&sm.ended), 8);
            for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&sm.s_full[i]), 1), mbar_init(smem_u32(&sm.p_full[i]), 4);
            mbar_init(smem_u32(&sm.pv_done), 1);
            mbar_init(smem_u32(&sm.merge), 8);
            mbar_init(smem_u32(&sm.done), 1);
            sm.bad_v[0] = sm.bad_v[1] = 0;
            if ((smem_u32(smem) & 1023) != 0) report_device_error(p.err, 10);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (lane == 0 && warp >= kKWarp) {
        const CUtensorMap* mine = warp == kKWarp ? &kmap : warp == kVWarp ? &vmap : warp == kQWarp ? &qmap : &ktmap;
        asm volatile("prefetch.tensormap [%0];" ::"l"(mine) : "memory");
        if (warp == kMmaWarp) asm volatile("prefetch.tensormap [%0];" ::"l"(&vtmap) : "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 0 && blockIdx.x == 0)
        for (int64_t b = lane; b < a.batch; b += 32)
            if (c.lens[b] < 0 || c.lens[b] > c.max_pages * c.page_size) report_device_error(p.err, 9);
    // this CTA's range of the tiles; every warp finds it for itself
    const int total = count_tiles(p, lane);
    const bool idle = (int)blockIdx.x >= ctas(total);
    const int range0 = idle ? total : first_tile(total, blockIdx.x), range1 = idle ? total : first_tile(total, blockIdx.x + 1);
    int b0, item0, off0;
    locate(p, lane, range0, b0, item0, off0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    const int count = (smem_u32(smem) & 1023) ? 0 : range1 - range0;
    Walker walk(p, b0, item0, off0, count, range0);
    Segment sg;
    bool ok = true;

    if (warp == kKWarp || warp == kVWarp) {
        // ------------------------------------------------------------ loads
        const int v = warp - kKWarp, slots = p.slots[v], page_size = (int)c.page_size;
        const uint32_t ring = smem_u32(smem) + (uint32_t)(v ? p.slots[0] : 0) * C::kSlotBytes;
        const CUtensorMap* ctx_map = v ? &vmap : &kmap;
        const CUtensorMap* tree_map = v ? &vtmap : &ktmap;
        int at = 0, filled = 0;
        uint32_t phase = 1;
        while (ok && walk.next(sg)) {
            int page_at = sg.t0 * kTok / page_size, row = sg.t0 * kTok - page_at * page_size;
            Pages pages;
            pages.start(c.page_table + (int64_t)sg.b * c.page_table_stride, (sg.len + page_size - 1) / page_size, page_at, lane);
            for (int tile = sg.t0; tile < sg.t1; ++tile) {
                const uint32_t bar = smem_u32(&sm.full[v][at]), slot = ring + (uint32_t)at * C::kSlotBytes;
                ok = all_ok(wait_bar(smem_u32(&sm.empty[v][at]), phase));
                if (!ok) break;
                if (++at == slots) at = 0, phase ^= 1;
                ++filled;
                if (tile == sg.tiles - 1) {
                    if (elect_one()) {
                        mbar_expect_tx(bar, 64 * C::kChunks * 128);
#pragma unroll
                        for (int k = 0; k < C::kChunks; ++k)
                            tma_load_4d(slot + k * kTok * 128, tree_map, k * 64, sg.head, 0, sg.b, bar);
                    }
                    __syncwarp();
                    continue;
                }
                const int boxes = (min(kTok, sg.len - tile * kTok) + p.box_rows - 1) / p.box_rows;
                pages.advance(page_at, lane);
                // four boxes at a time under one election
#pragma unroll 1
                for (int box = 0; box < boxes; box += 4) {
                    int page[4], first[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        page[i] = pages.at(page_at), first[i] = row;
                        if (box + i < boxes && (row += p.box_rows) == page_size) row = 0, ++page_at;
                    }
                    if (elect_one()) {
                        if (box == 0) mbar_expect_tx(bar, (uint32_t)(boxes * p.box_rows) * (C::kChunks * 128));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (box + i >= boxes) break;
                            if (page[i] < 0 || page[i] >= c.pages) report_device_error(p.err, 9);   // the load gives zeros
#pragma unroll
                            for (int k = 0; k < C::kChunks; ++k)
                                tma_load_4d(slot + (uint32_t)(k * kTok + (box + i) * p.box_rows) * 128, ctx_map, k * 64, sg.head, first[i],
                                            page[i], bar);
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok)   // a wait expired: let the loads in flight land before the CTA ends
            for (int i = 0; i < min(filled, slots); ++i)
                wait_bar(smem_u32(&sm.full[v][i]), (uint32_t)((filled - 1 - i) / slots) & 1);
    } else if (warp == kQWarp) {
        // a tile of Q is the heads of the group of tile_nodes nodes, node by node
        const uint32_t qb = smem_u32(q_smem), bar = smem_u32(&sm.q_full);
        const uint32_t bytes = (uint32_t)(p.tile_nodes * p.group) * (C::kChunks * 128);
        int seg = 0, cuts = 0;
        for (; ok && walk.next(sg); ++seg) {
            if (sg.t1 - sg.t0 < sg.tiles) {
                const int c0 = cta_of(total, sg.lo), c1 = cta_of(total, sg.lo + sg.tiles - 1);
                if (lane == 0) sm.cut[cuts] = Cut{sg, c0, c1 - c0 + 1};
                ++cuts;
            }
            ok = all_ok(seg == 0 || wait_bar(smem_u32(&sm.q_free), (seg - 1) & 1));
            if (!ok) break;
            if (elect_one()) {
                mbar_expect_tx(bar, by_rows ? 2 * bytes : bytes);
                for (int t = 0; t < (by_rows ? 2 : 1); ++t)
#pragma unroll
                    for (int k = 0; k < C::kChunks; ++k)
                        tma_load_4d(qb + t * C::kQBytes + k * 128 * 128, &qmap, k * 64, sg.head * p.group,
                                    sg.rt * p.item_nodes + t * p.tile_nodes, sg.b, bar);
            }
            __syncwarp();
        }
        if (lane == 0) {
            sm.cuts = cuts;
            mbar_arrive(smem_u32(&sm.cuts_known));
        }
        if (!ok && seg > 0) wait_bar(bar, (seg - 1) & 1);
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------ products
        constexpr uint32_t kFmt = BF ? (1u << 7) | (1u << 10) : 0u;
        constexpr uint32_t kIdescS = (1u << 4) | kFmt | ((uint32_t)(kTok >> 3) << 17) | (8u << 24);
        constexpr uint32_t kIdescO = (1u << 4) | kFmt | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | (8u << 24);
        const int ksteps = (int)(c.head_dim + 15) / 16, k_slots = p.slots[0], v_slots = p.slots[1];
        const int streams = by_rows ? 2 : 1;           // that take each tile
        const int ahead = by_rows ? 1 : 2;             // tiles whose scores come before the first weights
        const uint32_t k_ring = desc_lo(smem_u32(smem), 16), v_ring = desc_lo(smem_u32(smem) + (uint32_t)k_slots * C::kSlotBytes, kTok * 128);
        const uint32_t q_lo = desc_lo(smem_u32(q_smem), 16);
        const uint32_t k_full = smem_u32(&sm.full[0][0]), v_full = smem_u32(&sm.full[1][0]);
        const uint32_t k_empty = smem_u32(&sm.empty[0][0]), v_empty = smem_u32(&sm.empty[1][0]);
        const uint32_t s_full = smem_u32(&sm.s_full[0]), p_full = smem_u32(&sm.p_full[0]);
        int k_at = 0, v_at = 0, seg = 0;
        uint32_t k_phase = 0, v_phase = 0, p_phase = 0;   // p_phase: a bit for each buffer
        auto scores = [&](int buf, uint32_t kl) {
            const uint32_t ql = q_lo + (by_rows && buf ? C::kQBytes / 16 : 0), d = tmem + (uint32_t)buf * kTok;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                if (k < ksteps)
                    mma_ss(d, ql + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2, kl + (k >> 2) * (kTok * 128 / 16) + (k & 3) * 2,
                           kDescHi, kIdescS, k != 0);
            mma_commit(s_full + 8 * buf);
        };
        auto values = [&](int buf, uint32_t vl, int valid, bool acc) {
            const uint32_t d = tmem + C::kOCol + (C::kOne ? 0u : (uint32_t)buf * DP), w = tmem + (uint32_t)buf * kTok;
#pragma unroll
            for (int k = 0; k < kTok / 16; ++k)
                if (k * 16 < valid) mma_ts(d, w + k * 8, vl + k * (2048 / 16), kDescHi, kIdescO, acc || k);
            if (C::kOne) mma_commit(smem_u32(&sm.pv_done));
        };
        while (ok && walk.next(sg)) {
            const int n = sg.t1 - sg.t0;
            ok = all_ok(wait_bar(smem_u32(&sm.q_full), seg & 1));
            if (!ok) break;
            tc_fence_after();
            // scores run `ahead` tiles ahead of the second products
            for (int i = -ahead; i < n; ++i) {
                const bool more = i + ahead < n, first = i < (by_rows || C::kOne ? 1 : 2);
                const int tile = sg.t0 + i, valid = tile == sg.tiles - 1 ? (int)a.nodes : min(kTok, sg.len - tile * kTok);
                const uint32_t kl = k_ring + (uint32_t)k_at * (C::kSlotBytes / 16), vl = v_ring + (uint32_t)v_at * (C::kSlotBytes / 16);
                // K and V are waited for before the weights, where K is not late
                if (i >= 0) ok = wait_bar(v_full + 8 * v_at, v_phase);
                bool k_there = more && mbar_try(k_full + 8 * k_at, k_phase);
                k_there = __all_sync(0xffffffffu, k_there);
                for (int t = 0; t < streams; ++t) {
                    const int buf = by_rows ? t : i & 1;      // score buffer = stream, but for kOne
                    if (i >= 0) {
                        ok = all_ok(ok && wait_bar(p_full + 8 * buf, p_phase >> buf & 1));
                        p_phase ^= 1u << buf;
                        if (!ok) break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
                        if (i >= 0) values(buf, vl, valid, !first);
                        if (k_there) scores(buf, kl);
                    }
                    __syncwarp();
                    if (more && !k_there) {
                        k_there = ok = all_ok(wait_bar(k_full + 8 * k_at, k_phase));
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) scores(buf, kl);
                        __syncwarp();
                    }
                }
                if (!ok) break;
                if (elect_one()) {
                    if (i >= 0) mma_commit(v_empty + 8 * v_at);
                    if (more) mma_commit(k_empty + 8 * k_at);
                    if (i + ahead == n - 1) mma_commit(smem_u32(&sm.q_free));
                }
                __syncwarp();
                if (i >= 0 && ++v_at == v_slots) v_at = 0, v_phase ^= 1;
                if (more && ++k_at == k_slots) k_at = 0, k_phase ^= 1;
            }
            if (!ok) break;
            if (elect_one()) mma_commit(smem_u32(&sm.done));
            __syncwarp();
            ++seg;
        }
        if (!ok) {   // a wait expired: let the products in flight end before TMEM is freed
            if (elect_one()) mma_commit(smem_u32(&sm.done));
            __syncwarp();
            wait_bar(smem_u32(&sm.done), seg & 1);
        }
    } else {
        // ------------------------------------------------------------ softmax
        const int g = warp >> 2, quad = warp & 3, row_in = quad * 32 + lane;   // stream, lane quadrant, row = TMEM lane
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const int dim = (int)c.head_dim;
        // items of few rows leave warps without a row: those clear values (below), while the others work
        const int cleaner = p.rows_item <= 96 ? (p.rows_item + 31) / 32 : 0;
        int seg = 0, tile0 = 0;          // tiles of the segments so far: places in the ring of V
        int j = 0;                       // tiles of this stream so far
        uint32_t s_phase = 0;            // a bit for each score buffer
        uint64_t mask = 0;
        int mask_of = -1;                // the nodes that it belongs to: the next head of the sequence has the same
        while (ok && walk.next(sg)) {
            const int n = sg.t1 - sg.t0;
            const int row = (by_rows ? g * 128 : 0) + row_in;     // of the item
            int head;
            const int node = node_of(p, sg, row, head);
            const bool mine = node >= 0;
            const bool work = __any_sync(0xffffffffu, mine);
            const int nodes_of = sg.b * p.row_tiles + sg.rt;
            if (nodes_of != mask_of) mask = mine ? ancestors(a.parents + (int64_t)sg.b * a.parents_stride, node) : 0;
            mask_of = nodes_of;
            float m = -INFINITY, l = 0.f;
            int my_tiles = 0;
            if (!(C::kOne && g == 1)) {
                const int step = by_rows || C::kOne ? 1 : 2;
                const uint32_t o_t = tmem + lane_off + C::kOCol + (uint32_t)g * DP;
                for (int i = by_rows ? 0 : g; i < n; i += step) {
                    const int buf = C::kOne ? i & 1 : g, tile = sg.t0 + i;
                    const bool tree = tile == sg.tiles - 1;
                    const int valid = tree ? (int)a.nodes : min(kTok, sg.len - tile * kTok);
                    ok = all_ok(wait_bar(smem_u32(&sm.s_full[buf]), s_phase >> buf & 1));
                    s_phase ^= 1u << buf;
                    if (!ok) break;
                    tc_fence_after();
                    if (work) {
                        const uint32_t st = tmem + lane_off + (uint32_t)buf * kTok;
                        // scores are read twice, 64 at a time: kept, 128 would not fit the registers (next to no
                        // first-level cache is left beside the tiles, a spill costs more than the second read)
                        // Columns behind the last group of 16 that has a token are not multiplied: a tile of up to 64
                        // tokens, as every tree is, is done after the first 64 (many short contexts 49 -> 46 us).
                        const int cols = kTok > 64 && valid <= 64 ? 64 : kTok;
                        float x[64], most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                        for (int h = 0; h < cols; h += 64) {
                            tmem_ld32(st + h, x);
                            tmem_ld32(st + h + 32, x + 32);
                            tmem_wait_ld();
                            if (tree || valid < h + 64) hide(x, tree, mask, valid - h);
#pragma unroll
                            for (int e = 0; e < 64; e += 8)
#pragma unroll
                                for (int k = 0; k < 4; ++k) most[k] = fmaxf(most[k], fmaxf(x[e + 2 * k], x[e + 2 * k + 1]));
                        }
                        const float top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * p.scale;
                        const bool grow = mine && top > m + 8.f;
                        if (my_tiles == 0) {
                            m = top;
                        } else if (__any_sync(0xffffffffu, grow)) {
                            // O holds the tiles so far: these scores come after their products, but for kOne, whose
                            // scores run ahead of them
                            if (C::kOne) {
                                ok = all_ok(wait_bar(smem_u32(&sm.pv_done), (uint32_t)(j - 1) & 1));
                                if (!ok) break;
                                tc_fence_after();
                            }
                            const float f = grow ? (m == -INFINITY ? 0.f : exp2_approx(m - top)) : 1.f;
                            if (grow) m = top, l *= f;
#pragma unroll 1
                            for (int e0 = 0; e0 < DP; e0 += 32) {
                                float o[32];
                                tmem_ld32(o_t + e0, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] *= f;
                                tmem_st16(o_t + e0, reinterpret_cast<const uint32_t*>(o));
                                tmem_st16(o_t + e0 + 16, reinterpret_cast<const uint32_t*>(o) + 16);
                            }
                        }
                        const float ref = m == -INFINITY ? 0.f : m;
                        const float2 scale2 = make_float2(p.scale, p.scale), ref2 = make_float2(-ref, -ref);
                        float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
                        for (int h = 0; h < cols; h += 64) {
                            if (kTok > 64) {
                                tmem_ld32(st + h, x);
                                tmem_ld32(st + h + 32, x + 32);
                                tmem_wait_ld();
                                if (tree || valid < h + 64) hide(x, tree, mask, valid - h);
                            }
                            // the weights of h.. take the columns of the scores h / 2.., which are done with
#pragma unroll
                            for (int e0 = 0; e0 < 64; e0 += 32) {
                                uint32_t w[16];
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    float2 t = fma2(make_float2(x[e0 + 2 * e], x[e0 + 2 * e + 1]), scale2, ref2);
                                    t = make_float2(exp2_approx(t.x), exp2_approx(t.y));
                                    sums[e & 1] = add2(sums[e & 1], t);
                                    w[e] = pack2<BF>(t.x, t.y);
                                }
                                tmem_st16(st + (h + e0) / 2, w);
                            }
                        }
                        sums[0] = add2(sums[0], sums[1]);
                        l += sums[0].x + sums[0].y;
                        tmem_wait_st();
                    }
                    ++my_tiles;
                    ++j;
                    // values that meet weights of zero must be finite: clear what lies behind the context in the last
                    // group of 16, and the infinities and NaN of the tree (added back below)
                    if ((tree || (valid & 15)) && !(by_rows && g == 1) && quad >= cleaner) {
                        const int pos = tile0 + i, slot_i = pos % p.slots[1];
                        ok = all_ok(wait_bar(smem_u32(&sm.full[1][slot_i]), (uint32_t)(pos / p.slots[1]) & 1));
                        if (!ok) break;
                        uint8_t* slot = smem + (size_t)(p.slots[0] + slot_i) * C::kSlotBytes;
                        const int tid = row_in - cleaner * 32, step = 128 - cleaner * 32;
                        if (!tree) {
                            const int n_rows = ((valid + 15) & ~15) - valid;
                            for (int e = tid; e < n_rows * C::kChunks * 8; e += step) {
                                const int r = e / (C::kChunks * 8), u = e % (C::kChunks * 8);
                                *reinterpret_cast<uint4*>(slot + (u >> 3) * kTok * 128 + (valid + r) * 128 + (u & 7) * 16) =
                                    make_uint4(0, 0, 0, 0);
                            }
                        } else {
                            constexpr uint32_t kExp = BF ? 0x7f807f80u : 0x7c007c00u;
                            for (int e = tid; e < valid * C::kChunks * 8; e += step) {
                                const int r = e / (C::kChunks * 8), u = e % (C::kChunks * 8);
                                uint4* w = reinterpret_cast<uint4*>(slot + (u >> 3) * kTok * 128 + r * 128 + (u & 7) * 16);
                                const uint4 q4 = *w;
                                uint32_t v4[4] = {q4.x, q4.y, q4.z, q4.w};
                                bool hit = false;
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    if ((v4[k] & kExp & 0xffffu) == (kExp & 0xffffu)) v4[k] &= 0xffff0000u, hit = true;
                                    if ((v4[k] & kExp & 0xffff0000u) == (kExp & 0xffff0000u)) v4[k] &= 0xffffu, hit = true;
                                }
                                if (hit) {
                                    *w = make_uint4(v4[0], v4[1], v4[2], v4[3]);
                                    sm.bad_v[seg & 1] = seg + 1;
                                }
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    // the first product of an item starts O anew: all warps have read the last one's
                    if (my_tiles == 1 && seg > 0) {
                        ok = all_ok(wait_bar(smem_u32(&sm.ended), (seg - 1) & 1));
                        if (!ok) break;
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[buf]));
                }
            }
            if (!ok) break;
            // the item's end (or the range's): O of both groups, added
            if (!by_rows) {
                ok = all_ok(seg == 0 || wait_bar(smem_u32(&sm.ended), (seg - 1) & 1));
                if (!ok) break;
                sm.ml[g][row_in] = make_float2(m, my_tiles ? l : 0.f);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.merge));
            ok = all_ok(wait_bar(smem_u32(&sm.merge), seg & 1) && wait_bar(smem_u32(&sm.done), seg & 1));
            if (!ok) break;
            tc_fence_after();
            if (work) {
                const bool whole = n == sg.tiles;
                float2 ml[2];
                uint32_t o_col[2];
                int col0 = 0, col1 = DP;
                if (by_rows) {
                    ml[0] = make_float2(m, l), ml[1] = make_float2(-INFINITY, 0.f);
                    o_col[0] = o_col[1] = C::kOCol + (uint32_t)g * DP;
                } else {
                    ml[0] = sm.ml[0][row_in], ml[1] = sm.ml[1][row_in];
                    o_col[0] = C::kOCol, o_col[1] = C::kOCol + (C::kOne ? 0u : DP);
                    col0 = g * (DP / 2), col1 = col0 + DP / 2;       // each group half of the columns
                }
                const float top = fmaxf(ml[0].x, ml[1].x);
                // (an unused node: whatever its scores and the values are, a row of zeros)
                float f0 = !mask || ml[0].y == 0.f ? 0.f : exp2_approx(ml[0].x - top);
                float f1 = !mask || ml[1].y == 0.f ? 0.f : exp2_approx(ml[1].x - top);
                const float sum = mask ? ml[0].y * f0 + ml[1].y * f1 : 0.f;
                const bool second = __any_sync(0xffffffffu, f1 != 0.f), none = __any_sync(0xffffffffu, mine && (f0 == 0.f || (second && f1 == 0.f)));
                if (whole) {
                    const float norm = sum == 0.f ? 0.f : __fdividef(1.f, sum);   // (two units in fp32's last place)
                    f0 *= norm, f1 *= norm;
                }
                const bool fix = sm.bad_v[seg & 1] == seg + 1;
                float4* part = p.part + (size_t)(2 * (int)blockIdx.x + (sg.t0 == 0 ? 1 : 0)) * (DP / 4) * p.rows_item + row;
                uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)sg.b * a.out_stride[0] + node * a.out_stride[1] +
                                head * a.out_stride[2];
                const uint16_t* tv = reinterpret_cast<const uint16_t*>(a.v) + (int64_t)sg.b * a.vn_stride[0] + sg.head * a.vn_stride[2];
#pragma unroll 1
                for (int e0 = col0; e0 < col1 && e0 < dim; e0 += 32) {
                    float o[32], o1[32];
                    tmem_ld32(tmem + lane_off + o_col[0] + e0, o);
                    if (second) tmem_ld32(tmem + lane_off + o_col[1] + e0, o1);
                    tmem_wait_ld();
                    // (O of a stream without tiles is not defined)
                    if (none) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            if (f0 == 0.f) o[e] = 0.f;
                            if (second && f1 == 0.f) o1[e] = 0.f;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 t = mul2(make_float2(o[e], o[e + 1]), make_float2(f0, f0));
                        o[e] = t.x, o[e + 1] = t.y;
                    }
                    if (second) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 t = fma2(make_float2(o1[e], o1[e + 1]), make_float2(f1, f1), make_float2(o[e], o[e + 1]));
                            o[e] = t.x, o[e + 1] = t.y;
                        }
                    }
                    if (fix) {
                        for (uint64_t left = mask; left; left &= left - 1) {
                            const uint16_t* v = tv + (__ffsll((long long)left) - 1) * a.vn_stride[1] + e0;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                if (e0 + e >= dim) continue;
                                const uint16_t h = v[e];
                                if ((h & (BF ? 0x7f80 : 0x7c00)) != (BF ? 0x7f80 : 0x7c00)) continue;
                                o[e] += BF ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
                            }
                        }
                    }
                    if (!mine) {
                        // a lane without a row only takes part in the loads
                    } else if (whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            if (e0 + e < dim)
                                *reinterpret_cast<uint4*>(out + e0 + e) =
                                    make_uint4(pack2<BF>(o[e], o[e + 1]), pack2<BF>(o[e + 2], o[e + 3]),
                                               pack2<BF>(o[e + 4], o[e + 5]), pack2<BF>(o[e + 6], o[e + 7]));
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            part[(size_t)((e0 + e) / 4) * p.rows_item] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                    __syncwarp();
                }
                if (mine && col0 == 0) {
                    if (!whole)
                        p.part_ml[(size_t)(2 * (int)blockIdx.x + (sg.t0 == 0 ? 1 : 0)) * p.rows_item + row] = make_float2(top, sum);
                    else if (a.lse)
                        a.lse[((int64_t)sg.b * a.nodes + node) * a.q_heads + head] =
                            sum == 0.f ? -INFINITY : (__log2f(sum) + top) * 0.6931471805599453f;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.ended));
            tile0 += n;
            ++seg;
        }
        // items in parts: say that this warp's share is there, wait for the others', add
        ok = ok && all_ok(wait_bar(smem_u32(&sm.cuts_known), 0));
        const int cuts = ok ? sm.cuts : 0;
        if (lane < cuts) add_release(p.count + 2 * sm.cut[lane].c0, 1);
        for (int k = 0; k < cuts && ok; ++k) ok = await_parts(p.count + 2 * sm.cut[k].c0, sm.cut[k].parts, lane);
#pragma unroll 1
        for (int k = 0; k < cuts && ok; ++k) {
            const Cut& cut = sm.cut[k];
            // one value a lane: few rows, often many parts
            if (p.rows_item * DP <= cut.parts * 1024) add_parts<DP, BF, 1, 16>(p, cut.sg, cut.c0, cut.parts);
            else add_parts<DP, BF, 4, 4>(p, cut.sg, cut.c0, cut.parts);
        }
    }
    if (!ok) report_device_error(p.err, 10);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
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
    SPARK_REQUIRE(a->q_heads / a->cache.kv_heads <= 128, SPARK_ERR_UNSUPPORTED,
                  "spark_tree_attention: %lld query heads per kv head, at most 128",
                  (long long)(a->q_heads / a->cache.kv_heads));
    SPARK_REQUIRE(a->cache.page_size % 8 == 0, SPARK_ERR_UNSUPPORTED,
                  "spark_tree_attention: page_size %lld is no multiple of 8", (long long)a->cache.page_size);
    SPARK_REQUIRE(a->scale >= 1e-30 && a->scale <= 1e30, SPARK_ERR_INVALID,
                  "spark_tree_attention: scale must be positive, 1e-30 to 1e30");
    return SPARK_OK;
}

int padded_dim(int64_t d) { return d <= 64 ? 64 : (d <= 128 ? 128 : 256); }

// Sizes that follow from the shapes alone; the workspace's layout.
struct Plan {
    int dp, grid, group, by_rows, tile_nodes, item_nodes, rows_item, row_tiles;
    size_t count, part, part_ml, bytes;
};
Plan plan(const SparkTreeAttention* a) {
    Plan q;
    int dev = 0;
    cudaGetDevice(&dev);
    q.count = 256;
    // (148 on a B200; two counters each lie in the part that the caller zeroes)
    q.grid = std::min(tc::sm_count_cached(dev), (int)((SPARK_TREE_ATTENTION_ZEROED - q.count) / (2 * sizeof(int))));
    q.dp = padded_dim(a->cache.head_dim);
    q.group = (int)(a->q_heads / a->cache.kv_heads);
    q.tile_nodes = std::min(128 / q.group, (int)a->nodes);
    q.by_rows = q.dp < 256 && q.tile_nodes < a->nodes;
    q.item_nodes = q.by_rows ? 2 * q.tile_nodes : q.tile_nodes;
    q.row_tiles = (int)((a->nodes + q.item_nodes - 1) / q.item_nodes);
    q.rows_item = q.by_rows ? 256 : q.tile_nodes * q.group;
    q.part_ml = SPARK_TREE_ATTENTION_ZEROED;
    q.part = (q.part_ml + (size_t)2 * q.grid * q.rows_item * sizeof(float2) + 255) / 256 * 256;
    q.bytes = q.part + (size_t)2 * q.grid * q.rows_item * q.dp * sizeof(float);
    return q;
}

template <int DP, bool BF>
int launch(const SparkTreeAttention* a, const Plan& q, uint8_t* ws, cudaStream_t s) {
    using C = Cfg<DP>;
    const SparkPagedCache& c = a->cache;
    Params p;
    p.a = *a;
    p.err = reinterpret_cast<int*>(ws);
    p.count = reinterpret_cast<int*>(ws + q.count);
    p.part = reinterpret_cast<float4*>(ws + q.part);
    p.part_ml = reinterpret_cast<float2*>(ws + q.part_ml);
    p.rows_item = q.rows_item, p.row_tiles = q.row_tiles, p.group = q.group;
    p.inv_group = 1.f / (float)q.group, p.inv_rows = 1.f / (float)q.rows_item;
    p.by_rows = q.by_rows, p.tile_nodes = q.tile_nodes, p.item_nodes = q.item_nodes;
    p.scale = (float)(a->scale * 1.4426950408889634);
    // a box of a TMA load lies within a page and within a tile
    p.tok = C::kTok;
    p.per_seq = (int)c.kv_heads * q.row_tiles;
    p.box_rows = 8;
    while (p.box_rows < C::kTok && c.page_size % (2 * p.box_rows) == 0) p.box_rows *= 2;
    const int q_tiles = p.by_rows ? 2 : 1;
    const int slots = std::min(2 * kMaxSlots, (232448 - kHeader - q_tiles * C::kQBytes) / C::kSlotBytes);
    p.slots[0] = slots / 2, p.slots[1] = slots - slots / 2;
    const size_t smem = (size_t)slots * C::kSlotBytes + (size_t)q_tiles * C::kQBytes + kHeader;
    static_assert(sizeof(Smem) <= kHeader, "shared header");

    int rc = tc::get_encoder();
    if (rc) return rc;
    CUtensorMap map[5];
    const CUtensorMapDataType dt = BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    auto encode = [&](CUtensorMap* m, const void* base, int64_t heads, int64_t rows, int64_t outer, const int64_t* st, int box_heads,
                      int box_rows) {
        const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)heads, (uint64_t)rows, (uint64_t)outer};
        const uint64_t strides[3] = {(uint64_t)st[2] * 2, (uint64_t)st[1] * 2, (uint64_t)st[0] * 2};
        const uint32_t box[4] = {64, (uint32_t)box_heads, (uint32_t)box_rows, 1};
        return tc::encode_4d(m, dt, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    rc = encode(&map[0], a->q, a->q_heads, a->nodes, a->batch, a->q_stride, q.group, q.tile_nodes);
    if (!rc) rc = encode(&map[1], c.k, c.kv_heads, c.page_size, c.pages, c.k_stride, 1, p.box_rows);
    if (!rc) rc = encode(&map[2], c.v, c.kv_heads, c.page_size, c.pages, c.v_stride, 1, p.box_rows);
    if (!rc) rc = encode(&map[3], a->k, c.kv_heads, a->nodes, a->batch, a->kn_stride, 1, 64);
    if (!rc) rc = encode(&map[4], a->v, c.kv_heads, a->nodes, a->batch, a->vn_stride, 1, 64);
    if (rc) return rc;
    cudaError_t e = cudaFuncSetAttribute(k_tree_attention<DP, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e != cudaSuccess) return set_error((int)e, "spark_tree_attention: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)q.grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeCooperative;
    at[0].val.cooperative = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, k_tree_attention<DP, BF>, map[0], map[1], map[2], map[3], map[4], p);
    if (e != cudaSuccess) return set_error((int)e, "spark_tree_attention: launch failed: %s", cudaGetErrorString(e));
    return check_launch("spark_tree_attention");
}

}  // namespace ta
}  // namespace spark

namespace spark {
namespace ta {
// A dimension of extent 1 has no stride: one that suits every check.
void tidy(SparkTreeAttention& a) {
    SparkPagedCache& c = a.cache;
    for (int64_t* st : {a.q_stride, a.kn_stride, a.vn_stride, a.out_stride, c.k_stride, c.v_stride}) {
        const bool cache = st == c.k_stride || st == c.v_stride, q = st == a.q_stride || st == a.out_stride;
        const int64_t n[3] = {cache ? c.pages : a.batch, cache ? c.page_size : a.nodes, q ? a.q_heads : c.kv_heads};
        for (int i = 0; i < 3; ++i)
            if (n[i] == 1) st[i] = c.head_dim;
    }
}
}  // namespace ta
}  // namespace spark

extern "C" {

size_t spark_tree_attention_workspace_size(const SparkTreeAttention* a) {
    return spark::ta::check(a) == SPARK_OK ? spark::ta::plan(a).bytes : 0;
}

int spark_tree_attention(const SparkTreeAttention* args, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace spark;
    using namespace spark::ta;
    const int rc = check(args);
    if (rc) return rc;
    SparkTreeAttention tidied = *args;
    tidy(tidied);
    const SparkTreeAttention* a = &tidied;
    if (a->batch == 0) return SPARK_OK;
    const SparkPagedCache& c = a->cache;
    SPARK_REQUIRE(a->q && a->k && a->v && a->out && a->parents && c.k && c.v && c.lens && (c.page_table || c.max_pages == 0),
                  SPARK_ERR_INVALID, "spark_tree_attention: null pointer");
    const Plan q = plan(a);
    const int tok = q.dp == 256 ? 64 : 128;
    SPARK_REQUIRE((double)a->batch * c.kv_heads * q.row_tiles * ((double)c.max_pages * c.page_size / tok + 2 + kStart) < 2147483647.0,
                  SPARK_ERR_UNSUPPORTED, "spark_tree_attention: 2^31 tiles of %d tokens or more", tok);
    SPARK_REQUIRE(workspace && workspace_bytes >= q.bytes, SPARK_ERR_WORKSPACE,
                  "spark_tree_attention: the workspace has %zu of %zu bytes", workspace_bytes, q.bytes);
    bool al = aligned(workspace, 256);
    for (const void* ptr : {a->q, a->k, a->v, (const void*)a->out, (const void*)c.k, (const void*)c.v}) al = al && aligned(ptr, 16);
    for (const int64_t* st : {(const int64_t*)a->q_stride, a->kn_stride, a->vn_stride, a->out_stride, c.k_stride, c.v_stride})
        for (int i = 0; i < 3; ++i) al = al && st[i] % 8 == 0 && st[i] > 0 && st[i] < (1ll << 38);
    SPARK_REQUIRE(al, SPARK_ERR_ALIGNMENT,
                  "spark_tree_attention: 16-byte aligned tensors with strides of a positive multiple of 8, and a 256-byte "
                  "aligned workspace");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
    const bool bf = c.dtype == SPARK_DTYPE_BF16;
    if (q.dp == 64) return bf ? launch<64, true>(a, q, ws, s) : launch<64, false>(a, q, ws, s);
    if (q.dp == 128) return bf ? launch<128, true>(a, q, ws, s) : launch<128, false>(a, q, ws, s);
    return bf ? launch<256, true>(a, q, ws, s) : launch<256, false>(a, q, ws, s);
}

}  // extern "C"
