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
//
// Work: an item is (sequence, kv head, tile of rows), its tiles are the context
// in steps of kTok tokens and last the tree.  All tiles of all items form one
// sequence cut into equal contiguous ranges, one per CTA (one CTA per SM), so
// that ragged batches and single long sequences fill the GPU alike without the
// host knowing the lengths.  Where a range cuts an item, the parts leave O, m
// and l in the workspace and a second kernel adds them in order: the result
// does not depend on timing.
//
// Roles (320 threads):
//   warps 0-3, 4-7  softmax: two groups, a thread owns one row (TMEM lane).  Up
//                   to 128 rows: both groups have the same rows and take tiles in
//                   turn, each with its own m, l and O, added at the end of the
//                   item.  Above: group g has rows 128 g.. of the item's 256 and
//                   takes every tile.  Heads above 128 wide leave room for one O
//                   only: group 0 works alone on tiles of 64 tokens.
//                   A group writes its weights over the scores they came from (the
//                   A operand of the second product is read from TMEM).
//   warp 8          loads K and V tiles by TMA, page by page, into a ring of slots.
//   warp 9          allocates TMEM and issues the MMAs.
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

constexpr int kThreads = 320;
constexpr int kTmaWarp = 8, kMmaWarp = 9;
constexpr int kMaxSlots = 12;
constexpr int kHeader = 3072;   // barriers and the exchange of the two groups
constexpr uint32_t kTmemCols = 512;

// DP: head_dim padded to 64, 128 or 256.
template <int DP>
struct Cfg {
    static constexpr int kTok = DP == 256 ? 64 : 128;      // tokens of a tile
    static constexpr bool kOne = DP == 256;                // one O, one softmax group
    static constexpr int kChunks = DP / 64;                // 128-byte columns of a tile
    static constexpr int kSlotBytes = kTok * DP * 2;       // 16 or 32 KB
    static constexpr int kQBytes = 128 * DP * 2;           // one 128-row Q tile
    static constexpr uint32_t kSCol = kTok;                // columns of one S buffer
    static constexpr uint32_t kOCol = 256;                 // first column of O
    static constexpr int kRowTile = kOne ? 128 : 256;      // most rows of an item
};

struct Params {
    SparkTreeAttention a;
    int* err;
    float* part;            // [2 * grid][rows][DP] O of cut items
    float2* part_ml;        // [2 * grid][rows] their m, l
    int rows_total, rows_item, row_tiles, group, box_rows, slots, by_rows;
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

__device__ __forceinline__ int64_t tiles_of(const Params& p, int64_t b, int tok) {
    return b < p.a.batch ? (context_len(p, b) + tok - 1) / tok + 1 : 0;
}
// Number of tiles of all items, by one warp.
__device__ __forceinline__ int64_t count_tiles(const Params& p, int tok, int lane) {
    int64_t total = 0;
    for (int64_t b = lane; b < p.a.batch; b += 32) total += tiles_of(p, b, tok);
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    return total * p.a.cache.kv_heads * p.row_tiles;
}
// The sequence that holds tile `pos` of all, and the tile's place among its tiles, by one warp.
__device__ __forceinline__ void locate(const Params& p, int tok, int lane, int64_t pos, int64_t& b, int64_t& off) {
    const int64_t per = p.a.cache.kv_heads * p.row_tiles;
    int64_t at = 0;
    b = p.a.batch, off = 0;
    for (int64_t base = 0; base < p.a.batch; base += 32) {
        const int64_t n = tiles_of(p, base + lane, tok) * per;
        int64_t sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && pos < at + sum);
        if (hit) {
            const int l = __ffs(hit) - 1;
            b = base + l;
            off = pos - (at + __shfl_sync(0xffffffffu, sum - n, l));
            return;
        }
        at += __shfl_sync(0xffffffffu, sum, 31);
    }
}

// A run of tiles of one item.
struct Segment {
    int64_t b;
    int head, rt, t0, t1, tiles, len;   // tiles t0..t1-1 of `tiles`; the last is the tree
};

// Walks the CTA's range of tiles.
template <int TOK>
struct Walker {
    const Params& p;
    int64_t b, off, left;
    __device__ Walker(const Params& q, int64_t b0, int64_t off0, int64_t n) : p(q), b(b0), off(off0), left(n) {}
    __device__ bool next(Segment& s) {
        if (left <= 0 || b >= p.a.batch) return false;
        s.len = context_len(p, b);
        s.tiles = (s.len + TOK - 1) / TOK + 1;
        const int item = (int)(off / s.tiles);
        s.b = b;
        s.head = item / p.row_tiles;
        s.rt = item - s.head * p.row_tiles;
        s.t0 = (int)(off - (int64_t)item * s.tiles);
        s.t1 = (int)min((int64_t)s.tiles, s.t0 + left);
        off += s.t1 - s.t0;
        left -= s.t1 - s.t0;
        if (off == (int64_t)s.tiles * p.a.cache.kv_heads * p.row_tiles) off = 0, ++b;
        return true;
    }
};

template <int DP>
struct Smem {
    uint64_t full[kMaxSlots], empty[kMaxSlots];
    uint64_t q_full, s_full[2], p_full[2], pv_done, merge, done;
    int64_t b0, off0, count;
    uint32_t tmem;
    int bad_v;               // the segment whose tree values hold an infinity or NaN
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
// D (+)= A B, both from shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
// D (+)= A B, A from TMEM
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
// N-major B operand, 128-byte swizzle: 64-column chunks `chunk_bytes` apart
// (leading offset), groups of eight K rows 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t sdesc_mn128(uint32_t addr, uint32_t chunk_bytes) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(chunk_bytes >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
           ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
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
__device__ __forceinline__ bool all_ok(bool ok) { return __all_sync(0xffffffffu, ok); }

// Position of V of the i-th tile (of n) in the ring's order: K0 K1 V0 K2 V1 ...
// where the groups take tiles in turn, K0 V0 K1 V1 ... where both take each.
__device__ __forceinline__ int v_ordinal(int i, int n, bool by_rows) {
    return by_rows ? 2 * i + 1 : min(2, n) + i + min(i, max(n - 2, 0));
}

template <int DP, bool BF>
__global__ void __launch_bounds__(kThreads, 1)
    k_tree_attention(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ CUtensorMap ktmap, const __grid_constant__ CUtensorMap vtmap,
                     const __grid_constant__ Params p) {
    using C = Cfg<DP>;
    constexpr int TOK = C::kTok;
    extern __shared__ __align__(1024) uint8_t smem[];
    Smem<DP>& sm = *reinterpret_cast<Smem<DP>*>(smem + (size_t)p.slots * C::kSlotBytes + (size_t)(p.by_rows ? 2 : 1) * C::kQBytes);
    uint8_t* q_smem = smem + (size_t)p.slots * C::kSlotBytes;
    const SparkTreeAttention& a = p.a;
    const SparkPagedCache& c = a.cache;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;");

    if (threadIdx.x == 0) {
        for (int i = 0; i < p.slots; ++i) mbar_init(smem_u32(&sm.full[i]), 1), mbar_init(smem_u32(&sm.empty[i]), 1);
        mbar_init(smem_u32(&sm.q_full), 8);
        for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&sm.s_full[i]), 1), mbar_init(smem_u32(&sm.p_full[i]), 4);
        mbar_init(smem_u32(&sm.pv_done), 1);
        mbar_init(smem_u32(&sm.merge), 8);
        mbar_init(smem_u32(&sm.done), 1);
        sm.bad_v = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if ((smem_u32(smem) & 1023) != 0) report_device_error(p.err, 10);
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 0) {
        // this CTA's range of the tiles
        if (blockIdx.x == 0)
            for (int64_t b = lane; b < a.batch; b += 32)
                if (c.lens[b] < 0 || c.lens[b] > c.max_pages * c.page_size) report_device_error(p.err, 9);
        const int64_t total = count_tiles(p, TOK, lane);
        const int64_t first = total * blockIdx.x / gridDim.x, end = total * (blockIdx.x + 1) / gridDim.x;
        int64_t b0, off0;
        locate(p, TOK, lane, first, b0, off0);
        if (lane == 0) sm.b0 = b0, sm.off0 = off0, sm.count = end - first;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    Walker<TOK> walk(p, sm.b0, sm.off0, (smem_u32(smem) & 1023) ? 0 : sm.count);
    const bool by_rows = p.by_rows;
    Segment sg;
    bool ok = true;

    if (warp == kTmaWarp) {
        // ------------------------------------------------------------ loads
        int ring = 0, filled = 0;
        uint32_t phase = 1;
        auto load = [&](const Segment& s, int tile, bool values) {
            const uint32_t slot = smem_u32(smem) + (uint32_t)ring * C::kSlotBytes, bar = smem_u32(&sm.full[ring]);
            ok = all_ok(mbar_wait(smem_u32(&sm.empty[ring]), phase));
            if (!ok) return;
            if (++ring == p.slots) ring = 0, phase ^= 1;
            ++filled;
            if (tile == s.tiles - 1) {
                if (lane == 0) mbar_expect_tx(bar, C::kChunks * 64 * 128);
                __syncwarp();
                if (lane < C::kChunks)
                    tma_load_4d(slot + lane * TOK * 128, values ? &vtmap : &ktmap, lane * 64, s.head, 0, (int)s.b, bar);
                return;
            }
            const int tok0 = tile * TOK, valid = min(TOK, s.len - tok0);
            const int n = (valid + p.box_rows - 1) / p.box_rows * C::kChunks;
            if (lane == 0) mbar_expect_tx(bar, (uint32_t)n * p.box_rows * 128);
            __syncwarp();
            for (int i = lane; i < n; i += 32) {
                const int box = i / C::kChunks, chunk = i - box * C::kChunks, tok = tok0 + box * p.box_rows;
                const int page_at = tok / (int)c.page_size, row = tok - page_at * (int)c.page_size;
                const int page = c.page_table[s.b * c.page_table_stride + page_at];
                if (page < 0 || page >= c.pages) report_device_error(p.err, 9);   // the load gives zeros
                tma_load_4d(slot + (uint32_t)(chunk * TOK + box * p.box_rows) * 128, values ? &vmap : &kmap, chunk * 64,
                            s.head, row, page, bar);
            }
        };
        while (ok && walk.next(sg)) {
            const int n = sg.t1 - sg.t0;
            const int ahead = by_rows ? 1 : 2;
            for (int i = 0; i < min(ahead, n) && ok; ++i) load(sg, sg.t0 + i, false);
            for (int i = 0; i < n && ok; ++i) {
                load(sg, sg.t0 + i, true);
                if (ok && i + ahead < n) load(sg, sg.t0 + i + ahead, false);
            }
        }
        if (!ok)   // a wait expired: let the loads in flight land before the CTA ends
            for (int i = 0; i < min(filled, p.slots); ++i)
                mbar_wait(smem_u32(&sm.full[i]), (uint32_t)((filled - 1 - i) / p.slots) & 1);
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------ products
        constexpr uint32_t kFmt = BF ? (1u << 7) | (1u << 10) : 0u;
        constexpr uint32_t kIdescS = (1u << 4) | kFmt | ((uint32_t)(TOK >> 3) << 17) | (8u << 24);
        constexpr uint32_t kIdescO = (1u << 4) | kFmt | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | (8u << 24);
        if (lane == 0) {
            const uint32_t base = smem_u32(smem), qb = smem_u32(q_smem);
            const int ksteps = (int)(c.head_dim + 15) / 16;
            int ring = 0, seg = 0;
            uint32_t phase = 0, p_phase[2] = {0, 0};
            uint32_t k_slot[2], v_slot, v_bar;
            // next slot of the ring, once its tile has landed
            auto take = [&](uint32_t& slot, uint32_t& bar) {
                slot = base + (uint32_t)ring * C::kSlotBytes;
                bar = smem_u32(&sm.empty[ring]);
                ok = mbar_wait(smem_u32(&sm.full[ring]), phase);
                tc_fence_after();
                if (++ring == p.slots) ring = 0, phase ^= 1;
                return ok;
            };
            auto scores = [&](int s, int qt, uint32_t slot) {
                for (int k = 0; k < ksteps; ++k) {
                    const uint32_t o = (uint32_t)(k & 3) * 32;
                    mma_ss(tmem + (uint32_t)s * C::kSCol, sdesc_sw128(qb + (uint32_t)qt * C::kQBytes + (k >> 2) * 128 * 128 + o),
                           sdesc_sw128(slot + (k >> 2) * TOK * 128 + o), kIdescS, k != 0);
                }
                mma_commit(smem_u32(&sm.s_full[s]));
            };
            auto values = [&](int s, uint32_t slot, int valid, bool acc) {
                const int n = (valid + 15) / 16;
                const uint32_t o = tmem + C::kOCol + (C::kOne ? 0u : (uint32_t)s * DP);
                for (int k = 0; k < n; ++k)
                    mma_ts(o, tmem + (uint32_t)s * C::kSCol + k * 8, sdesc_mn128(slot + k * 2048, TOK * 128), kIdescO, acc || k);
            };
            while (ok && walk.next(sg)) {
                const int n = sg.t1 - sg.t0;
                auto valid = [&](int i) {
                    const int t = sg.t0 + i;
                    return t == sg.tiles - 1 ? (int)a.nodes : min(TOK, sg.len - t * TOK);
                };
                ok = mbar_wait(smem_u32(&sm.q_full), seg & 1);
                if (!ok) break;
                tc_fence_after();
                uint32_t bar;
                if (by_rows) {
                    if (!take(k_slot[0], bar)) break;
                    scores(0, 0, k_slot[0]);
                    scores(1, 1, k_slot[0]);
                    mma_commit(bar);
                    for (int i = 0; i < n && ok; ++i) {
                        uint32_t k_bar = 0;
                        if (!take(v_slot, v_bar)) break;
                        for (int s = 0; s < 2 && ok; ++s) {
                            ok = mbar_wait(smem_u32(&sm.p_full[s]), p_phase[s]);
                            p_phase[s] ^= 1;
                            if (!ok) break;
                            tc_fence_after();
                            values(s, v_slot, valid(i), i > 0);
                            if (s == 1) mma_commit(v_bar);
                            if (i + 1 < n) {
                                if (s == 0 && !take(k_slot[0], k_bar)) break;
                                scores(s, s, k_slot[0]);
                                if (s == 1) mma_commit(k_bar);
                            }
                        }
                    }
                } else {
                    for (int i = 0; i < min(2, n) && ok; ++i) {
                        if (!take(k_slot[i], bar)) break;
                        scores(i, 0, k_slot[i]);
                        mma_commit(bar);
                    }
                    for (int i = 0; i < n && ok; ++i) {
                        const int s = i & 1;
                        if (!take(v_slot, v_bar)) break;
                        ok = mbar_wait(smem_u32(&sm.p_full[s]), p_phase[s]);
                        p_phase[s] ^= 1;
                        if (!ok) break;
                        tc_fence_after();
                        values(s, v_slot, valid(i), C::kOne ? i > 0 : i > 1);
                        if (C::kOne) mma_commit(smem_u32(&sm.pv_done));
                        mma_commit(v_bar);
                        if (i + 2 < n) {
                            if (!take(k_slot[s], bar)) break;
                            scores(s, 0, k_slot[s]);
                            mma_commit(bar);
                        }
                    }
                }
                if (!ok) break;
                mma_commit(smem_u32(&sm.done));
                ++seg;
            }
            if (!ok) {   // a wait expired: let the products in flight end before TMEM is freed
                mma_commit(smem_u32(&sm.done));
                mbar_wait(smem_u32(&sm.done), seg & 1);
            }
        }
    } else {
        // ------------------------------------------------------------ softmax
        const int g = warp >> 2, quad = warp & 3, row_in = quad * 32 + lane;   // group, lane quadrant, row = TMEM lane
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const int dim = (int)c.head_dim;
        int seg = 0, ring0 = 0;          // ring position of the segment's first tile, counted on
        uint32_t s_phase[2] = {0, 0};
        int pv = 0;                      // second products so far (kOne)
        while (ok && walk.next(sg)) {
            const int n = sg.t1 - sg.t0;
            const int row_base = sg.rt * C::kRowTile;
            const int rows = min(p.rows_total - row_base, C::kRowTile);   // of this item
            // Q: rows in the order of nodes, then the heads of the group
            {
                const int units = DP / 8, first = by_rows ? g * 128 : 0;
                const int n_rows = by_rows ? min(max(rows - first, 0), 128) : rows;
                const int tid = by_rows ? (int)threadIdx.x & 127 : (int)threadIdx.x, nt = by_rows ? 128 : 256;
                uint8_t* qs = q_smem + (by_rows ? g : 0) * C::kQBytes;
                for (int i = tid; i < n_rows * units; i += nt) {
                    const int r = i / units, u = i - r * units, rr = row_base + first + r;
                    const int t = rr / p.group, h = sg.head * p.group + rr - t * p.group;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (u * 8 < dim)
                        v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + sg.b * a.q_stride[0] +
                                                            t * a.q_stride[1] + h * a.q_stride[2] + u * 8);
                    *reinterpret_cast<uint4*>(qs + (u >> 3) * 128 * 128 + r * 128 + (((u & 7) ^ (r & 7)) << 4)) = v;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sm.q_full));
            }
            // (a group without tiles may not run ahead of the other's last item either)
            ok = all_ok(mbar_wait(smem_u32(&sm.q_full), seg & 1));
            if (!ok) break;
            const int row = (by_rows ? g * 128 : 0) + row_in;     // of the item
            const bool mine = row < rows;
            const bool work = (by_rows ? g * 128 : 0) + quad * 32 < rows;   // any row of this warp
            const int node = mine ? (row_base + row) / p.group : 0;
            const uint64_t mask = mine ? ancestors(a.parents + sg.b * a.parents_stride, node) : 0;
            float m = -INFINITY, l = 0.f;
            int my_tiles = 0;
            if (!(C::kOne && g == 1)) {
                const int step = by_rows || C::kOne ? 1 : 2;
                for (int i = by_rows || C::kOne ? 0 : g; i < n; i += step) {
                    const int s = by_rows ? g : (i & 1);          // S buffer
                    const int tile = sg.t0 + i;
                    const bool tree = tile == sg.tiles - 1;
                    const int valid = tree ? (int)a.nodes : min(TOK, sg.len - tile * TOK);
                    ok = all_ok(mbar_wait(smem_u32(&sm.s_full[s]), s_phase[s]));
                    s_phase[s] ^= 1;
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t st = tmem + lane_off + (uint32_t)s * C::kSCol;
                    float x[TOK];
                    if (work) {
#pragma unroll
                        for (int j = 0; j < TOK; j += 32) tmem_ld32(st + j, x + j);
                        tmem_wait_ld();
                        if (tree) {
#pragma unroll
                            for (int j = 0; j < TOK; ++j)
                                if (j >= 64 || !((mask >> (j & 63)) & 1)) x[j] = -INFINITY;
                        } else if (valid < TOK) {
#pragma unroll
                            for (int j = 0; j < TOK; ++j)
                                if (j >= valid) x[j] = -INFINITY;
                        }
                        float top = x[0];
#pragma unroll
                        for (int j = 1; j < TOK; ++j) top = fmaxf(top, x[j]);
                        top *= p.scale;
                        if (C::kOne && pv > 0) {
                            ok = all_ok(mbar_wait(smem_u32(&sm.pv_done), (uint32_t)(pv - 1) & 1));
                            if (!ok) break;
                            tc_fence_after();
                        }
                        const bool grow = mine && top > m + 8.f;
                        if (my_tiles == 0) {
                            m = top;
                        } else if (__any_sync(0xffffffffu, grow)) {
                            const float f = grow ? (m == -INFINITY ? 0.f : exp2_approx(m - top)) : 1.f;
                            if (grow) m = top, l *= f;
                            const uint32_t ot = tmem + lane_off + C::kOCol + (C::kOne ? 0u : (uint32_t)(by_rows ? g : s) * DP);
#pragma unroll
                            for (int j = 0; j < DP; j += 32) {
                                float o[32];
                                tmem_ld32(ot + j, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] *= f;
                                tmem_st16(ot + j, reinterpret_cast<const uint32_t*>(o));
                                tmem_st16(ot + j + 16, reinterpret_cast<const uint32_t*>(o) + 16);
                            }
                        }
                        const float ref = m == -INFINITY ? 0.f : m;
                        float sum = 0.f;
#pragma unroll
                        for (int j = 0; j < TOK; j += 32) {
                            uint32_t w[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float u = exp2_approx(fmaf(x[j + 2 * e], p.scale, -ref));
                                const float v = exp2_approx(fmaf(x[j + 2 * e + 1], p.scale, -ref));
                                sum += u + v;
                                w[e] = pack2<BF>(u, v);
                            }
                            tmem_st16(st + j / 2, w);
                        }
                        l += sum;
                        tmem_wait_st();
                    } else if (C::kOne && pv > 0) {
                        ok = all_ok(mbar_wait(smem_u32(&sm.pv_done), (uint32_t)(pv - 1) & 1));
                        if (!ok) break;
                    }
                    ++my_tiles;
                    ++pv;
                    // values that meet weights of zero must be finite: clear what lies behind the context in the last
                    // group of 16, and the infinities and NaN of the tree (added back below)
                    if ((tree || (valid & 15)) && !(by_rows && g == 1)) {
                        const int at = ring0 + v_ordinal(i, n, by_rows), slot_i = at % p.slots;
                        ok = all_ok(mbar_wait(smem_u32(&sm.full[slot_i]), (uint32_t)(at / p.slots) & 1));
                        if (!ok) break;
                        uint8_t* slot = smem + (size_t)slot_i * C::kSlotBytes;
                        const int tid = (int)threadIdx.x & 127;
                        if (!tree) {
                            const int n_rows = ((valid + 15) & ~15) - valid;
                            for (int e = tid; e < n_rows * C::kChunks * 8; e += 128) {
                                const int r = e / (C::kChunks * 8), u = e % (C::kChunks * 8);
                                *reinterpret_cast<uint4*>(slot + (u >> 3) * TOK * 128 + (valid + r) * 128 + (u & 7) * 16) =
                                    make_uint4(0, 0, 0, 0);
                            }
                        } else {
                            constexpr uint32_t kExp = BF ? 0x7f807f80u : 0x7c007c00u;
                            for (int e = tid; e < valid * C::kChunks * 8; e += 128) {
                                const int r = e / (C::kChunks * 8), u = e % (C::kChunks * 8);
                                uint32_t* w = reinterpret_cast<uint32_t*>(slot + (u >> 3) * TOK * 128 + r * 128 + (u & 7) * 16);
                                uint4 q4 = *reinterpret_cast<uint4*>(w);
                                uint32_t v4[4] = {q4.x, q4.y, q4.z, q4.w};
                                bool hit = false;
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    if ((v4[k] & kExp & 0xffffu) == (kExp & 0xffffu)) v4[k] &= 0xffff0000u, hit = true;
                                    if ((v4[k] & kExp & 0xffff0000u) == (kExp & 0xffff0000u)) v4[k] &= 0xffffu, hit = true;
                                }
                                if (hit) {
                                    *reinterpret_cast<uint4*>(w) = make_uint4(v4[0], v4[1], v4[2], v4[3]);
                                    sm.bad_v = seg + 1;
                                }
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[s]));
                }
            }
            if (!ok) break;
            // the item's end (or the range's): O of both groups, added
            if (!by_rows) sm.ml[g][row_in] = make_float2(m, my_tiles ? l : 0.f);
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.merge));
            ok = all_ok(mbar_wait(smem_u32(&sm.merge), seg & 1) && mbar_wait(smem_u32(&sm.done), seg & 1));
            if (!ok) break;
            tc_fence_after();
            if (work) {
                float2 ml[2];
                uint32_t o_col[2];
                int c0 = 0, c1 = DP;
                if (by_rows) {
                    ml[0] = make_float2(m, l), ml[1] = make_float2(-INFINITY, 0.f);
                    o_col[0] = o_col[1] = C::kOCol + (C::kOne ? 0u : (uint32_t)g * DP);
                } else {
                    ml[0] = sm.ml[0][row_in], ml[1] = sm.ml[1][row_in];
                    o_col[0] = C::kOCol, o_col[1] = C::kOCol + (C::kOne ? 0u : DP);
                    c0 = g * (DP / 2), c1 = c0 + DP / 2;           // each group half of the columns
                }
                const float top = fmaxf(ml[0].x, ml[1].x);
                const float f0 = ml[0].y == 0.f ? 0.f : exp2_approx(ml[0].x - top);
                const float f1 = ml[1].y == 0.f ? 0.f : exp2_approx(ml[1].x - top);
                const float sum = mask ? ml[0].y * f0 + ml[1].y * f1 : 0.f;
                const bool whole = n == sg.tiles;
                const float norm = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
                const bool second = __any_sync(0xffffffffu, f1 != 0.f);
                const bool fix = sm.bad_v == seg + 1;
                const int slot = 2 * (int)blockIdx.x + (sg.t0 == 0 ? 1 : 0);
                float* part = p.part + ((size_t)slot * p.rows_item + row) * DP;
                const int head = sg.head * p.group + (row_base + row) - node * p.group;
                uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + sg.b * a.out_stride[0] + node * a.out_stride[1] +
                                head * a.out_stride[2];
                const uint16_t* tv = reinterpret_cast<const uint16_t*>(a.v) + sg.b * a.vn_stride[0] + sg.head * a.vn_stride[2];
                for (int j = c0; j < c1 && j < dim; j += 16) {
                    float o[16];
                    tmem_ld16(tmem + lane_off + o_col[0] + j, o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = f0 == 0.f ? 0.f : o[e] * f0;
                    if (second) {
                        float o1[16];
                        tmem_ld16(tmem + lane_off + o_col[1] + j, o1);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] += f1 == 0.f ? 0.f : o1[e] * f1;
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = sum == 0.f ? 0.f : o[e] * norm;
                    if (fix) {
                        for (uint64_t left = mask; left; left &= left - 1) {
                            const int t = __ffsll((long long)left) - 1;
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                if (j + e >= dim) continue;
                                const float v = load_as_float(tv, (int)c.dtype, t * a.vn_stride[1] + j + e);
                                if (!isfinite(v)) o[e] += v;
                            }
                        }
                    }
                    if (!mine) {
                        // a lane without a row only takes part in the loads
                    } else if (whole) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) w[e] = pack2<BF>(o[2 * e], o[2 * e + 1]);
                        *reinterpret_cast<uint4*>(out + j) = make_uint4(w[0], w[1], w[2], w[3]);
                        if (j + 8 < dim) *reinterpret_cast<uint4*>(out + j + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            *reinterpret_cast<float4*>(part + j + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                    __syncwarp();
                }
                if (mine && c0 == 0) {
                    if (!whole)
                        p.part_ml[(size_t)slot * p.rows_item + row] = make_float2(top, sum);
                    else if (a.lse)
                        a.lse[(sg.b * a.nodes + node) * a.q_heads + head] =
                            sum == 0.f ? -INFINITY : (log2f(sum) + top) * 0.6931471805599453f;
                }
            }
            ring0 += 2 * n;
            ++seg;
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

// Adds the parts of the items that several CTAs worked on, in the CTAs' order.
// Block y stands for the cut between CTAs y and y + 1 of the first kernel (of
// `grid` CTAs) and does the item it cuts, unless an earlier cut has that item.
// A warp adds a row.
constexpr int kCombineRows = 32;
template <int DP>
__global__ void __launch_bounds__(256) k_tree_combine(const __grid_constant__ Params p, int grid) {
    constexpr int TOK = Cfg<DP>::kTok, kRowTile = Cfg<DP>::kRowTile;
    const SparkTreeAttention& a = p.a;
    const SparkPagedCache& c = a.cache;
    const int lane = threadIdx.x & 31;
    const int64_t total = count_tiles(p, TOK, lane);
    const int64_t cut = total * (blockIdx.y + 1) / grid;
    int64_t b, off;
    locate(p, TOK, lane, cut, b, off);
    const int64_t tiles = tiles_of(p, b, TOK);
    const int item = tiles ? (int)(off / tiles) : 0;
    const int64_t lo = cut - (off - (int64_t)item * tiles), hi = lo + tiles;   // the item's tiles among all
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (b >= a.batch || cut == lo || total * blockIdx.y / grid > lo) return;
    const int head = item / p.row_tiles, rt = item - head * p.row_tiles;
    const int c0 = (int)blockIdx.y, c1 = (int)((hi * grid - 1) / total);   // first and last CTA of the item
    for (int r = threadIdx.x >> 5; r < kCombineRows; r += 8) {
        const int row = blockIdx.x * kCombineRows + r, rr = rt * kRowTile + row;
        if (row >= p.rows_item || rr >= p.rows_total) break;
        float top = -INFINITY, sum = 0.f, o[DP / 32];
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) o[i] = 0.f;
        for (int cta = c0; cta <= c1; ++cta) {
            const int64_t first = total * cta / grid;
            if (first == total * (cta + 1) / grid) continue;
            const size_t at = (size_t)(2 * cta + (lo >= first ? 1 : 0)) * p.rows_item + row;
            const float2 ml = p.part_ml[at];
            if (ml.y == 0.f) continue;
            const float m2 = fmaxf(top, ml.x), f = top == -INFINITY ? 0.f : exp2_approx(top - m2);
            const float g = exp2_approx(ml.x - m2);
            top = m2;
            sum = sum * f + ml.y * g;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const int d = lane + 32 * i;
                if (d < c.head_dim) o[i] = (f == 0.f ? 0.f : o[i] * f) + p.part[at * DP + d] * g;
            }
        }
        const int node = rr / p.group, h = head * p.group + rr - node * p.group;
        const int64_t out = b * a.out_stride[0] + node * a.out_stride[1] + h * a.out_stride[2];
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
            const int d = lane + 32 * i;
            if (d < c.head_dim) store_from_float(a.out, (int)c.dtype, out + d, sum == 0.f ? 0.f : o[i] / sum);
        }
        if (a.lse && lane == 0)
            a.lse[(b * a.nodes + node) * a.q_heads + h] = sum == 0.f ? -INFINITY : (log2f(sum) + top) * 0.6931471805599453f;
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
    SPARK_REQUIRE(a->cache.page_size % 8 == 0, SPARK_ERR_UNSUPPORTED,
                  "spark_tree_attention: page_size %lld is no multiple of 8", (long long)a->cache.page_size);
    SPARK_REQUIRE(a->scale > 0 && a->scale < 1e30, SPARK_ERR_INVALID, "spark_tree_attention: scale must be positive");
    return SPARK_OK;
}

int padded_dim(int64_t d) { return d <= 64 ? 64 : (d <= 128 ? 128 : 256); }

// Sizes that follow from the shapes alone; the workspace's layout.
struct Plan {
    int dp, grid, rows_total, rows_item, row_tiles;
    size_t part, part_ml, bytes;
};
Plan plan(const SparkTreeAttention* a) {
    Plan q;
    int dev = 0;
    cudaGetDevice(&dev);
    q.grid = tc::sm_count_cached(dev);
    q.dp = padded_dim(a->cache.head_dim);
    const int tile = q.dp == 256 ? 128 : 256;
    q.rows_total = (int)(a->nodes * (a->q_heads / a->cache.kv_heads));
    q.row_tiles = (q.rows_total + tile - 1) / tile;
    q.rows_item = std::min(q.rows_total, tile);
    q.part_ml = 256;
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
    p.part = reinterpret_cast<float*>(ws + q.part);
    p.part_ml = reinterpret_cast<float2*>(ws + q.part_ml);
    p.rows_total = q.rows_total, p.rows_item = q.rows_item, p.row_tiles = q.row_tiles;
    p.group = (int)(a->q_heads / c.kv_heads);
    p.by_rows = !C::kOne && q.rows_total > 128;
    p.scale = (float)(a->scale * 1.4426950408889634);
    // a box of a TMA load lies within a page and within a tile
    p.box_rows = 8;
    while (p.box_rows < C::kTok && c.page_size % (2 * p.box_rows) == 0) p.box_rows *= 2;
    const int q_tiles = p.by_rows ? 2 : 1;
    p.slots = std::min(kMaxSlots, (232448 - kHeader - q_tiles * C::kQBytes) / C::kSlotBytes);
    const size_t smem = (size_t)p.slots * C::kSlotBytes + (size_t)q_tiles * C::kQBytes + kHeader;
    static_assert(sizeof(Smem<DP>) <= kHeader, "shared header");

    int rc = tc::get_encoder();
    if (rc) return rc;
    CUtensorMap map[4];
    const CUtensorMapDataType dt = BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    for (int i = 0; i < 4; ++i) {
        const bool tree = i >= 2, v = i & 1;
        const int64_t* st = tree ? (v ? a->vn_stride : a->kn_stride) : (v ? c.v_stride : c.k_stride);   // outer, row, head
        const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)c.kv_heads, (uint64_t)(tree ? a->nodes : c.page_size),
                                  (uint64_t)(tree ? a->batch : c.pages)};
        const uint64_t strides[3] = {(uint64_t)st[2] * 2, (uint64_t)st[1] * 2, (uint64_t)st[0] * 2};
        const uint32_t box[4] = {64, 1, (uint32_t)(tree ? 64 : p.box_rows), 1};
        rc = tc::encode_4d(&map[i], dt, tree ? (v ? a->v : a->k) : (v ? c.v : c.k), dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc) return rc;
    }
    cudaError_t e = cudaFuncSetAttribute(k_tree_attention<DP, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e != cudaSuccess) return set_error((int)e, "spark_tree_attention: %s", cudaGetErrorString(e));
    k_tree_attention<DP, BF><<<q.grid, kThreads, smem, s>>>(map[0], map[1], map[2], map[3], p);
    rc = check_launch("spark_tree_attention");
    if (rc) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((q.rows_item + kCombineRows - 1) / kCombineRows), (unsigned)(q.grid - 1));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, k_tree_combine<DP>, p, q.grid);
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
    SPARK_REQUIRE(workspace && workspace_bytes >= q.bytes, SPARK_ERR_WORKSPACE,
                  "spark_tree_attention: the workspace has %zu of %zu bytes", workspace_bytes, q.bytes);
    bool al = aligned(workspace, 256);
    for (const void* ptr : {a->q, a->k, a->v, (const void*)a->out, (const void*)c.k, (const void*)c.v}) al = al && aligned(ptr, 16);
    for (const int64_t* st : {(const int64_t*)a->q_stride, a->kn_stride, a->vn_stride, a->out_stride, c.k_stride, c.v_stride})
        for (int i = 0; i < 3; ++i) al = al && st[i] % 8 == 0 && st[i] >= 0 && st[i] < (1ll << 38);
    SPARK_REQUIRE(al, SPARK_ERR_ALIGNMENT,
                  "spark_tree_attention: 16-byte aligned tensors with strides of a multiple of 8, and a 256-byte aligned "
                  "workspace");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
    const bool bf = c.dtype == SPARK_DTYPE_BF16;
    if (q.dp == 64) return bf ? launch<64, true>(a, q, ws, s) : launch<64, false>(a, q, ws, s);
    if (q.dp == 128) return bf ? launch<128, true>(a, q, ws, s) : launch<128, false>(a, q, ws, s);
    return bf ? launch<256, true>(a, q, ws, s) : launch<256, false>(a, q, ws, s);
}

}  // extern "C"
