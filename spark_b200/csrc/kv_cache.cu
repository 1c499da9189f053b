// kv_cache.cu -- append of new tokens to a paged K/V cache.
//
// Position n of sequence b is row n % page_size of page page_table[b, n /
// page_size].  The kernel moves rows of kv_heads x head_dim values; its bound
// is HBM (each value is read and written once).  A group of threads, as many as
// a row has 16-byte pieces (a power of two of 8 to 256), moves K and V of two
// tokens, four loads of a thread on the way together: 8192 tokens of 32 heads of
// 128 in bf16 44 us (6.1 TB/s; four tokens a group, whose pointers take half as
// many registers again, 47 us).  A block has as many groups as fit: with one of
// 256 threads, most of them idle in short rows, 8192 tokens of one head of 80 in
// fp32 took 14.6 us, now 4.4, and of 8 heads of 64 8.6, now 4.6.
#include <algorithm>

#include "common.cuh"

namespace spark {
namespace kv {

struct Params {
    SparkPagedCache c;
    const void *k, *v;
    int64_t ks[3], vs[3];
    int64_t batch, tokens, width;
    const int *index, *counts;
    int *new_lens, *err;
    int group;   // threads that move a row, a power of two
};

// T: what is moved at a time.
constexpr int kTokens = 2;   // of a group
template <typename T, int E>   // E values in a T
__global__ void __launch_bounds__(256) k_kv_append(const __grid_constant__ Params p) {
    grid_wait();
    const int64_t b = blockIdx.y;
    const int64_t len = p.c.lens[b];
    const int64_t room = p.c.max_pages * p.c.page_size - len;
    int64_t n = p.counts ? p.counts[b] : p.width;
    bool bad = n < 0 || n > p.width || len < 0 || n > room;
    n = len < 0 || n < 0 ? 0 : n;
    n = n > p.width ? p.width : n;
    n = n > room ? (room < 0 ? 0 : room) : n;
    const int slot = (int)threadIdx.x / p.group, lane = (int)threadIdx.x % p.group;
    if (blockIdx.x == 0 && threadIdx.x == 0) p.new_lens[b] = (int)(len + n);
    const int per_head = (int)p.c.head_dim / E, row = (int)p.c.kv_heads * per_head;
    const int64_t j0 = ((int64_t)blockIdx.x * (256 / p.group) + slot) * kTokens;
    const T *kx[kTokens], *vx[kTokens];
    T *ky[kTokens], *vy[kTokens];
    bool move[kTokens];
#pragma unroll
    for (int q = 0; q < kTokens; ++q) {
        const int64_t j = j0 + q, at = len + j;
        move[q] = j < n;
        if (!move[q]) continue;
        const int64_t src = p.index ? p.index[b * p.width + j] : j;
        const int64_t page = p.c.page_table[b * p.c.page_table_stride + at / p.c.page_size], r = at % p.c.page_size;
        move[q] = src >= 0 && src < p.tokens && page >= 0 && page < p.c.pages;
        bad |= !move[q];
        kx[q] = reinterpret_cast<const T*>(p.k) + (b * p.ks[0] + src * p.ks[1]) / E;
        vx[q] = reinterpret_cast<const T*>(p.v) + (b * p.vs[0] + src * p.vs[1]) / E;
        ky[q] = reinterpret_cast<T*>(p.c.k) + (page * p.c.k_stride[0] + r * p.c.k_stride[1]) / E;
        vy[q] = reinterpret_cast<T*>(p.c.v) + (page * p.c.v_stride[0] + r * p.c.v_stride[1]) / E;
    }
    for (int i = lane; i < row; i += p.group) {
        const int h = i / per_head, d = i - h * per_head;
        const int64_t xk = h * (p.ks[2] / E) + d, xv = h * (p.vs[2] / E) + d;
        const int64_t yk = h * (p.c.k_stride[2] / E) + d, yv = h * (p.c.v_stride[2] / E) + d;
        T a[kTokens], c[kTokens];
#pragma unroll
        for (int q = 0; q < kTokens; ++q)
            if (move[q]) a[q] = kx[q][xk], c[q] = vx[q][xv];
#pragma unroll
        for (int q = 0; q < kTokens; ++q)
            if (move[q]) ky[q][yk] = a[q], vy[q][yv] = c[q];
    }
    if (bad && lane == 0) report_device_error(p.err, 9);
}

}  // namespace kv

// The checks that every call on a paged cache makes.
int check_cache(const SparkPagedCache* c, const char* who) {
    SPARK_REQUIRE(c, SPARK_ERR_INVALID, "%s: null pointer", who);
    SPARK_REQUIRE(c->pages >= 1 && c->pages < (1ll << 31) && c->page_size >= 1 && c->page_size < (1 << 24) &&
                      c->kv_heads >= 1 && c->kv_heads < (1 << 16) && c->head_dim >= 1 && c->head_dim < (1 << 16) &&
                      c->kv_heads * c->head_dim < (1ll << 31) && c->max_pages >= 0 && c->page_table_stride >= 0,
                  SPARK_ERR_INVALID, "%s: bad cache size", who);
    SPARK_REQUIRE(c->max_pages * c->page_size < (1ll << 31), SPARK_ERR_INVALID,
                  "%s: a sequence's pages hold 2^31 tokens or more", who);
    SPARK_REQUIRE(c->dtype >= 0 && c->dtype <= 2, SPARK_ERR_INVALID, "%s: bad dtype %d", who, (int)c->dtype);
    return SPARK_OK;
}

}  // namespace spark

extern "C" {

int spark_kv_append(const SparkPagedCache* cache, int64_t batch, int64_t tokens, const void* k, const int64_t* k_stride,
                    const void* v, const int64_t* v_stride, const int* index, int64_t width, const int* counts,
                    int* new_lens, int* err, void* stream) {
    using namespace spark;
    using namespace spark::kv;
    const int rc = check_cache(cache, "spark_kv_append");
    if (rc) return rc;
    SPARK_REQUIRE(batch >= 0 && batch < 65536 && tokens >= 0 && width >= 0, SPARK_ERR_INVALID,
                  "spark_kv_append: bad size (at most 65535 sequences)");
    SPARK_REQUIRE(index || width == tokens || width == 0, SPARK_ERR_INVALID, "spark_kv_append: without an index, width is tokens");
    if (batch == 0) return SPARK_OK;
    SPARK_REQUIRE(new_lens && new_lens != cache->lens, SPARK_ERR_INVALID,
                  "spark_kv_append: new_lens is null or lens itself");
    SPARK_REQUIRE(cache->k && cache->v && cache->lens && (cache->page_table || cache->max_pages == 0), SPARK_ERR_INVALID,
                  "spark_kv_append: null pointer in the cache");
    SPARK_REQUIRE((k && v && k_stride && v_stride) || width == 0, SPARK_ERR_INVALID, "spark_kv_append: null pointer");
    const int64_t extent[3] = {cache->pages, cache->page_size, cache->kv_heads};
    for (int i = 0; i < 3; ++i)
        SPARK_REQUIRE(extent[i] == 1 || (cache->k_stride[i] != 0 && cache->v_stride[i] != 0), SPARK_ERR_INVALID,
                      "spark_kv_append: rows of the cache in one place");
    Params p{};
    p.c = *cache;
    p.k = k, p.v = v;
    for (int i = 0; i < 3 && k_stride && v_stride; ++i) p.ks[i] = k_stride[i], p.vs[i] = v_stride[i];
    p.batch = batch, p.tokens = tokens, p.width = width, p.index = index, p.counts = counts;
    p.new_lens = new_lens, p.err = err;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    // 16 bytes at a time where sizes, addresses and strides let it
    const int vec = cache->dtype == SPARK_DTYPE_F32 ? 4 : 8;
    bool fits = cache->head_dim % vec == 0;
    for (const void* ptr : {k, v, (const void*)cache->k, (const void*)cache->v}) fits = fits && aligned(ptr, 16);
    for (const int64_t* st : {(const int64_t*)p.ks, (const int64_t*)p.vs, cache->k_stride, cache->v_stride})
        for (int i = 0; i < 3; ++i) fits = fits && st[i] % vec == 0;
    const int64_t row = cache->kv_heads * cache->head_dim / (fits ? vec : 1);
    p.group = 256;
    while (p.group > 8 && p.group / 2 >= row) p.group /= 2;
    const int64_t per_block = kTokens * (256 / p.group);
    const int64_t blocks = std::max<int64_t>((width + per_block - 1) / per_block, 1);
    SPARK_REQUIRE(blocks < (1ll << 31), SPARK_ERR_INVALID, "spark_kv_append: bad size");
    const dim3 grid((unsigned)blocks, (unsigned)batch);
    if (fits && vec == 4)
        launch_overlapped(k_kv_append<uint4, 4>, grid, 256, 0, s, p);
    else if (fits)
        launch_overlapped(k_kv_append<uint4, 8>, grid, 256, 0, s, p);
    else if (vec == 4)
        launch_overlapped(k_kv_append<float, 1>, grid, 256, 0, s, p);
    else
        launch_overlapped(k_kv_append<uint16_t, 1>, grid, 256, 0, s, p);
    return check_launch("spark_kv_append");
}

}  // extern "C"
