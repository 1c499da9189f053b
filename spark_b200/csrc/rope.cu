// rope.cu -- rotary positions of q and k.
//
// For pair i of a head at position p, with c = table[p, i] and
// s = table[p, r / 2 + i]:  (a, b) -> (a c - b s, b c + a s), the rotation of
// (a, b) by the pair's angle; its transpose, the backward pass, is s -> -s.
// Arithmetic is fp32, rounded once to the tensors' type.
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
        store_from_float(t.y, p.dtype, yo + da, good ? va * c - vb * sn : 0.f);
        store_from_float(t.y, p.dtype, yo + db, good ? vb * c + va * sn : 0.f);
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
    const int64_t n = p.n_tokens * (p.part[0].heads + p.part[1].heads) * (rot_dim / 2 + head_dim - rot_dim);
    if (n == 0) return SPARK_OK;
    const int grid = (int)std::min<int64_t>((n + 255) / 256, 148 * 16);
    k_rope<<<grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
    return check_launch("spark_rope");
}

}  // extern "C"
