// torch_binding.cpp -- the tree-decoding calls on torch tensors: checks, output
// allocation and the C call in one step.  These calls are a few microseconds of
// GPU work at decode sizes; through ctypes their checks alone took longer.
//
// The functions return their outputs and the C entry point's status; spark_b200.ops
// raises SparkError on a status other than 0.  Workspace and stream are the
// caller's (an address and a handle).
#include <torch/extension.h>

#include <limits>
#include <variant>

#include "../../include/spark_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

int dtype_of(const Tensor& t, const char* what, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return SPARK_DTYPE_F32;
        case at::kBFloat16: return SPARK_DTYPE_BF16;
        case at::kHalf: return SPARK_DTYPE_F16;
        default: break;
    }
    TORCH_CHECK_TYPE(false, what, ": ", name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
}

void on_device(const char* what, const char* name, const Tensor& t, const Tensor& like) {
    TORCH_CHECK(t.device() == like.device(), "spark_b200.", what, ": ", name, " must be on ", like.device(), ", it is on ", t.device());
}
void need_cuda(const char* what, const char* name, const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "spark_b200.", what, ": ", name, " must be a CUDA tensor");
}
Tensor unit(const Tensor& t) { return t.dim() == 0 || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// t, or a copy where the kernels' 16-byte loads do not fit its address or strides (4-D); a tensor map has no stride 0.
Tensor tma(const Tensor& t) {
    bool fits = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) fits = fits && (t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0));
    return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
void strides(int64_t* to, const Tensor& t) {
    for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

// ------------------------------------------------------------------ rope
void rope_part(SparkRopeHeads& part, Tensor& x, OptTensor& y) {
    x = unit(x);
    if (!y) {
        y = at::empty(x.sizes(), x.options());
    } else {
        TORCH_CHECK_VALUE(y->sizes() == x.sizes() && y->scalar_type() == x.scalar_type() && y->device() == x.device() &&
                              (y->stride(-1) == 1 || y->size(-1) == 1),
                          "rope: out must have the shapes, type and device of q and k, with unit stride along the head");
    }
    part.x = x.data_ptr();
    part.y = y->data_ptr();
    part.heads = x.size(-2);
    const int first = x.dim() == 4 ? 0 : 1;   // without a batch its stride is 0
    part.xs[0] = part.ys[0] = 0;
    for (int i = first; i < 3; ++i) part.xs[i] = x.stride(i - first), part.ys[i] = y->stride(i - first);
}

std::tuple<Tensor, OptTensor, int> rope(Tensor q, OptTensor k, Tensor positions, const Tensor& table, bool interleaved,
                                        bool inverse, OptTensor q_out, OptTensor k_out, uint64_t ws, uint64_t stream) {
    need_cuda("rope", "q", q);
    on_device("rope", "positions", positions, q);
    on_device("rope", "table", table, q);
    if (k) on_device("rope", "k", *k, q);
    const at::DeviceGuard guard(q.device());
    const int64_t dim = q.dim();
    TORCH_CHECK_VALUE((dim == 3 || dim == 4) && (!k || (k->dim() == dim && k->sizes().slice(0, dim - 2) == q.sizes().slice(0, dim - 2) &&
                                                        k->size(-1) == q.size(-1))),
                      "rope: q and k must be [(batch,) tokens, heads, head_dim] of the same tokens, got ", q.sizes(), " and ",
                      k ? k->sizes() : at::IntArrayRef());
    TORCH_CHECK_TYPE(!k || k->scalar_type() == q.scalar_type(), "rope: q and k differ in type");
    TORCH_CHECK_VALUE(positions.sizes() == q.sizes().slice(0, dim - 2), "rope: positions are ", positions.sizes(),
                      ", the tokens ", q.sizes().slice(0, dim - 2));
    TORCH_CHECK_TYPE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
                     "rope: positions must be int32 or int64, got ", positions.scalar_type());
    TORCH_CHECK_TYPE(table.dim() == 2 && table.scalar_type() == at::kFloat && table.is_contiguous(),
                     "rope: table must be a contiguous float32 [rows, rot_dim]");
    const int dt = dtype_of(q, "rope", "q");
    TORCH_CHECK_VALUE(q.size(-1) <= std::numeric_limits<int>::max() && table.size(1) <= std::numeric_limits<int>::max(),
                      "rope: size");
    SparkRopeHeads part[2];
    rope_part(part[0], q, q_out);
    if (k) rope_part(part[1], *k, k_out);
    positions = positions.contiguous();
    const int64_t batch = dim == 4 ? q.size(0) : 1, tokens = q.size(dim - 3);
    const int rc = spark_rope(&part[0], k ? &part[1] : nullptr, dt, batch, tokens, (int)q.size(-1), (int)table.size(1), interleaved,
                              inverse, positions.data_ptr(), (int)positions.element_size(), table.const_data_ptr<float>(),
                              table.size(0), reinterpret_cast<int*>(ws), reinterpret_cast<void*>(stream));
    return {*q_out, k ? k_out : std::nullopt, rc};
}

// The differentiable form.  Turning is linear, its transpose is the turn back: the gradients are turned back by this
// function, so that gradients of gradients are right too.  A step backward runs on its forward's stream, with its workspace (which
// stays for as long as the process).
struct Turn : torch::autograd::Function<Turn> {
    static std::vector<Tensor> forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& positions,
                                       const Tensor& table, bool interleaved, bool inverse, uint64_t ws, uint64_t stream, int* status) {
        auto [y, z, rc] = rope(q, k, positions, table, interleaved, inverse, std::nullopt, std::nullopt, ws, stream);
        *status = rc;
        ctx->save_for_backward({positions, table});
        ctx->saved_data["how"] = (int64_t)(k.has_value() * 4 + interleaved * 2 + inverse);
        ctx->saved_data["ws"] = (int64_t)ws, ctx->saved_data["stream"] = (int64_t)stream;
        ctx->set_materialize_grads(false);
        return z ? std::vector<Tensor>{y, *z} : std::vector<Tensor>{y};
    }

    static std::vector<Tensor> backward(torch::autograd::AutogradContext* ctx, std::vector<Tensor> grads) {
        const auto saved = ctx->get_saved_variables();
        const int64_t how = ctx->saved_data["how"].toInt();
        const bool need[2] = {grads[0].defined() && ctx->needs_input_grad(0), (how & 4) && grads[1].defined() && ctx->needs_input_grad(1)};
        std::vector<Tensor> out(9);
        if (!need[0] && !need[1]) return out;
        const int first = need[0] ? 0 : 1;
        int rc = SPARK_OK;
        const auto turned = turn(grads[first], need[0] && need[1] ? OptTensor(grads[1]) : std::nullopt, saved[0], saved[1], how & 2, !(how & 1),
                                 (uint64_t)ctx->saved_data["ws"].toInt(), (uint64_t)ctx->saved_data["stream"].toInt(), &rc);
        TORCH_CHECK(rc == SPARK_OK, "spark_rope: ", spark_last_error());
        for (size_t i = 0; i < turned.size(); ++i) out[first + i] = turned[i];
        return out;
    }

    static std::vector<Tensor> turn(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& table, bool interleaved,
                                    bool inverse, uint64_t ws, uint64_t stream, int* rc) {
        if (at::GradMode::is_enabled() && (q.requires_grad() || (k && k->requires_grad())))
            return apply(q, k, positions, table, interleaved, inverse, ws, stream, rc);
        auto [y, z, status] = rope(q, k, positions, table, interleaved, inverse, std::nullopt, std::nullopt, ws, stream);
        *rc = status;
        return z ? std::vector<Tensor>{y, *z} : std::vector<Tensor>{y};
    }
};

std::tuple<Tensor, OptTensor, int> apply_rope(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& table,
                                              bool interleaved, uint64_t ws, uint64_t stream) {
    for (const Tensor* t : {&q, k ? &*k : &q, &table})
        TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "apply_rope: no forward-mode differentiation");
    int rc = SPARK_OK;
    const auto out = Turn::turn(q, k, positions, table, interleaved, false, ws, stream, &rc);
    return {out[0], k ? OptTensor(out[1]) : std::nullopt, rc};
}

// ------------------------------------------------------------------ norms of q and k with rope
// What the parts' heads are read from: x with unit stride along the head, interleaved pairs on their bytes.
Tensor pairs(const Tensor& x_, bool interleaved) {
    const Tensor x = unit(x_);
    bool fits = !interleaved || reinterpret_cast<uintptr_t>(x.data_ptr()) % (2 * x.element_size()) == 0;
    for (int64_t i = 0; interleaved && i < x.dim() - 1; ++i) fits = fits && (x.size(i) <= 1 || x.stride(i) % 2 == 0);
    return fits ? x : x.clone(at::MemoryFormat::Contiguous);
}
// strides of [(batch,) tokens, heads, head_dim]; without a batch its stride is 0
void head_strides(int64_t* to, const Tensor& x) {
    const int first = x.dim() == 4 ? 0 : 1;
    to[0] = 0;
    for (int i = first; i < 3; ++i) to[i] = x.stride(i - first);
}
struct NormInputs {
    Tensor q;
    OptTensor k, q_weight, k_weight;
    Tensor positions, table;
    double eps;
    bool interleaved;
};
// The arguments of both passes, checked; what had to be copied is held by `in`.
SparkNormRope norm_args(NormInputs& in) {
    const char* what = "qk_norm_rope";
    need_cuda(what, "q", in.q);
    on_device(what, "positions", in.positions, in.q);
    on_device(what, "table", in.table, in.q);
    const int64_t dim = in.q.dim();
    TORCH_CHECK_VALUE((dim == 3 || dim == 4) && (!in.k || (in.k->dim() == dim && in.k->sizes().slice(0, dim - 2) == in.q.sizes().slice(0, dim - 2) &&
                                                           in.k->size(-1) == in.q.size(-1))),
                      "qk_norm_rope: q and k must be [(batch,) tokens, heads, head_dim] of the same tokens, got ", in.q.sizes(), " and ",
                      in.k ? in.k->sizes() : at::IntArrayRef());
    if (in.k) on_device(what, "k", *in.k, in.q);
    TORCH_CHECK_TYPE(!in.k || in.k->scalar_type() == in.q.scalar_type(), "qk_norm_rope: q and k differ in type");
    TORCH_CHECK_VALUE(in.k || !in.k_weight, "qk_norm_rope: k_weight without k");
    TORCH_CHECK_VALUE(in.positions.sizes() == in.q.sizes().slice(0, dim - 2), "qk_norm_rope: positions are ", in.positions.sizes(),
                      ", the tokens ", in.q.sizes().slice(0, dim - 2));
    TORCH_CHECK_TYPE(in.positions.scalar_type() == at::kInt || in.positions.scalar_type() == at::kLong,
                     "qk_norm_rope: positions must be int32 or int64, got ", in.positions.scalar_type());
    TORCH_CHECK_TYPE(in.table.dim() == 2 && in.table.scalar_type() == at::kFloat && in.table.is_contiguous(),
                     "qk_norm_rope: table must be a contiguous float32 [rows, rot_dim]");
    SparkNormRope a{};
    a.dtype = dtype_of(in.q, what, "q");
    a.batch = dim == 4 ? in.q.size(0) : 1, a.tokens = in.q.size(dim - 3);
    a.head_dim = in.q.size(-1), a.rot_dim = in.table.size(1), a.interleaved = in.interleaved;
    for (int w = 0; w < 2; ++w) {
        if (w && !in.k) continue;
        Tensor& x = w ? *in.k : in.q;
        OptTensor& weight = w ? in.k_weight : in.q_weight;
        const char* name = w ? "k_weight" : "q_weight";
        x = pairs(x, in.interleaved);
        SparkNormRopeHeads& part = a.part[w];
        part.x = x.data_ptr(), part.heads = x.size(-2);
        head_strides(part.xs, x);
        if (!weight) continue;
        on_device(what, name, *weight, in.q);
        TORCH_CHECK_VALUE(weight->dim() == 1 && weight->size(0) == a.head_dim, "qk_norm_rope: ", name, " must be [", a.head_dim, "], got ",
                          weight->sizes());
        weight = weight->contiguous();
        part.weight = weight->data_ptr(), part.weight_dtype = dtype_of(*weight, what, name);
    }
    in.positions = in.positions.contiguous();
    a.positions = in.positions.data_ptr(), a.position_bytes = (int64_t)in.positions.element_size();
    a.table = in.table.const_data_ptr<float>(), a.table_rows = in.table.size(0);
    a.eps = in.eps;
    return a;
}

std::tuple<Tensor, OptTensor, int> qk_norm_rope(Tensor q, OptTensor k, OptTensor q_weight, OptTensor k_weight, Tensor positions,
                                                const Tensor& table, double eps, bool interleaved, OptTensor q_out, OptTensor k_out,
                                                uint64_t ws, uint64_t stream) {
    need_cuda("qk_norm_rope", "q", q);
    const at::DeviceGuard guard(q.device());
    TORCH_CHECK_VALUE(k || !k_out, "qk_norm_rope: an output for k without k");
    NormInputs in{q, k, q_weight, k_weight, positions, table, eps, interleaved};
    SparkNormRope a = norm_args(in);
    for (int w = 0; w < 2; ++w) {
        if (w && !k) continue;
        const Tensor& x = w ? *k : q;
        OptTensor& y = w ? k_out : q_out;
        if (!y) {
            y = at::empty(x.sizes(), x.options());
        } else {
            TORCH_CHECK_VALUE(y->sizes() == x.sizes() && y->scalar_type() == x.scalar_type() && y->device() == x.device() &&
                                  (y->stride(-1) == 1 || y->size(-1) == 1),
                              "qk_norm_rope: out must have the shapes, type and device of q and k, with unit stride along the head");
        }
        a.part[w].y = y->data_ptr();
        head_strides(a.part[w].ys, *y);
    }
    const int rc = spark_qk_norm_rope(&a, reinterpret_cast<int*>(ws), reinterpret_cast<void*>(stream));
    return {*q_out, k ? k_out : std::nullopt, rc};
}

// The gradients of q, k and the weights (undefined where not wanted), from those of the outputs (undefined: none).
std::vector<Tensor> norm_gradients(NormInputs in, const Tensor& dq, const Tensor& dk, std::array<bool, 4> want, uint64_t ws,
                                   uint64_t stream) {
    const at::DeviceGuard guard(in.q.device());
    SparkNormRope a = norm_args(in);
    std::vector<Tensor> out(4), held;
    bool weights = false;
    for (int w = 0; w < 2; ++w) {
        SparkNormRopeHeads& part = a.part[w];
        if (!(w ? dk : dq).defined() || !(want[w] || want[2 + w])) {
            part = SparkNormRopeHeads{};
            continue;
        }
        const Tensor& x = w ? *in.k : in.q;
        const Tensor g = pairs((w ? dk : dq).to(x.scalar_type()), in.interleaved);
        const Tensor dx = at::empty(x.sizes(), x.options());
        part.dy = g.data_ptr(), part.y = dx.data_ptr();
        head_strides(part.dys, g), head_strides(part.ys, dx);
        held.push_back(g), held.push_back(dx);
        if (want[w]) out[w] = dx;
        if (!want[2 + w]) continue;
        const Tensor& weight = w ? *in.k_weight : *in.q_weight;
        out[2 + w] = at::empty(weight.sizes(), weight.options());
        part.dweight = out[2 + w].data_ptr();
        weights = true;
    }
    Tensor partial;
    const size_t bytes = weights ? spark_qk_norm_rope_backward_workspace_size(a.head_dim) : 0;
    if (weights) partial = at::empty({(int64_t)bytes}, in.q.options().dtype(at::kByte));
    const int rc = spark_qk_norm_rope_backward(&a, weights ? partial.data_ptr() : nullptr, bytes, reinterpret_cast<int*>(ws),
                                               reinterpret_cast<void*>(stream));
    TORCH_CHECK(rc == SPARK_OK, "spark_qk_norm_rope_backward: ", spark_last_error());
    return out;
}

// Gradients that a graph was asked for (create_graph): they have none of their own.
struct NormGradients : torch::autograd::Function<NormGradients> {
    static std::vector<Tensor> forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const OptTensor& k, const OptTensor& q_weight,
                                       const OptTensor& k_weight, const OptTensor& dq, const OptTensor& dk, const NormInputs* in,
                                       std::array<bool, 4> want, uint64_t ws, uint64_t stream, int64_t* where) {
        NormInputs now = *in;
        now.q = q, now.k = k, now.q_weight = q_weight, now.k_weight = k_weight;
        const auto out = norm_gradients(now, dq ? *dq : Tensor(), dk ? *dk : Tensor(), want, ws, stream);
        std::vector<Tensor> defined;
        for (int i = 0; i < 4; ++i) {
            where[i] = out[i].defined() ? (int64_t)defined.size() : -1;
            if (out[i].defined()) defined.push_back(out[i]);
        }
        return defined;
    }
    static std::vector<Tensor> backward(torch::autograd::AutogradContext*, std::vector<Tensor>) {
        TORCH_CHECK_NOT_IMPLEMENTED(false, "apply_qk_norm_rope: no gradients of gradients");
        return {};
    }
};

// The differentiable form.  A step backward runs on its forward's stream, with its error word (which stays for as long as
// the process).
struct NormRope : torch::autograd::Function<NormRope> {
    static std::vector<Tensor> forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const OptTensor& k, const OptTensor& q_weight,
                                       const OptTensor& k_weight, const Tensor& positions, const Tensor& table, double eps,
                                       bool interleaved, uint64_t ws, uint64_t stream, int* status) {
        auto [y, z, rc] = qk_norm_rope(q, k, q_weight, k_weight, positions, table, eps, interleaved, std::nullopt, std::nullopt, ws, stream);
        *status = rc;
        ctx->save_for_backward({q, k ? *k : Tensor(), q_weight ? *q_weight : Tensor(), k_weight ? *k_weight : Tensor(), positions, table});
        ctx->saved_data["eps"] = eps, ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["ws"] = (int64_t)ws, ctx->saved_data["stream"] = (int64_t)stream;
        ctx->set_materialize_grads(false);
        return z ? std::vector<Tensor>{y, *z} : std::vector<Tensor>{y};
    }

    static std::vector<Tensor> backward(torch::autograd::AutogradContext* ctx, std::vector<Tensor> grads) {
        const auto saved = ctx->get_saved_variables();
        auto optional = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
        NormInputs in{saved[0], optional(saved[1]), optional(saved[2]), optional(saved[3]), saved[4], saved[5],
                      ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool()};
        const uint64_t ws = (uint64_t)ctx->saved_data["ws"].toInt(), stream = (uint64_t)ctx->saved_data["stream"].toInt();
        // (only tensors that were given have an edge)
        std::array<bool, 4> want{};
        int64_t edge = 0;
        for (int i : {0, 1, 2, 3})
            if (saved[i].defined()) want[i] = ctx->needs_input_grad(edge++);
        const Tensor dq = grads[0], dk = grads.size() > 1 ? grads[1] : Tensor();
        std::vector<Tensor> out(11);
        if (!dq.defined() && !dk.defined()) return out;
        if (at::GradMode::is_enabled()) {
            int64_t where[4];
            const auto got = NormGradients::apply(in.q, in.k, in.q_weight, in.k_weight, optional(dq), optional(dk), &in, want, ws, stream,
                                                  &where[0]);
            for (int i = 0; i < 4; ++i)
                if (where[i] >= 0) out[i] = got[where[i]];
            return out;
        }
        const auto got = norm_gradients(in, dq, dk, want, ws, stream);
        for (int i = 0; i < 4; ++i) out[i] = got[i];
        return out;
    }
};

std::tuple<Tensor, OptTensor, int> apply_qk_norm_rope(const Tensor& q, const OptTensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                                                      const Tensor& positions, const Tensor& table, double eps, bool interleaved,
                                                      bool capturing, uint64_t ws, uint64_t stream) {
    bool grad = q.requires_grad();
    TORCH_CHECK_NOT_IMPLEMENTED(!q._fw_grad(0).defined() && !table._fw_grad(0).defined(), "apply_qk_norm_rope: no forward-mode differentiation");
    for (const OptTensor* t : {&k, &q_weight, &k_weight}) {
        if (!*t) continue;
        TORCH_CHECK_NOT_IMPLEMENTED(!(*t)->_fw_grad(0).defined(), "apply_qk_norm_rope: no forward-mode differentiation");
        grad = grad || (*t)->requires_grad();
    }
    if (!grad || !at::GradMode::is_enabled())
        return qk_norm_rope(q, k, q_weight, k_weight, positions, table, eps, interleaved, std::nullopt, std::nullopt, ws, stream);
    // An eager graph of a leaf keeps the node that its gradient goes to, with its stream: the default stream's would draw that into the
    // capture when the backward pass is captured, which ends the process.
    for (const Tensor* t : {&q, k ? &*k : nullptr, q_weight ? &*q_weight : nullptr, k_weight ? &*k_weight : nullptr}) {
        if (!capturing || !t || !t->requires_grad() || t->grad_fn()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto on = node ? node->stream() : std::nullopt;
        TORCH_CHECK(!on || on->native_handle() != nullptr,
                    "apply_qk_norm_rope: under capture no graph of the same leaves on the default stream may live (drop its outputs, or make "
                    "it on another stream)");
    }
    int rc = SPARK_OK;
    const auto out = NormRope::apply(q, k, q_weight, k_weight, positions, table, eps, interleaved, ws, stream, &rc);
    return {out[0], k ? OptTensor(out[1]) : std::nullopt, rc};
}

// ------------------------------------------------------------------ the cache
SparkPagedCache paged(const char* what, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens,
                      const Tensor& tokens) {
    need_cuda(what, "k_cache", k);
    on_device(what, "v_cache", v, k);
    on_device(what, "page_table", table, k);
    on_device(what, "context_lens", lens, k);
    TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && k.stride(3) == 1 && v.stride(3) == 1, what,
                      ": k_cache and v_cache must be [pages, page_size, kv_heads, head_dim] with unit stride along the head");
    TORCH_CHECK_TYPE(k.scalar_type() == tokens.scalar_type() && v.scalar_type() == tokens.scalar_type(), what, ": the cache is ",
                     k.scalar_type(), " and ", v.scalar_type(), ", the tokens are ", tokens.scalar_type());
    TORCH_CHECK_TYPE(table.scalar_type() == at::kInt && lens.scalar_type() == at::kInt && table.dim() == 2 && lens.dim() == 1 &&
                         (table.stride(1) == 1 || table.size(1) <= 1) && lens.is_contiguous() && lens.size(0) == table.size(0),
                     what, ": page_table must be int32 [batch, max_pages], context_lens a contiguous int32 [batch]");
    SparkPagedCache c;
    c.k = k.data_ptr(), c.v = v.data_ptr();
    strides(c.k_stride, k), strides(c.v_stride, v);
    c.pages = k.size(0), c.page_size = k.size(1), c.kv_heads = k.size(2), c.head_dim = k.size(3);
    c.page_table = table.const_data_ptr<int>();
    c.page_table_stride = table.stride(0), c.max_pages = table.size(1);
    c.lens = lens.const_data_ptr<int>();
    c.dtype = dtype_of(tokens, what, "the tokens");
    return c;
}

std::tuple<Tensor, int> kv_append(const Tensor& k_new, const Tensor& v_new, const Tensor& k_cache, const Tensor& v_cache,
                                  const Tensor& page_table, const Tensor& lens, OptTensor index, const OptTensor& counts,
                                  uint64_t ws, uint64_t stream) {
    const char* what = "kv_append";
    TORCH_CHECK_VALUE(k_new.dim() == 4 && v_new.sizes() == k_new.sizes() && k_cache.dim() == 4 &&
                          k_new.sizes().slice(2) == k_cache.sizes().slice(2),
                      "kv_append: k_new and v_new must be [batch, tokens, kv_heads, head_dim] with the cache's heads, got ",
                      k_new.sizes(), " and ", v_new.sizes());
    TORCH_CHECK_TYPE(v_new.scalar_type() == k_new.scalar_type(), "kv_append: k_new and v_new differ in type");
    const SparkPagedCache cache = paged(what, k_cache, v_cache, page_table, lens, k_new);
    on_device(what, "k_new", k_new, k_cache);
    on_device(what, "v_new", v_new, k_cache);
    const int64_t batch = k_new.size(0), tokens = k_new.size(1);
    TORCH_CHECK_VALUE(lens.size(0) == batch, "kv_append: ", batch, " sequences of tokens, ", lens.size(0), " in the page table");
    int64_t width = tokens;
    if (index) {
        on_device(what, "index", *index, k_cache);
        TORCH_CHECK_TYPE(index->scalar_type() == at::kInt && index->dim() == 2 && index->size(0) == batch,
                         "kv_append: index must be int32 [batch, n]");
        index = index->contiguous();
        width = index->size(1);
    }
    if (counts) {
        on_device(what, "counts", *counts, k_cache);
        TORCH_CHECK_TYPE(counts->scalar_type() == at::kInt && counts->dim() == 1 && counts->size(0) == batch && counts->is_contiguous(),
                         "kv_append: counts must be a contiguous int32 [batch]");
    }
    const at::DeviceGuard guard(k_cache.device());
    const Tensor k = unit(k_new), v = unit(v_new);
    Tensor out = at::empty({batch}, lens.options());
    int64_t ks[3], vs[3];
    strides(ks, k), strides(vs, v);
    const int rc = spark_kv_append(&cache, batch, tokens, k.data_ptr(), ks, v.data_ptr(), vs, index ? index->const_data_ptr<int>() : nullptr,
                                   width, counts ? counts->const_data_ptr<int>() : nullptr, out.data_ptr<int>(),
                                   reinterpret_cast<int*>(ws), reinterpret_cast<void*>(stream));
    return {out, rc};
}

// ------------------------------------------------------------------ attention
// (out, lse or None, status, bytes that the workspace has to have)
std::tuple<Tensor, OptTensor, int, size_t> tree_attention(const Tensor& q_, const Tensor& k_tree, const Tensor& v_tree,
                                                          const Tensor& k_cache, const Tensor& v_cache, const Tensor& page_table,
                                                          const Tensor& lens, Tensor parents, std::optional<double> scale,
                                                          OptTensor out, bool return_lse, uint64_t ws, size_t ws_bytes,
                                                          uint64_t stream) {
    const char* what = "tree_attention";
    need_cuda(what, "q", q_);
    TORCH_CHECK_VALUE(q_.dim() == 4 && k_tree.dim() == 4 && v_tree.sizes() == k_tree.sizes() && k_tree.size(0) == q_.size(0) &&
                          k_tree.size(1) == q_.size(1),
                      "tree_attention: q must be [batch, nodes, q_heads, head_dim], k_tree and v_tree the same with kv_heads, got ",
                      q_.sizes(), ", ", k_tree.sizes(), ", ", v_tree.sizes());
    TORCH_CHECK_VALUE(k_cache.dim() == 4 && k_tree.sizes().slice(2) == k_cache.sizes().slice(2) && q_.size(3) == k_tree.size(3),
                      "tree_attention: q, k_tree, v_tree and the cache differ in heads or head_dim");
    const auto type = q_.scalar_type();
    TORCH_CHECK_TYPE((type == at::kBFloat16 || type == at::kHalf) && k_tree.scalar_type() == type && v_tree.scalar_type() == type,
                     "tree_attention: bfloat16 or float16 throughout, got ", type, ", ", k_tree.scalar_type(), ", ",
                     v_tree.scalar_type());
    on_device(what, "k_cache", k_cache, q_);
    const at::DeviceGuard guard(q_.device());
    SparkTreeAttention a;
    a.cache = paged(what, k_cache, v_cache, page_table, lens, q_);
    on_device(what, "k_tree", k_tree, q_);
    on_device(what, "v_tree", v_tree, q_);
    on_device(what, "parents", parents, q_);
    a.batch = q_.size(0), a.nodes = q_.size(1), a.q_heads = q_.size(2);
    TORCH_CHECK_VALUE(lens.size(0) == a.batch, "tree_attention: ", a.batch, " sequences of queries, ", lens.size(0),
                      " in the page table");
    const bool per_sequence = parents.dim() == 2;
    TORCH_CHECK_TYPE(parents.scalar_type() == at::kInt && (per_sequence ? parents.size(0) == a.batch : parents.dim() == 1) &&
                         parents.size(-1) == a.nodes,
                     "tree_attention: parents must be int32 [", a.nodes, "] or [", a.batch, ", ", a.nodes, "]");
    parents = unit(parents);
    if (!out)
        out = at::empty(q_.sizes(), q_.options());
    else
        TORCH_CHECK_VALUE(out->sizes() == q_.sizes() && out->scalar_type() == type && out->device() == q_.device() && out->stride(3) == 1,
                          "tree_attention: out must have q's shape, type and device, with unit stride along the head");
    const Tensor q = tma(q_), k = tma(k_tree), v = tma(v_tree);
    OptTensor lse;
    if (return_lse) lse = at::empty({a.batch, a.nodes, a.q_heads}, q_.options().dtype(at::kFloat));
    a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr(), a.out = out->data_ptr();
    strides(a.q_stride, q), strides(a.kn_stride, k), strides(a.vn_stride, v), strides(a.out_stride, *out);
    a.parents = parents.const_data_ptr<int>();
    a.parents_stride = per_sequence ? parents.stride(0) : 0;
    a.lse = lse ? lse->data_ptr<float>() : nullptr;
    a.scale = scale ? *scale : 1.0 / std::sqrt((double)q.size(3));
    const int rc = spark_tree_attention(&a, reinterpret_cast<void*>(ws), ws_bytes, reinterpret_cast<void*>(stream));
    return {*out, lse, rc, rc == SPARK_ERR_WORKSPACE ? spark_tree_attention_workspace_size(&a) : 0};
}

// ------------------------------------------------------------------ verification
std::tuple<Tensor, Tensor, Tensor, int> tree_verify(const Tensor& logits, Tensor tokens, Tensor parents, Tensor uniforms, Tensor noise,
                                                    OptTensor draft, OptTensor temperature, uint64_t ws, uint64_t stream) {
    const char* what = "tree_verify";
    need_cuda(what, "logits", logits);
    TORCH_CHECK_VALUE(logits.dim() == 3, "tree_verify: logits must be [batch, nodes, vocab], got ", logits.sizes());
    const int64_t batch = logits.size(0), nodes = logits.size(1), vocab = logits.size(2);
    on_device(what, "tokens", tokens, logits);
    on_device(what, "parents", parents, logits);
    on_device(what, "uniforms", uniforms, logits);
    on_device(what, "noise", noise, logits);
    const auto per_node = logits.sizes().slice(0, 2);
    TORCH_CHECK_VALUE(tokens.sizes() == per_node && uniforms.sizes() == per_node && noise.dim() == 2 && noise.size(0) == batch &&
                          noise.size(1) == vocab,
                      "tree_verify: tokens and uniforms must be [", batch, ", ", nodes, "], noise [", batch, ", ", vocab, "]");
    TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong && uniforms.scalar_type() == at::kFloat && noise.scalar_type() == at::kFloat,
                     "tree_verify: tokens must be int64, uniforms and noise float32");
    const bool per_sequence = parents.dim() == 2;
    TORCH_CHECK_TYPE(parents.scalar_type() == at::kInt && (per_sequence ? parents.size(0) == batch : parents.dim() == 1) &&
                         parents.size(-1) == nodes,
                     "tree_verify: parents must be int32 [", nodes, "] or [", batch, ", ", nodes, "]");
    const at::DeviceGuard guard(logits.device());
    SparkTreeVerify a{};
    a.batch = batch, a.nodes = nodes, a.vocab = vocab;
    const Tensor x = unit(logits);
    a.logits = x.data_ptr(), a.logits_dtype = dtype_of(x, what, "logits");
    a.logits_stride[0] = x.stride(0), a.logits_stride[1] = x.stride(1);
    if (draft) {
        on_device(what, "draft_probs", *draft, logits);
        TORCH_CHECK_VALUE(draft->sizes() == logits.sizes(), "tree_verify: draft_probs are ", draft->sizes(), ", logits ", logits.sizes());
        draft = unit(*draft);
        a.draft = draft->data_ptr(), a.draft_dtype = dtype_of(*draft, what, "draft_probs");
        a.draft_stride[0] = draft->stride(0), a.draft_stride[1] = draft->stride(1);
    }
    if (temperature) {
        TORCH_CHECK_TYPE(temperature->scalar_type() == at::kFloat && temperature->dim() == 1 && temperature->size(0) == batch &&
                             temperature->device() == logits.device(),
                         "tree_verify: temperature must be a number or float32 [", batch, "] on ", logits.device());
        temperature = temperature->contiguous();
        a.temperature = temperature->const_data_ptr<float>();
    }
    tokens = unit(tokens), parents = unit(parents), uniforms = unit(uniforms), noise = unit(noise);
    const auto ints = logits.options().dtype(at::kInt);
    Tensor path = at::empty(per_node, ints), accepted = at::empty({batch}, ints), next = at::empty({batch}, ints.dtype(at::kLong));
    a.tokens = tokens.const_data_ptr<int64_t>(), a.tokens_stride = tokens.stride(0);
    a.parents = parents.const_data_ptr<int>(), a.parents_stride = per_sequence ? parents.stride(0) : 0;
    a.uniforms = uniforms.const_data_ptr<float>(), a.uniforms_stride = uniforms.stride(0);
    a.noise = noise.const_data_ptr<float>(), a.noise_stride = noise.stride(0);
    a.path = path.data_ptr<int>(), a.accepted = accepted.data_ptr<int>(), a.next = next.data_ptr<int64_t>();
    const int rc = spark_tree_verify(&a, reinterpret_cast<int*>(ws), reinterpret_cast<void*>(stream));
    return {path, accepted, next, rc};
}

// ------------------------------------------------------------------ sampling
// One setting of all sequences, or a tensor [batch] (which comes first: one of a single value converts to a number, on the host).
template <typename N>
using Setting = std::variant<Tensor, N>;
template <typename T, typename N>
const T* setting(const char* what, const char* name, Setting<N>& s, N& all, at::ScalarType type, int64_t batch, const Tensor& like) {
    if (const N* one = std::get_if<N>(&s)) {
        all = *one;
        return nullptr;
    }
    Tensor& t = std::get<Tensor>(s);
    TORCH_CHECK_TYPE(t.scalar_type() == type && t.dim() == 1 && t.size(0) == batch && t.device() == like.device(), what, ": ", name,
                     " must be a number or ", type, " [", batch, "] on ", like.device());
    t = t.contiguous();
    return t.const_data_ptr<T>();
}
SparkSample sample_args(const char* what, const Tensor& logits, int64_t batch, Setting<double>& temperature, Setting<int64_t>& top_k,
                        Setting<double>& top_p, Setting<double>& min_p) {
    SparkSample a{};
    a.batch = batch, a.nodes = logits.dim() == 3 ? logits.size(1) : 1, a.vocab = logits.size(-1);
    a.logits = logits.data_ptr(), a.dtype = dtype_of(logits, what, "logits");
    a.logits_stride[0] = logits.stride(0), a.logits_stride[1] = logits.dim() == 3 ? logits.stride(1) : 0;
    a.temperature = setting<float>(what, "temperature", temperature, a.temperature_all, at::kFloat, batch, logits);
    a.top_k = setting<int>(what, "top_k", top_k, a.top_k_all, at::kInt, batch, logits);
    a.top_p = setting<float>(what, "top_p", top_p, a.top_p_all, at::kFloat, batch, logits);
    a.min_p = setting<float>(what, "min_p", min_p, a.min_p_all, at::kFloat, batch, logits);
    TORCH_CHECK_VALUE(a.temperature || a.temperature_all >= 0, what, ": temperature must be 0 or above, got ", a.temperature_all);
    TORCH_CHECK_VALUE(a.top_k || a.top_k_all >= 0, what, ": top_k must be 0 (all) or above, got ", a.top_k_all);
    TORCH_CHECK_VALUE(a.top_p || (a.top_p_all >= 0 && a.top_p_all <= 1), what, ": top_p must be in 0..1, got ", a.top_p_all);
    TORCH_CHECK_VALUE(a.min_p || (a.min_p_all >= 0 && a.min_p_all <= 1), what, ": min_p must be in 0..1, got ", a.min_p_all);
    return a;
}

std::tuple<Tensor, OptTensor, int> sample(const Tensor& logits, Tensor noise, Setting<double> temperature, Setting<int64_t> top_k,
                                          Setting<double> top_p, Setting<double> min_p, bool return_logprob, uint64_t stream) {
    const char* what = "sample";
    need_cuda(what, "logits", logits);
    TORCH_CHECK_VALUE(logits.dim() == 2 && logits.size(1) >= 1, "sample: logits must be [batch, vocab], got ", logits.sizes());
    on_device(what, "noise", noise, logits);
    TORCH_CHECK_TYPE(noise.scalar_type() == at::kFloat, "sample: noise must be float32");
    TORCH_CHECK_VALUE(noise.sizes() == logits.sizes(), "sample: noise is ", noise.sizes(), ", logits ", logits.sizes());
    const at::DeviceGuard guard(logits.device());
    const Tensor x = unit(logits);
    noise = unit(noise);
    SparkSample a = sample_args(what, x, x.size(0), temperature, top_k, top_p, min_p);
    a.noise = noise.const_data_ptr<float>(), a.noise_stride = noise.stride(0);
    Tensor token = at::empty({a.batch}, x.options().dtype(at::kLong));
    OptTensor logprob;
    if (return_logprob) logprob = at::empty({a.batch}, x.options().dtype(at::kFloat));
    a.token = token.data_ptr<int64_t>(), a.logprob = logprob ? logprob->data_ptr<float>() : nullptr;
    return {token, logprob, spark_sample(&a, reinterpret_cast<void*>(stream))};
}

std::tuple<Tensor, int> filter_logits(const Tensor& logits, Setting<double> temperature, Setting<int64_t> top_k, Setting<double> top_p,
                                      Setting<double> min_p, OptTensor out, uint64_t stream) {
    const char* what = "filter_logits";
    need_cuda(what, "logits", logits);
    TORCH_CHECK_VALUE((logits.dim() == 2 || logits.dim() == 3) && logits.size(-1) >= 1,
                      "filter_logits: logits must be [batch, (nodes,) vocab], got ", logits.sizes());
    const at::DeviceGuard guard(logits.device());
    const Tensor x = unit(logits);
    if (!out)
        out = at::empty(x.sizes(), x.options());
    else
        TORCH_CHECK_VALUE(out->sizes() == x.sizes() && out->scalar_type() == x.scalar_type() && out->device() == x.device() &&
                              (out->stride(-1) == 1 || out->size(-1) == 1),
                          "filter_logits: out must have the logits' shape, type and device, with unit stride along the vocabulary");
    SparkSample a = sample_args(what, x, x.size(0), temperature, top_k, top_p, min_p);
    a.out = out->data_ptr(), a.out_stride[0] = out->stride(0), a.out_stride[1] = out->dim() == 3 ? out->stride(1) : 0;
    return {*out, spark_sample(&a, reinterpret_cast<void*>(stream))};
}

// ------------------------------------------------------------------ adapters
// [rows, n] of a tensor [..., n], its rows at one distance.
Tensor rows_of(const Tensor& t) { return unit(t.reshape({-1, t.size(-1)})); }

std::tuple<Tensor, int> lora_add(const Tensor& y_, const Tensor& x_, const Tensor& a, const Tensor& b, Tensor adapter, Setting<double> scale,
                                 OptTensor out, uint64_t ws, uint64_t stream) {
    const char* what = "lora_add";
    need_cuda(what, "y", y_);
    for (const auto& [name, t] : {std::pair<const char*, const Tensor*>{"x", &x_}, {"a", &a}, {"b", &b}, {"adapter", &adapter}})
        on_device(what, name, *t, y_);
    TORCH_CHECK_VALUE(y_.dim() >= 1 && x_.dim() == y_.dim() && x_.sizes().slice(0, x_.dim() - 1) == y_.sizes().slice(0, y_.dim() - 1),
                      "lora_add: x must be [..., in_features] and y [..., out_features] of the same tokens, got ", x_.sizes(), " and ",
                      y_.sizes());
    const int64_t ic = x_.size(-1), oc = y_.size(-1);
    TORCH_CHECK_VALUE(a.dim() == 3 && b.dim() == 3 && a.size(0) == b.size(0) && a.size(1) == b.size(2) && a.size(2) == ic && b.size(1) == oc,
                      "lora_add: a must be [adapters, rank, ", ic, "] and b [adapters, ", oc, ", rank], got ", a.sizes(), " and ", b.sizes());
    TORCH_CHECK_VALUE(ic >= 1 && a.size(1) >= 1, "lora_add: no features or a rank of 0");
    const auto type = x_.scalar_type();
    TORCH_CHECK_TYPE((type == at::kBFloat16 || type == at::kHalf) && a.scalar_type() == type && b.scalar_type() == type &&
                         (y_.scalar_type() == type || y_.scalar_type() == at::kFloat),
                     "lora_add: x, a and b must be bfloat16 or float16 alike, y of that type or float32, got ", type, ", ", a.scalar_type(), ", ",
                     b.scalar_type(), ", ", y_.scalar_type());
    TORCH_CHECK_TYPE(adapter.scalar_type() == at::kInt, "lora_add: adapter must be int32, got ", adapter.scalar_type());
    SparkLora p{};
    p.tokens = 1;
    for (int64_t i = 0; i < x_.dim() - 1; ++i) p.tokens *= x_.size(i);
    TORCH_CHECK_VALUE(p.tokens == 0 || (adapter.numel() >= 1 && p.tokens % adapter.numel() == 0), "lora_add: ", adapter.numel(),
                      " adapter numbers for ", p.tokens, " tokens: their number must divide the tokens'");
    const at::DeviceGuard guard(y_.device());
    if (!out) {
        out = at::empty(y_.sizes(), y_.options());
    } else {
        TORCH_CHECK_VALUE(out->sizes() == y_.sizes() && out->scalar_type() == y_.scalar_type() && out->device() == y_.device(),
                          "lora_add: out must have y's shape, type and device");
    }
    if (p.tokens == 0 || oc == 0) return {*out, SPARK_OK};
    // (a copy of out would take the result with it)
    const Tensor to = out->view({-1, oc}), x = rows_of(x_), y = out->is_same(y_) ? to : rows_of(y_);
    TORCH_CHECK_VALUE(to.stride(1) == 1 || oc == 1, "lora_add: out must have unit stride along the features");
    const Tensor ac = a.contiguous(), bc = b.contiguous();
    adapter = adapter.contiguous();
    p.ic = ic, p.oc = oc, p.rank = a.size(1), p.adapters = a.size(0), p.repeat = p.tokens / adapter.numel();
    p.dtype = dtype_of(x, what, "x"), p.y_dtype = dtype_of(y, what, "y");
    p.x = x.data_ptr(), p.a = ac.data_ptr(), p.b = bc.data_ptr(), p.y = y.data_ptr(), p.out = to.data_ptr();
    p.ldx = x.stride(0), p.ldy = y.stride(0), p.ldo = to.stride(0);
    p.adapter = adapter.const_data_ptr<int>();
    p.scale = setting<float>(what, "scale", scale, p.scale_all, at::kFloat, p.adapters, y_);
    const size_t bytes = spark_lora_workspace_size(p.tokens, ic, p.rank);
    const Tensor h = at::empty({(int64_t)bytes}, y_.options().dtype(at::kByte));
    return {*out, spark_lora(&p, h.data_ptr(), bytes, reinterpret_cast<int*>(ws), reinterpret_cast<void*>(stream))};
}

}  // namespace

PYBIND11_MODULE(_native, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const c10::TypeError& e) {
            PyErr_SetString(PyExc_TypeError, e.what_without_backtrace());
        } catch (const c10::ValueError& e) {
            PyErr_SetString(PyExc_ValueError, e.what_without_backtrace());
        } catch (const c10::NotImplementedError& e) {
            PyErr_SetString(PyExc_NotImplementedError, e.what_without_backtrace());
        } catch (const c10::Error& e) {
            PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
        }
    });
    m.def("rope", &rope);
    m.def("apply_rope", &apply_rope);
    m.def("qk_norm_rope", &qk_norm_rope);
    m.def("apply_qk_norm_rope", &apply_qk_norm_rope);
    m.def("kv_append", &kv_append);
    m.def("tree_attention", &tree_attention);
    m.def("tree_verify", &tree_verify);
    m.def("sample", &sample);
    m.def("filter_logits", &filter_logits);
    m.def("lora_add", &lora_add);
}
