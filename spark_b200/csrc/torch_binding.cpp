// torch_binding.cpp -- the tree-decoding calls on torch tensors: checks, output
// allocation and the C call in one step.  These calls are a few microseconds of
// GPU work at decode sizes; through ctypes their checks alone took longer.
//
// The functions return their outputs and the C entry point's status; spark_b200.ops
// raises SparkError on a status other than 0.  Workspace and stream are the
// caller's (an address and a handle).
#include <torch/extension.h>

#include <limits>

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
    m.def("kv_append", &kv_append);
    m.def("tree_attention", &tree_attention);
    m.def("tree_verify", &tree_verify);
}
