// torch_ops.cpp — the training operators as autograd nodes over the C ABI.
//
// A step of a small model is bound by the host: written in Python, forward and
// backward of one operator took 115 us of it (a Python function in the
// engine's thread, a dozen converted arguments a call), of which the kernels
// need a third.  Here a call allocates its outputs, hands over plain pointers
// and links one node into the graph.  Arguments are checked by the Python
// functions that call these (norm.py, distill.py, attention.py, embed.py, rotary.py, saved8.py).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <initializer_list>
#include <limits>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/concord_b200.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

void check(int status, const char* name) {
    if (status == 0) return;
    static const char* const kinds[] = {"invalid argument", "unsupported shape/stride", "unsupported alignment",
                                        "workspace missing or too small", "CUDA launch/runtime error",
                                        "no usable CUDA device", "size above the fixed maximum",
                                        "a wait ran out"};
    const char* kind = status <= -1 && status >= -8 ? kinds[-status - 1] : "error";
    throw std::runtime_error(std::string(name) + " failed: " + kind + ": " + concord_last_error());
}

int32_t type_code(const Tensor& t) {
    return t.scalar_type() == at::kFloat ? CONCORD_F32 : t.scalar_type() == at::kBFloat16 ? CONCORD_BF16 : CONCORD_F16;
}

void* current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
template <typename T> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor get(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }

// The kernels are no torch operators: a trace would record the allocation of
// their outputs alone.  And a tangent of forward-mode differentiation is no part
// of what they read: it would be lost, and the derivative read as zero.
void refuse_transforms(std::initializer_list<Tensor> inputs, const char* name) {
    using c10::impl::TorchDispatchModeKey;
    TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                    !c10::impl::TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY).has_value(),
                name, " cannot be traced: its kernels are not torch operators");
    for (const Tensor& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), name,
                                    ": forward-mode differentiation is not supported (it has a backward pass only)");
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A gradient that has no gradient itself: where the upstream one would pass on
// a second derivative, the results get a node that says so when it is reached
// (which DelayedError attaches to inputs that require a gradient only).
variable_list once(variable_list grads, const variable_list& upstream) {
    if (!at::GradMode::is_enabled()) return grads;
    bool second = false;
    for (const Tensor& g : upstream) second |= wants_grad(g);
    if (!second) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g.set_requires_grad(true);
    return torch::autograd::DelayedError(
        "trying to differentiate twice a function that was marked with @once_differentiable",
        (int64_t)grads.size())(std::move(grads));
}

template <typename Node, typename... In> std::shared_ptr<Node> link(const In&... in) {
    std::shared_ptr<Node> node(new Node(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(in...));
    return node;
}

// t as [N, D] with contiguous columns (a copy only where it has none)
Tensor rows(const Tensor& t, int64_t D) {
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, D});
    if (!r.is_contiguous() && (r.stride(1) != 1 || (r.size(0) > 1 && r.stride(0) < D))) r = r.contiguous();
    return r;
}
int64_t ld(const Tensor& r, int64_t D) { return r.size(0) > 1 ? r.stride(0) : D; }

// ---------------------------------------------------------------- layer norm
struct LayerNormBackward : public torch::autograd::Node {
    SavedVariable x_, weight_, stats_;
    std::vector<int64_t> shape;
    std::string name() const override { return "ConcordLayerNormBackward"; }
    void release_variables() override { x_.reset_data(); weight_.reset_data(); stats_.reset_data(); }
    variable_list apply(variable_list&& g) override {
        const Tensor x = x_.unpack(), w = weight_.unpack(), stats = stats_.unpack();
        variable_list out(3);
        if (!g[0].defined()) return out;
        variable_list res;
        {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(x.device());
            const int64_t N = x.size(0), D = x.size(1);
            const Tensor dy = rows(g[0], D);
            const bool need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
            out[0] = at::empty(shape, x.options());
            if (need_w) out[1] = at::empty({D}, stats.options());
            if (need_b) out[2] = at::empty({D}, stats.options());
            Tensor ws;
            size_t bytes = 0;
            if (need_w || need_b) {
                bytes = concord_layer_norm_bwd_workspace_bytes(N, D);
                ws = at::empty({(int64_t)(bytes / 4 + 1)}, stats.options());
            }
            const float* mean = ptr<float>(stats);
            check(concord_layer_norm_bwd(ptr(x), type_code(x), ld(x, D), ptr(dy), type_code(dy), ld(dy, D), ptr<float>(w),
                                         mean, mean + N, ptr(out[0]), ptr<float>(out[1]), ptr<float>(out[2]), N, D,
                                         ptr(ws), bytes, current_stream()),
                  "concord_layer_norm_bwd");
        }
        return once(std::move(out), g);
    }
};

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, int64_t out_code) {
    const Tensor w = get(weight), b = get(bias);
    refuse_transforms({x, w, b}, "layer_norm");
    const bool grad = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b));
    c10::cuda::CUDAGuard guard(x.device());
    Tensor y, x2, stats;
    const int64_t D = x.size(-1);
    {
        at::NoGradGuard no_grad;
        x2 = rows(x, D);
        const int64_t N = x2.size(0);
        y = at::empty(x.sizes(), x.options().requires_grad(false).dtype(
                                     out_code == CONCORD_F32 ? at::kFloat : out_code == CONCORD_BF16 ? at::kBFloat16 : at::kHalf));
        if (grad) stats = at::empty({2 * N}, y.options().dtype(at::kFloat));     // means, then 1 / deviations
        float* mean = ptr<float>(stats);
        check(concord_layer_norm_fwd(ptr(x2), type_code(x2), ld(x2, D), ptr<float>(w), ptr<float>(b), ptr(y),
                                     (int32_t)out_code, mean, mean ? mean + N : nullptr, N, D, (float)eps, current_stream()),
              "concord_layer_norm_fwd");
    }
    if (grad) {
        auto node = link<LayerNormBackward>(x, w, b);
        node->x_ = SavedVariable(x2, false);
        node->weight_ = SavedVariable(w, false);
        node->stats_ = SavedVariable(stats, false);
        node->shape = x.sizes().vec();
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---------------------------------------------------------------- distillation loss
concord_distill_params distill_params(const Tensor& ids, const Tensor& labels, double temperature, double alpha,
                                      int64_t ignore, bool mean, double scale) {
    concord_distill_params p{};
    p.temperature = (float)temperature;
    p.alpha = (float)alpha;
    p.grad_scale = (float)scale;
    p.mean = mean;
    p.ids64 = ids.scalar_type() == at::kLong;
    p.labels64 = labels.defined() && labels.scalar_type() == at::kLong;
    p.ignore_index = ignore;
    return p;
}

struct DistillBackward : public torch::autograd::Node {
    SavedVariable z_, ids_, t_, labels_, stats_;
    std::vector<int64_t> shape;
    concord_distill_params params{};
    bool per_row = false;
    std::string name() const override { return "ConcordDistillBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&z_, &ids_, &t_, &labels_, &stats_}) v->reset_data();
    }
    variable_list apply(variable_list&& g) override {
        const Tensor z = z_.unpack(), ids = ids_.unpack(), t = t_.unpack(), labels = labels_.unpack(),
                     stats = stats_.unpack();
        variable_list out(1);
        if (!g[0].defined()) return out;
        {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(z.device());
            const int64_t N = z.size(0), V = z.size(1);
            const Tensor up = g[0].contiguous();
            out[0] = at::empty(shape, z.options());
            check(concord_distill_grad(&params, ptr(z), type_code(z), ld(z, V), ptr(ids), ptr<float>(t), ptr(labels),
                                       ptr<float>(stats), ptr<float>(up), per_row, ptr(out[0]), N, V, ids.size(1),
                                       current_stream()),
                  "concord_distill_grad");
        }
        return once(std::move(out), g);
    }
};

struct DistillArgs {
    Tensor z, ids, t, labels;
    DistillArgs(const Tensor& logits, const Tensor& top_ids, const Tensor& top_logits, const MaybeTensor& lab) {
        const int64_t V = logits.size(-1), K = top_ids.size(-1);
        z = rows(logits, V);
        ids = (top_ids.dim() == 2 ? top_ids : top_ids.reshape({-1, K})).contiguous();
        t = (top_logits.dim() == 2 ? top_logits : top_logits.reshape({-1, K})).to(at::kFloat).contiguous();
        if (lab.has_value()) labels = lab->reshape({-1}).contiguous();
    }
    void loss(const concord_distill_params& p, float* loss, float* row_loss, float* stats, void* dz) const {
        const int64_t N = z.size(0), V = z.size(1);
        const size_t bytes = concord_distill_workspace_bytes(N);
        const Tensor ws = at::empty({(int64_t)bytes}, z.options().requires_grad(false).dtype(at::kByte));
        check(concord_distill_loss(&p, ptr(z), type_code(z), ld(z, V), ptr(ids), ptr<float>(t), ptr(labels), loss,
                                   row_loss, stats, dz, N, V, ids.size(1), ptr(ws), bytes, current_stream()),
              "concord_distill_loss");
    }
};

// reduction: 0 mean, 1 sum, 2 none
Tensor distill_loss(const Tensor& logits, const Tensor& top_ids, const Tensor& top_logits, const MaybeTensor& labels,
                    double temperature, double alpha, int64_t ignore, int64_t reduction) {
    refuse_transforms({logits, top_logits}, "distill_loss");
    const bool grad = at::GradMode::is_enabled() && wants_grad(logits), per_row = reduction == 2;
    c10::cuda::CUDAGuard guard(logits.device());
    Tensor out, stats;
    std::shared_ptr<DistillBackward> node;
    {
        at::NoGradGuard no_grad;
        const DistillArgs A(logits, top_ids, top_logits, labels);
        const auto p = distill_params(A.ids, A.labels, temperature, alpha, ignore, reduction == 0, 1.0);
        const auto f32 = logits.options().requires_grad(false).dtype(at::kFloat);
        out = per_row ? at::empty(logits.sizes().slice(0, logits.dim() - 1), f32) : at::empty({}, f32);
        if (grad) stats = at::empty({3 * A.z.size(0) + 1}, f32);
        A.loss(p, per_row ? nullptr : ptr<float>(out), per_row ? ptr<float>(out) : nullptr, ptr<float>(stats), nullptr);
        if (grad) {
            node = link<DistillBackward>(logits);
            node->z_ = SavedVariable(A.z, false);
            node->ids_ = SavedVariable(A.ids, false);
            node->t_ = SavedVariable(A.t, false);
            node->labels_ = SavedVariable(A.labels, false);
            node->stats_ = SavedVariable(stats, false);
            node->shape = logits.sizes().vec();
            node->params = p;
            node->per_row = per_row;
        }
    }
    if (node) torch::autograd::set_history(out, node);
    return out;
}

std::tuple<Tensor, Tensor> distill_loss_and_grad(const Tensor& logits, const Tensor& top_ids, const Tensor& top_logits,
                                                 const MaybeTensor& labels, double temperature, double alpha,
                                                 int64_t ignore, bool mean, double grad_scale) {
    refuse_transforms({logits, top_logits}, "distill_loss_and_grad");
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(logits.device());
    const DistillArgs A(logits, top_ids, top_logits, labels);
    const auto p = distill_params(A.ids, A.labels, temperature, alpha, ignore, mean, grad_scale);
    const Tensor loss = at::empty({}, logits.options().requires_grad(false).dtype(at::kFloat));
    const Tensor dz = at::empty(logits.sizes(), logits.options().requires_grad(false));
    A.loss(p, ptr<float>(loss), nullptr, nullptr, ptr(dz));
    return {loss, dz};
}

// ---------------------------------------------------------------- attention
// t [T, H, D] as the kernels read it (a copy only where its strides or its
// address do not fit 16-byte rows).  The stride of a dimension of size one says
// nothing: the dense one is taken for it.
Tensor operand(const Tensor& t) {
    const int64_t H = t.size(1), D = t.size(2);
    const int64_t ts = t.size(0) > 1 ? t.stride(0) : H * D, hs = H > 1 ? t.stride(1) : D;
    if (t.stride(2) == 1 && ts % 8 == 0 && hs % 8 == 0 && ts > 0 && hs > 0 &&
        reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
        return ts == t.stride(0) && hs == t.stride(1) ? t : t.as_strided(t.sizes(), {ts, hs, 1});
    return at::empty(t.sizes(), t.options()).copy_(t);
}

concord_attention_params attention_params(const Tensor& q, const Tensor& k, const Tensor& cu_q, const Tensor& cu_k,
                                          bool causal, double scale) {
    concord_attention_params p{};
    p.cu_q = ptr<int32_t>(cu_q);
    p.cu_k = ptr<int32_t>(cu_k);
    p.seqs = cu_q.numel() - 1;
    p.tokens_q = q.size(0);
    p.tokens_k = k.size(0);
    p.heads = q.size(1);
    p.kv_heads = k.size(1);
    p.head_dim = q.size(2);
    p.type = type_code(q);
    p.causal = causal;
    p.scale = (float)scale;
    return p;
}

struct AttentionBackward : public torch::autograd::Node {
    SavedVariable q_, k_, v_, cu_q_, cu_k_, o_, rest_, lse_;
    bool causal = false;
    double scale = 0;
    std::string name() const override { return "ConcordAttentionBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&q_, &k_, &v_, &cu_q_, &cu_k_, &o_, &rest_, &lse_}) v->reset_data();
    }
    variable_list apply(variable_list&& g) override {
        const Tensor q = q_.unpack(), k = k_.unpack(), v = v_.unpack(), cu_q = cu_q_.unpack(), cu_k = cu_k_.unpack(),
                     o = o_.unpack(shared_from_this()), rest = rest_.unpack(), lse = lse_.unpack();
        variable_list out(3);
        if (!g[0].defined()) return out;
        {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(q.device());
            const auto plain = q.options().requires_grad(false);
            if (q.size(0) == 0 || k.size(0) == 0) {
                out = {at::zeros(q.sizes(), plain), at::zeros(k.sizes(), plain), at::zeros(v.sizes(), plain)};
            } else {
                out = {at::empty(q.sizes(), plain), at::empty(k.sizes(), plain), at::empty(v.sizes(), plain)};
                const Tensor up = operand(g[0]), delta = at::empty(lse.sizes(), lse.options());
                const auto p = attention_params(q, k, cu_q, cu_k, causal, scale);
                const size_t bytes = concord_attention_bwd_workspace_bytes(&p);
                Tensor ws;
                if (bytes > 0) ws = at::empty({(int64_t)bytes}, plain.dtype(at::kByte));
                check(concord_attention_bwd(&p, ptr(q), q.stride(0), q.stride(1), ptr(k), k.stride(0), k.stride(1),
                                            ptr(v), v.stride(0), v.stride(1), ptr(o), ptr(rest), ptr<float>(lse),
                                            ptr(up), up.stride(0), up.stride(1), ptr<float>(delta), ptr(out[0]),
                                            ptr(out[1]), ptr(out[2]), ptr(ws), bytes, current_stream()),
                      "concord_attention_bwd");
            }
        }
        return once(std::move(out), g);
    }
};

std::tuple<Tensor, Tensor> attention(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& cu_q,
                                     const Tensor& cu_k, bool causal, double scale) {
    refuse_transforms({q0, k0, v0}, "packed_attention");
    const bool grad = at::GradMode::is_enabled() && (wants_grad(q0) || wants_grad(k0) || wants_grad(v0));
    c10::cuda::CUDAGuard guard(q0.device());
    Tensor q, k, v, o, rest, lse;
    {
        at::NoGradGuard no_grad;
        q = operand(q0);
        k = operand(k0);
        v = operand(v0);
        const auto plain = q0.options().requires_grad(false);
        o = at::empty(q.sizes(), plain);
        if (grad) rest = at::empty(q.sizes(), plain);
        lse = at::empty({q.size(1), q.size(0)}, plain.dtype(at::kFloat));
        if (k.size(0) == 0) {
            // (a row of no sequence has lse 0, as the kernels give it)
            const Tensor row = at::arange(q.size(0), cu_q.options());
            const Tensor none = row.lt(cu_q[0]).logical_or_(row.ge(cu_q[-1]));
            o.zero_();
            lse.fill_(-std::numeric_limits<float>::infinity()).masked_fill_(none, 0.f);
        } else if (q.size(0) > 0) {
            const auto p = attention_params(q, k, cu_q, cu_k, causal, scale);
            check(concord_attention_fwd(&p, ptr(q), q.stride(0), q.stride(1), ptr(k), k.stride(0), k.stride(1), ptr(v),
                                        v.stride(0), v.stride(1), ptr(o), ptr(rest), ptr<float>(lse), current_stream()),
                  "concord_attention_fwd");
        }
    }
    if (grad) {
        auto node = link<AttentionBackward>(q0, k0, v0);
        node->q_ = SavedVariable(q, false);
        node->k_ = SavedVariable(k, false);
        node->v_ = SavedVariable(v, false);
        node->cu_q_ = SavedVariable(cu_q, false);
        node->cu_k_ = SavedVariable(cu_k, false);
        node->rest_ = SavedVariable(rest, false);
        node->lse_ = SavedVariable(lse, false);
        node->causal = causal;
        node->scale = scale;
        torch::autograd::set_history(o, node);
        node->o_ = SavedVariable(o, true);
    }
    return {o, lse};
}

// ---------------------------------------------------------------- embedding
at::ScalarType type_of(int64_t code) {
    return code == CONCORD_F32 ? at::kFloat : code == CONCORD_BF16 ? at::kBFloat16 : at::kHalf;
}
Tensor bytes_like(const Tensor& t, size_t bytes) {
    return at::empty({(int64_t)bytes}, t.options().requires_grad(false).dtype(at::kByte));
}

struct EmbeddingBackward : public torch::autograd::Node {
    SavedVariable ids_;
    at::TensorOptions options;
    int64_t V = 0, D = 0, padding = -1;
    double scale = 1;
    std::string name() const override { return "ConcordEmbeddingBackward"; }
    void release_variables() override { ids_.reset_data(); }
    variable_list apply(variable_list&& g) override {
        const Tensor ids = ids_.unpack();
        variable_list out(1);
        if (!g[0].defined()) return out;
        {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(ids.device());
            const Tensor dy = rows(g[0], D);
            const int64_t T = ids.numel();
            out[0] = at::empty({V, D}, options);
            const size_t bytes = concord_embedding_bwd_workspace_bytes(T, V, D);
            const Tensor ws = bytes_like(ids, bytes);
            check(concord_embedding_bwd(ptr(ids), ids.scalar_type() == at::kLong, ptr(dy), type_code(dy), ld(dy, D),
                                        ptr(out[0]), type_code(out[0]), T, V, D, (float)scale, padding, ptr(ws), bytes,
                                        current_stream()),
                  "concord_embedding_bwd");
        }
        return once(std::move(out), g);
    }
};

Tensor embedding(const Tensor& ids0, const Tensor& weight, double scale, int64_t padding, int64_t out_code) {
    refuse_transforms({weight}, "embedding");
    const bool grad = at::GradMode::is_enabled() && wants_grad(weight);
    c10::cuda::CUDAGuard guard(weight.device());
    const int64_t V = weight.size(0), D = weight.size(1);
    Tensor y, ids;
    {
        at::NoGradGuard no_grad;
        ids = ids0.reshape({-1}).contiguous();
        const Tensor w = rows(weight, D);
        auto shape = ids0.sizes().vec();
        shape.push_back(D);
        y = at::empty(shape, weight.options().requires_grad(false).dtype(type_of(out_code)));
        check(concord_embedding_fwd(ptr(ids), ids.scalar_type() == at::kLong, ptr(w), type_code(w), ld(w, D), ptr(y),
                                    (int32_t)out_code, ids.numel(), V, D, (float)scale, current_stream()),
              "concord_embedding_fwd");
    }
    if (grad) {
        auto node = link<EmbeddingBackward>(weight);
        node->ids_ = SavedVariable(ids, false);
        node->options = weight.options().requires_grad(false);
        node->V = V;
        node->D = D;
        node->padding = padding;
        node->scale = scale;
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---------------------------------------------------------------- norm and rotation of queries and keys
// t [T, H, D] with contiguous columns, and its strides (of a dimension of size one: the dense one)
struct Heads {
    Tensor t;
    int64_t ts = 0, hs = 0;
    explicit Heads(const Tensor& x) {
        if (!x.defined()) return;
        t = x.size(2) > 1 && x.stride(2) != 1 ? x.contiguous() : x;
        hs = t.size(1) > 1 ? t.stride(1) : t.size(2);
        ts = t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
    }
};

struct QKArgs {
    Tensor cos, sin, pos;
    bool norm = true, interleaved = false;
    double eps = 0;
    concord_qk_params params(const Tensor& like, int64_t heads, int64_t kv_heads) const {
        concord_qk_params p{};
        p.cos = ptr<const float>(cos);
        p.sin = ptr<const float>(sin);
        p.pos = ptr(pos);
        p.pos64 = pos.defined() && pos.scalar_type() == at::kLong;
        p.tokens = like.size(0);
        p.heads = heads;
        p.kv_heads = kv_heads;
        p.head_dim = like.size(2);
        p.rot = cos.defined() ? 2 * cos.size(1) : 0;
        p.positions = cos.defined() ? cos.size(0) : 0;
        p.type = type_code(like);
        p.norm = norm;
        p.interleaved = interleaved;
        p.eps = (float)eps;
        return p;
    }
};

struct QKNormRopeBackward : public torch::autograd::Node {
    SavedVariable q_, k_, qw_, kw_, cos_, sin_, pos_;
    bool norm = true, interleaved = false, has_k = false;
    double eps = 0;
    std::string name() const override { return "ConcordQKNormRopeBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&q_, &k_, &qw_, &kw_, &cos_, &sin_, &pos_}) v->reset_data();
    }
    variable_list apply(variable_list&& g) override {
        const Tensor q = q_.unpack(), k = k_.unpack(), qw = qw_.unpack(), kw = kw_.unpack();
        QKArgs A;
        A.cos = cos_.unpack();
        A.sin = sin_.unpack();
        A.pos = pos_.unpack();
        A.norm = norm;
        A.interleaved = interleaved;
        A.eps = eps;
        variable_list out(4);
        const bool has_q = g[0].defined(), with_k = has_k && g.size() > 1 && g[1].defined();
        if (!has_q && !with_k) return out;
        {
            at::NoGradGuard no_grad;
            const Tensor& like = has_q ? g[0] : g[1];
            c10::cuda::CUDAGuard guard(like.device());
            const Heads dq(has_q ? g[0] : Tensor()), dk(with_k ? g[1] : Tensor());
            const Heads xq(has_q ? q : Tensor()), xk(with_k ? k : Tensor());
            const auto plain = like.options().requires_grad(false);
            if (has_q) out[0] = at::empty(g[0].sizes(), plain);
            if (with_k) out[1] = at::empty(g[1].sizes(), plain);
            if (has_q && qw.defined() && task_should_compute_output(2)) out[2] = at::empty(qw.sizes(), qw.options().requires_grad(false));
            if (with_k && kw.defined() && task_should_compute_output(3)) out[3] = at::empty(kw.sizes(), kw.options().requires_grad(false));
            const auto p = A.params(like, has_q ? g[0].size(1) : 0, with_k ? g[1].size(1) : 0);
            Tensor ws;
            size_t bytes = 0;
            if (out[2].defined() || out[3].defined()) {
                bytes = concord_qk_norm_rope_bwd_workspace_bytes(&p);
                ws = bytes_like(like, bytes);
            }
            check(concord_qk_norm_rope_bwd(&p, ptr(xq.t), xq.ts, xq.hs, ptr(xk.t), xk.ts, xk.hs, ptr<const float>(qw),
                                           ptr<const float>(kw), ptr(dq.t), dq.ts, dq.hs, ptr(dk.t), dk.ts, dk.hs, ptr(out[0]),
                                           ptr(out[1]), ptr<float>(out[2]), ptr<float>(out[3]), ptr(ws), bytes,
                                           current_stream()),
                  "concord_qk_norm_rope_bwd");
        }
        return once(std::move(out), g);
    }
};

std::tuple<Tensor, MaybeTensor> qk_norm_rope(const Tensor& q, const MaybeTensor& k_in, const MaybeTensor& cos,
                                             const MaybeTensor& sin, const MaybeTensor& pos, const MaybeTensor& q_weight,
                                             const MaybeTensor& k_weight, bool norm, double eps, bool interleaved) {
    const Tensor k = get(k_in);
    refuse_transforms({q, k, get(q_weight), get(k_weight), get(cos), get(sin)}, "qk_norm_rope");
    // (converted where a gradient passes through; most weights and tables are fp32 already)
    auto floats = [](const MaybeTensor& m) {
        const Tensor t = get(m);
        return !t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous()) ? t : t.to(at::kFloat).contiguous();
    };
    c10::cuda::CUDAGuard guard(q.device());
    const Tensor qw = floats(q_weight), kw = floats(k_weight);
    QKArgs A;
    A.cos = floats(cos);
    A.sin = floats(sin);
    A.pos = pos.has_value() ? pos->contiguous() : Tensor();
    A.norm = norm;
    A.interleaved = interleaved;
    A.eps = eps;
    const bool grad = at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(qw) || wants_grad(kw));
    Tensor q_out, k_out;
    const Heads hq(q.detach()), hk(k.defined() ? k.detach() : k);
    {
        at::NoGradGuard no_grad;
        const auto plain = q.options().requires_grad(false);
        q_out = at::empty(q.sizes(), plain);
        if (k.defined()) k_out = at::empty(k.sizes(), plain);
        const auto p = A.params(q, q.size(1), k.defined() ? k.size(1) : 0);
        check(concord_qk_norm_rope_fwd(&p, ptr(hq.t), hq.ts, hq.hs, ptr(hk.t), hk.ts, hk.hs, ptr<const float>(qw),
                                       ptr<const float>(kw), ptr(q_out), ptr(k_out), current_stream()),
              "concord_qk_norm_rope_fwd");
    }
    if (grad) {
        auto node = link<QKNormRopeBackward>(q, k, qw, kw);
        if (norm) {                      // (the rotation's gradient does not read them)
            node->q_ = SavedVariable(hq.t, false);
            node->k_ = SavedVariable(hk.t, false);
            node->qw_ = SavedVariable(qw, false);
            node->kw_ = SavedVariable(kw, false);
        }
        node->cos_ = SavedVariable(A.cos, false);
        node->sin_ = SavedVariable(A.sin, false);
        node->pos_ = SavedVariable(A.pos, false);
        node->norm = norm;
        node->interleaved = interleaved;
        node->eps = eps;
        node->has_k = k.defined();
        torch::autograd::set_history(q_out, node);
        if (k.defined()) torch::autograd::set_history(k_out, node);
    }
    return {q_out, k_out.defined() ? MaybeTensor(k_out) : MaybeTensor()};
}

// ---------------------------------------------------------------- activations in 8 bits
Tensor save8(const Tensor& x) {
    refuse_transforms({x}, "save8");
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t K = x.size(-1);
    const Tensor x2 = rows(x, K);
    const Tensor out = bytes_like(x, concord_saved8_bytes(x2.size(0), K));
    check(concord_save8(ptr(x2), type_code(x2), ld(x2, K), ptr(out), x2.size(0), K, current_stream()), "concord_save8");
    return out;
}

// a Saved8's bytes are the caller's to make: whole ones, as many as its shape has
void check_saved(const Tensor& saved, int64_t M, int64_t K) {
    TORCH_CHECK(saved.scalar_type() == at::kByte && saved.is_cuda() && saved.is_contiguous() &&
                    saved.numel() == (int64_t)concord_saved8_bytes(M, K),
                "saved must hold ", concord_saved8_bytes(M, K), " bytes for ", M, " x ", K, " values, got ", saved.sizes(), " of ",
                saved.scalar_type());
}

Tensor dense8(const Tensor& saved, int64_t M, int64_t K, int64_t code) {
    at::NoGradGuard no_grad;
    check_saved(saved, M, K);
    c10::cuda::CUDAGuard guard(saved.device());
    const Tensor out = at::empty({M, K}, saved.options().dtype(type_of(code)));
    check(concord_dense8(ptr(saved), ptr(out), (int32_t)code, K, M, K, current_stream()), "concord_dense8");
    return out;
}

Tensor grad_weight8(const Tensor& dy0, const Tensor& saved, int64_t M, int64_t K) {
    refuse_transforms({dy0}, "grad_weight8");
    at::NoGradGuard no_grad;
    check_saved(saved, M, K);
    c10::cuda::CUDAGuard guard(saved.device());
    const int64_t N = dy0.size(-1);
    Tensor dy = rows(dy0, N);
    if (reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 || ld(dy, N) % 8) dy = at::empty(dy.sizes(), dy.options()).copy_(dy);
    const Tensor dw = at::empty({N, K}, dy.options().requires_grad(false));
    const size_t bytes = concord_gemm_dw8_workspace_bytes(M, N, K);
    const Tensor ws = bytes_like(dy, bytes);
    check(concord_gemm_dw8(ptr<const uint16_t>(dy), ld(dy, N), ptr(saved), ptr<uint16_t>(dw), M, N, K, ptr(ws), bytes,
                           current_stream()),
          "concord_gemm_dw8");
    return dw;
}

struct GatedBackward : public torch::autograd::Node {
    SavedVariable gate_, up_;            // [M, K], or their 8-bit form
    bool eight = false;
    int64_t act = 0, M = 0, K = 0;
    std::vector<int64_t> shape;
    std::string name() const override { return "ConcordGatedBackward"; }
    void release_variables() override { gate_.reset_data(); up_.reset_data(); }
    variable_list apply(variable_list&& g) override {
        const Tensor gate = gate_.unpack(), up = up_.unpack();
        variable_list out(2);
        if (!g[0].defined()) return out;
        {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(gate.device());
            const Tensor dh = rows(g[0], K);
            out[0] = at::empty(shape, dh.options().requires_grad(false));
            out[1] = at::empty(shape, dh.options().requires_grad(false));
            check(concord_gated_bwd(eight ? nullptr : ptr(gate), eight ? 0 : ld(gate, K), eight ? nullptr : ptr(up),
                                    eight ? 0 : ld(up, K), eight ? ptr(gate) : nullptr, eight ? ptr(up) : nullptr,
                                    type_code(dh), (int32_t)act, ptr(dh), ld(dh, K), ptr(out[0]), K, ptr(out[1]), K, M, K,
                                    current_stream()),
                  "concord_gated_bwd");
        }
        return once(std::move(out), g);
    }
};

std::tuple<Tensor, MaybeTensor> gated_unit(const Tensor& gate0, const Tensor& up0, int64_t act, bool keep8, bool out8) {
    refuse_transforms({gate0, up0}, "gated_unit");
    const bool grad = at::GradMode::is_enabled() && (wants_grad(gate0) || wants_grad(up0));
    c10::cuda::CUDAGuard guard(gate0.device());
    const int64_t K = gate0.size(-1);
    Tensor gate, up, h, g8, u8, h8;
    int64_t M;
    {
        at::NoGradGuard no_grad;
        gate = rows(gate0, K);
        up = rows(up0, K);
        M = gate.size(0);
        h = at::empty(gate0.sizes(), gate0.options().requires_grad(false));
        const size_t bytes = concord_saved8_bytes(M, K);
        if (grad && keep8) {
            g8 = bytes_like(gate, bytes);
            u8 = bytes_like(gate, bytes);
        }
        if (out8) h8 = bytes_like(gate, bytes);
        check(concord_gated_fwd(ptr(gate), ld(gate, K), ptr(up), ld(up, K), type_code(gate), (int32_t)act, ptr(h), ptr(g8),
                                ptr(u8), ptr(h8), M, K, current_stream()),
              "concord_gated_fwd");
    }
    if (grad) {
        auto node = link<GatedBackward>(gate0, up0);
        node->gate_ = SavedVariable(keep8 ? g8 : gate, false);
        node->up_ = SavedVariable(keep8 ? u8 : up, false);
        node->eight = keep8;
        node->act = act;
        node->M = M;
        node->K = K;
        node->shape = gate0.sizes().vec();
        torch::autograd::set_history(h, node);
    }
    return {h, h8.defined() ? MaybeTensor(h8) : MaybeTensor()};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "The training operators as autograd nodes over libconcord_b200.";
    using release = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("layer_norm", &layer_norm, release());
    m.def("distill_loss", &distill_loss, release());
    m.def("distill_loss_and_grad", &distill_loss_and_grad, release());
    m.def("attention", &attention, release());
    m.def("embedding", &embedding, release());
    m.def("qk_norm_rope", &qk_norm_rope, release());
    m.def("save8", &save8, release());
    m.def("dense8", &dense8, release());
    m.def("grad_weight8", &grad_weight8, release());
    m.def("gated_unit", &gated_unit, release());
}
