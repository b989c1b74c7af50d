// The trainable operators as native autograd nodes: topk_attention's modified and training form,
// qk_norm_rope, rope_to_heads and top_logit_distillation_loss.
//
// Python checks the arguments; allocation, the calls of the C ABI and the backward pass are here, so that the
// autograd engine's thread runs no Python: it runs on another core than the caller, and Python took twice its
// time there.  Host time of small calls, the same steps as Python functions and here: qk_norm_rope forward
// and backward 162 us, 97 (of which torch's own part of any such call is about 50); forward alone 25, 17.
// The distillation loss and its gradient 126, 78.
//
// Every gradient is that of the C entry points in ossa_b200.h; each node is differentiable once, and refuses to be
// differentiated twice where the second derivative is not zero.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <mutex>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>

#include "ossa_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Failure : std::runtime_error {
    int status;
    Failure(int s, const std::string& m) : std::runtime_error(m), status(s) {}
};

void check(int status) {
    if (status != OSSA_OK) throw Failure(status, ossa_last_error_string());
}

// A call on the tensor's device and that device's current stream.
struct On {
    c10::cuda::OptionalCUDAGuard guard;
    ossa_stream_t stream;
    explicit On(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

// A size as the C ABI takes it.
int i32(int64_t n) {
    TORCH_CHECK_VALUE(n <= INT32_MAX, "a size of ", n, " exceeds 32 bits");
    return (int)n;
}

const void* in(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* to(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
template <typename T>
const T* in_as(const Tensor& t) { return static_cast<const T*>(in(t)); }
float* to_f32(const Tensor& t) { return static_cast<float*>(to(t)); }

int dtype_code(const Tensor& t) { return t.scalar_type() == at::kFloat ? OSSA_F32 : OSSA_BF16; }
int is_64(const Tensor& t) { return t.scalar_type() == at::kLong ? 1 : 0; }
bool on_16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

// t contiguous and on a 16-byte boundary: itself, or a copy (a gradient may be a piece of a larger one).
Tensor packed(const Tensor& t) {
    if (!t.defined()) return t;
    Tensor c = t.contiguous();
    return on_16(c) ? c : c.clone();
}

// The saved tensors of a backward pass: hooks (checkpointing, offloading, compression) may bring them back in another
// place and layout, and the C ABI takes addresses.
variable_list saved(AutogradContext* ctx) {
    variable_list s = ctx->get_saved_variables();
    for (Tensor& t : s) t = packed(t);
    return s;
}

Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

// Operands that may be absent: an undefined tensor is no argument of a node's forward.
using Maybe = std::optional<Tensor>;
Tensor opt(const Maybe& t) { return t.has_value() ? *t : Tensor(); }

// What a backward pass returns when a graph of it is wanted: the gradients, which refuse to be differentiated
// where they depend on something that has a gradient: an incoming one, or (bent) the operator's own inputs.
variable_list once(variable_list grads, const variable_list& incoming, bool graph, bool bent) {
    bool any = bent;
    for (const Tensor& g : incoming) any = any || (g.defined() && g.requires_grad());
    if (!graph || !any) return grads;
    variable_list leaves;
    for (Tensor& g : grads) leaves.push_back(g.defined() ? g.detach().set_requires_grad(true) : Tensor());
    auto refuse = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice an operator that is differentiable once", (int64_t)leaves.size());
    at::AutoGradMode on(true);
    return (*refuse)(std::move(leaves));
}

// ------------------------------------------------------------------ head norms and rotation

// A tensor (B, N, heads * D) or (B, N, heads, D) as it is where each (b, n) row of its heads lies in one piece
// on a 16-byte boundary, else a contiguous copy; strides in elements.
struct Rows {
    Tensor x;
    int64_t H = 0, D = 0, sb = 0, sn = 0;
    Rows() = default;
    Rows(const Tensor& t, int64_t heads) : x(t), H(heads) {
        const int64_t B = t.size(0), N = t.size(1), es = (int64_t)t.element_size();
        D = t.dim() == 4 ? t.size(3) : t.size(2) / heads;
        bool whole = t.is_contiguous();
        if (!whole) {
            whole = t.stride(-1) == 1 && (t.dim() == 3 || heads == 1 || t.stride(2) == D);
            sb = B > 1 ? t.stride(0) : 0;
            sn = N > 1 ? t.stride(1) : 0;
        } else {
            sn = heads * D;
            sb = N * sn;
        }
        if (!whole || sb * es % 16 || sn * es % 16 || !on_16(t)) {
            x = packed(t);
            sn = heads * D;
            sb = N * sn;
        }
    }
};

int batched(const Tensor& cos, int64_t B) { return cos.defined() && B > 1 && cos.size(0) == B ? 1 : 0; }

// Gradients of the (B, Hx, N, D) outputs -> of the inputs; side k may be absent (k.H = 0).
void norm_rope_backward(const Rows& q, const Rows& k, const Tensor& wq, const Tensor& wk, const Tensor& cos,
                        const Tensor& sin, double eps, const Tensor& gq, const Tensor& gk, const Tensor& dq,
                        const Tensor& dk, const Tensor& dwq, const Tensor& dwk) {
    const int B = i32(gq.size(0)), N = i32(gq.size(2)), D = i32(gq.size(3));
    const Tensor& w = wq.defined() ? wq : wk;
    On on(gq);
    Tensor ws;
    size_t n = 0;
    if (w.defined()) ws = bytes(n = ossa_qk_norm_rope_bwd_workspace_size(D), gq);
    check(ossa_qk_norm_rope_bwd(
        in(q.x), in(k.x), in(wq), in(wk), in(cos), in(sin), batched(cos, B), dtype_code(gq),
        w.defined() ? dtype_code(w) : OSSA_F32, B, N, i32(q.H), i32(k.H), D, q.sb, q.sn, k.sb, k.sn, (float)eps, in(gq),
        in(gk), to(dq), to(dk), to(dwq), to(dwk), to(ws), n, on.stream));
}

struct QkNormRope : torch::autograd::Function<QkNormRope> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Maybe& wq_,
                                 const Maybe& wk_, const Maybe& cos_, const Maybe& sin_, int64_t Hq, int64_t Hk, double eps,
                                 bool grad) {
        const Rows a(q, Hq), b(k, Hk);
        const Tensor wq = opt(wq_), wk = opt(wk_), cos = packed(opt(cos_)), sin = packed(opt(sin_));
        const int64_t B = q.size(0), N = q.size(1);
        Tensor oq = at::empty({B, Hq, N, a.D}, q.options()), ok = at::empty({B, Hk, N, a.D}, q.options());
        if (B * N > 0) {
            const Tensor& w = wq.defined() ? wq : wk;
            On on(q);
            check(ossa_qk_norm_rope_fwd(in(a.x), in(b.x), in(wq), in(wk), in(cos), in(sin), batched(cos, B), dtype_code(q),
                                        w.defined() ? dtype_code(w) : OSSA_F32, i32(B), i32(N), i32(Hq), i32(Hk), i32(a.D),
                                        a.sb, a.sn, b.sb, b.sn, (float)eps, to(oq), to(ok), on.stream));
        }
        if (grad) {
            ctx->save_for_backward({q, k, wq, wk, cos, sin});
            ctx->saved_data["Hq"] = Hq;
            ctx->saved_data["Hk"] = Hk;
            ctx->saved_data["eps"] = eps;
            // without its weight a tensor is only rotated, and the output is linear in a weight alone
            ctx->saved_data["bent"] = (wq.defined() && q.requires_grad()) || (wk.defined() && k.requires_grad());
            ctx->set_materialize_grads(false);
        }
        return {oq, ok};
    }

    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const bool graph = at::GradMode::is_enabled();
        at::AutoGradMode off(false);
        variable_list out(10);
        if (!g[0].defined() && !g[1].defined()) return out;
        const variable_list s = ctx->get_saved_variables();  // q and k as rows, wherever they lie now
        const Tensor &q = s[0], &k = s[1], wq = packed(s[2]), wk = packed(s[3]), cos = packed(s[4]), sin = packed(s[5]), none;
        const Rows a(q, ctx->saved_data["Hq"].toInt()), b(k, ctx->saved_data["Hk"].toInt());
        const double eps = ctx->saved_data["eps"].toDouble();
        Tensor gq, gk;
        if (g[0].defined()) {
            gq = packed(g[0]);
            out[0] = at::empty(q.sizes(), q.options());
            if (wq.defined() && ctx->needs_input_grad(2)) out[2] = at::empty_like(wq);
        }
        if (g[1].defined()) {
            gk = packed(g[1]);
            out[1] = at::empty(k.sizes(), k.options());
            if (wk.defined() && ctx->needs_input_grad(wq.defined() ? 3 : 2)) out[3] = at::empty_like(wk);
        }
        if (!gk.defined())  // one output has no gradient: the other tensor alone, in the place of the queries
            norm_rope_backward(a, Rows(), wq, none, cos, sin, eps, gq, none, out[0], none, out[2], none);
        else if (!gq.defined())
            norm_rope_backward(b, Rows(), wk, none, cos, sin, eps, gk, none, out[1], none, out[3], none);
        else
            norm_rope_backward(a, b, wq, wk, cos, sin, eps, gq, gk, out[0], out[1], out[2], out[3]);
        return once(std::move(out), g, graph, ctx->saved_data["bent"].toBool());
    }
};

struct RopeToHeads : torch::autograd::Function<RopeToHeads> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& cos_, const Maybe& sin_, int64_t H) {
        const Tensor xc = packed(x), cos = packed(opt(cos_)), sin = packed(opt(sin_));
        const int64_t B = x.size(0), N = x.size(1), D = x.dim() == 4 ? x.size(3) : x.size(2) / H;
        Tensor out = at::empty({B, H, N, D}, x.options());
        if (out.numel() > 0) {
            On on(x);
            check(ossa_rope_to_heads(in(xc), in(cos), in(sin), batched(cos, B), dtype_code(x), i32(B), i32(N), i32(H), i32(D),
                                     to(out), on.stream));
        }
        ctx->save_for_backward({cos, sin});
        ctx->saved_data["shape"] = x.sizes();
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const bool graph = at::GradMode::is_enabled();
        at::AutoGradMode off(false);
        const variable_list s = saved(ctx);
        const Tensor gq = packed(g[0]), none;
        Tensor dx = at::empty(ctx->saved_data["shape"].toIntVector(), gq.options());
        Rows a;
        a.H = gq.size(1);
        norm_rope_backward(a, Rows(), none, none, s[0], s[1], 0.0, gq, none, dx, none, none, none);
        return once({dx, Tensor(), Tensor(), Tensor()}, g, graph, false);
    }
};

// ------------------------------------------------------------------ modified attention

#define OSSA_ATTENTION_ARGS(q, k, v, slopes, idx, segments, prefix, causal, q0, cap)                                       \
    in(q), in(k), in(v), in(idx), is_64(idx), dtype_code(q), i32(q.size(0)), i32(q.size(1)), i32(k.size(1)), i32(q.size(2)), \
        i32(k.size(2)), i32(q.size(3)), i32(idx.size(3)), (float)(1.0 / std::sqrt((double)q.size(3))), causal ? 1 : 0,       \
        i32(q0), (float)cap, in_as<float>(slopes), in_as<int32_t>(segments), in_as<int32_t>(prefix)

struct TopkAttention : torch::autograd::Function<TopkAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Maybe& slopes_,
                          const Tensor& idx_, const Maybe& segments_, const Maybe& prefix_, bool causal, int64_t q0,
                          double cap, bool grad) {
        const Tensor q = packed(q_), k = packed(k_), v = packed(v_), idx = idx_.contiguous();
        const Tensor slopes = opt(slopes_), segments = opt(segments_), prefix = opt(prefix_);
        Tensor out = at::empty(q.sizes(), q.options()), lse2, rest;
        if (grad) {
            lse2 = at::empty(q.sizes().slice(0, 3), q.options().dtype(at::kFloat));
            if (q.scalar_type() == at::kBFloat16) rest = at::empty(q.sizes(), q.options());
        }
        if (out.numel() > 0) {
            On on(q);
            check(ossa_topk_attention_mod_fwd(OSSA_ATTENTION_ARGS(q, k, v, slopes, idx, segments, prefix, causal, q0, cap),
                                              to(out), to_f32(lse2), to(rest), on.stream));
        }
        if (grad) {
            ctx->save_for_backward({q, k, v, slopes, idx, segments, prefix, out, lse2, rest});
            ctx->saved_data["causal"] = causal;
            ctx->saved_data["q0"] = q0;
            ctx->saved_data["cap"] = cap;
        }
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const bool graph = at::GradMode::is_enabled();
        at::AutoGradMode off(false);
        const variable_list s = saved(ctx);
        const Tensor &q = s[0], &k = s[1], &v = s[2], &slopes = s[3], &idx = s[4], &segments = s[5], &prefix = s[6];
        const bool causal = ctx->saved_data["causal"].toBool();
        const int64_t q0 = ctx->saved_data["q0"].toInt();
        const double cap = ctx->saved_data["cap"].toDouble();
        const Tensor dout = packed(g[0]);
        Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v), dslopes;
        if (slopes.defined() && ctx->needs_input_grad(3)) dslopes = at::empty_like(slopes);
        On on(q);
        const size_t n = ossa_topk_attention_bwd_workspace_size(
            dtype_code(q), i32(q.size(0)), i32(q.size(1)), i32(k.size(1)), i32(q.size(2)), i32(k.size(2)), i32(q.size(3)),
            i32(idx.size(3)), dslopes.defined() ? 1 : 0);
        const Tensor ws = bytes(n, q);
        check(ossa_topk_attention_bwd(OSSA_ATTENTION_ARGS(q, k, v, slopes, idx, segments, prefix, causal, q0, cap), in(s[7]),
                                      in_as<float>(s[8]), in(s[9]), in(dout), to(dq), to(dk), to(dv), to_f32(dslopes), to(ws), n,
                                      on.stream));
        variable_list out(11);
        out[0] = dq;
        out[1] = dk;
        out[2] = dv;
        out[3] = dslopes;
        return once(std::move(out), g, graph, true);
    }
};

// ------------------------------------------------------------------ top-logit distillation

// Logits (rows, V) or (outer, inner, V), rows where they lie.
struct Logits {
    Tensor z;
    int outer = 1, inner = 0, V = 0;
    long long so = 0, si = 0;
    explicit Logits(const Tensor& t) : z(t.stride(-1) == 1 ? t : t.contiguous()) {
        const int64_t d = z.dim();
        if (d == 3) {
            outer = i32(z.size(0));
            so = z.stride(0);
        }
        inner = i32(z.size(d - 2));
        si = z.stride(d - 2);
        V = i32(z.size(d - 1));
    }
    int64_t rows() const { return (int64_t)outer * inner; }
};

// Its own node: the gradient taken with the loss is held as a saved variable, so that hooks (checkpointing, offloading)
// and the graph's release reach it, and is given away by the first backward pass, which a list of saved variables cannot do.
struct TopLogitDistillBackward : torch::autograd::Node {
    torch::autograd::SavedVariable z, ids, ws, dz;
    bool waiting = false;  // dz is there for the first backward pass
    double tau = 1.0;
    int64_t reduction = 0;  // 0 none, 1 sum, 2 mean

    std::string name() const override { return "TopLogitDistillBackward"; }

    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto* v : {&z, &ids, &ws, &dz}) v->reset_data();
    }

    variable_list apply(variable_list&& g) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool graph = at::GradMode::is_enabled();
        at::AutoGradMode off(false);
        if (!g[0].defined()) return {Tensor()};
        const Logits l(z.unpack());  // rows, wherever they lie now
        const Tensor list = packed(ids.unpack()), work = packed(ws.unpack()), up = g[0].contiguous();  // fp32, as the loss
        const bool first = std::exchange(waiting, false);
        Tensor out;
        if (first) {
            out = packed(dz.unpack());
            dz.reset_data();
        } else {
            out = at::empty({l.rows(), l.V}, l.z.options());
        }
        {
            On on(l.z);
            check(ossa_top_logit_distill_bwd(in(l.z), dtype_code(l.z), l.outer, l.inner, l.V, l.so, l.si, in(list), is_64(list),
                                             i32(list.size(1)), (float)tau, reduction == 2 ? 1 : 0, in_as<float>(up),
                                             reduction == 0 ? 1 : 0, first ? 1 : 0, to(out), in(work), (size_t)work.numel(),
                                             on.stream));
        }
        return once({out.view(l.z.sizes())}, g, graph, true);
    }
};

Tensor top_logit_distill(const Tensor& z, const Tensor& teacher, const Tensor& ids, const Maybe& weight_, double tau,
                         int64_t reduction, bool grad) {
    TORCH_CHECK_NOT_IMPLEMENTED(!z._fw_grad(0).defined(), "top_logit_distillation_loss has no forward-mode derivative");
    const bool each = reduction == 0;
    Tensor loss, ws, dz;
    {
        at::AutoGradMode off(false);
        const Logits l(z);
        const Tensor weight = opt(weight_);
        const int K = i32(ids.size(1));
        const size_t n = ossa_top_logit_distill_workspace_size(l.rows(), K);
        ws = bytes(n, z);
        const auto f32 = z.options().dtype(at::kFloat);
        loss = each ? at::empty({l.rows()}, f32) : at::empty({}, f32);
        // a single incoming gradient is 1 as a rule: the gradient is taken with the loss
        if (grad && !each) dz = at::empty({l.rows(), l.V}, z.options());
        On on(z);
        check(ossa_top_logit_distill_fwd(in(l.z), dtype_code(z), l.outer, l.inner, l.V, l.so, l.si, in_as<float>(teacher),
                                         in(ids), is_64(ids), K, (float)tau, in_as<float>(weight), reduction == 2 ? 1 : 0,
                                         each ? to_f32(loss) : nullptr, each ? nullptr : to_f32(loss), to(dz), to(ws), n,
                                         on.stream));
        if (each && weight.defined()) loss.mul_(weight);
    }
    if (grad) {
        std::shared_ptr<TopLogitDistillBackward> node(new TopLogitDistillBackward, torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(z));
        node->z = torch::autograd::SavedVariable(z, false);
        node->ids = torch::autograd::SavedVariable(ids, false);
        node->ws = torch::autograd::SavedVariable(ws, false);
        node->waiting = dz.defined();
        if (dz.defined()) node->dz = torch::autograd::SavedVariable(dz, false);
        node->tau = tau;
        node->reduction = reduction;
        torch::autograd::set_history(loss, node);
    }
    return loss;
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
    using T = const Tensor&;
    using O = const Maybe&;
    using NoGil = py::call_guard<py::gil_scoped_release>;
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure& f) {
            const py::object type = py::module_::import("ossa_b200._lib").attr("OssaError");
            PyErr_SetObject(type.ptr(), type(f.status, f.what()).ptr());
        } catch (python_error& e) {  // raised by a hook on the saved tensors (checkpointing ends its second run so)
            e.restore();
        }
    });
    m.def("qk_norm_rope", [](T q, T k, O wq, O wk, O cos, O sin, int64_t Hq, int64_t Hk, double eps, bool grad) {
        variable_list o = QkNormRope::apply(q, k, wq, wk, cos, sin, Hq, Hk, eps, grad);
        return std::make_tuple(o[0], o[1]);
    }, NoGil());
    m.def("rope_to_heads", [](T x, O cos, O sin, int64_t H) { return RopeToHeads::apply(x, cos, sin, H); }, NoGil());
    m.def("topk_attention", [](T q, T k, T v, O slopes, T idx, O segments, O prefix, bool causal, int64_t q0, double cap,
                               bool grad) {
        return TopkAttention::apply(q, k, v, slopes, idx, segments, prefix, causal, q0, cap, grad);
    }, NoGil());
    m.def("top_logit_distill", &top_logit_distill, NoGil());
}
