// PyTorch side of the differentiable operators (block_ops.py): builds the C ABI's argument structures
// from tensors, allocates outputs and scratch, and records the call for autograd.
//
// These two operators are called several times per transformer block and, for single tokens, run for
// a few microseconds. The ctypes path of the other operators costs 30 us per call and a Python
// autograd.Function another 150 us per training step (its backward needs the interpreter on the engine's
// thread); here it is a function call and a C++ node. Arguments have been checked by block_ops.py.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/pa_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct PaFailure {
    int code;
    std::string msg;
};

// In a backward pass an exception crosses the autograd engine, which knows std::exception only.
[[noreturn]] void raise(int code, bool backward) {
    const std::string msg = pa_last_error();
    if (backward) throw std::runtime_error("libpa_b200 error " + std::to_string(code) + ": " + msg);
    throw PaFailure{code, msg};
}
void check(int rc, bool backward) {
    if (rc != PA_OK) raise(rc, backward);
}

// These operators have no forward-mode rule. A tensor with a tangent need not require a gradient, and a result computed
// below the autograd keys carries none, which PyTorch takes for zero: refused instead. (Not where forward mode is off, as in the
// forward of a function that has a rule of its own.)
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), what,
                                    ": forward-mode derivatives are not built (an input has a tangent)");
}

// x itself if the kernels can address it in place (unit stride on head_dim, 16-byte aligned base and strides,
// no broadcast dimensions), else a contiguous copy.
Tensor ready(const Tensor& x) {
    bool ok = x.stride(3) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
    for (int i = 0; ok && i < 3; ++i) ok = x.size(i) == 1 || (x.stride(i) > 0 && x.stride(i) % 8 == 0);
    return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}
Tensor aligned(const Tensor& x) {
    if (!x.defined() || (x.is_contiguous() && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0)) return x;
    return x.clone(at::MemoryFormat::Contiguous);
}
// [B, H, S, D] view of fresh [B, S, H, D] memory, the layout attention outputs have here.
Tensor bshd(const Tensor& like) {
    return at::empty({like.size(0), like.size(2), like.size(1), like.size(3)}, like.options()).transpose(1, 2);
}
// Element strides of (batch, head, row); dimensions of size 1 are never stepped over: 0.
void strides(const Tensor& x, int64_t* s) {
    for (int i = 0; i < 3; ++i) s[i] = x.size(i) > 1 ? x.stride(i) : 0;
}
int dtype_of(const Tensor& x) { return x.scalar_type() == at::kBFloat16 ? PA_BF16 : PA_F16; }
void* stream_of(const Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.device().index()).stream(); }

// ---- cross attention -----------------------------------------------------------------------------

// The device's status word and its pinned mirror, which these kernels write themselves when a wait gives up
// (block_ops.py passes their addresses; 0: none).
struct Status {
    int64_t word, host;
};

pa_xattn_args cross_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& rows, const Tensor& out,
                         const Tensor& lse, double scale) {
    pa_xattn_args a = {};
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.out = out.data_ptr();
    a.lse = lse.defined() ? lse.data_ptr<float>() : nullptr;
    a.batch = static_cast<int32_t>(q.size(0));
    a.heads = static_cast<int32_t>(q.size(1));
    a.seq_q = static_cast<int32_t>(q.size(2));
    a.head_dim = static_cast<int32_t>(q.size(3));
    a.kv_batch = static_cast<int32_t>(k.size(0));
    a.kv_heads = static_cast<int32_t>(k.size(1));
    a.seq_kv = static_cast<int32_t>(k.size(2));
    a.dtype = dtype_of(q);
    a.scale = static_cast<float>(scale);
    strides(q, a.q_stride);
    strides(k, a.k_stride);
    strides(v, a.v_stride);
    strides(out, a.o_stride);
    if (rows.defined()) {
        a.key_mask = static_cast<const uint8_t*>(rows.data_ptr());
        a.mask_stride = rows.size(0) > 1 ? rows.stride(0) : 0;
    }
    return a;
}

void launch_cross(pa_xattn_args& a, bool backward, const Tensor& q, Status st) {
    // a wait that ran out in an earlier launch is reported here
    if (st.host != 0) {
        const int code = *reinterpret_cast<volatile int32_t*>(st.host);
        if (code != 0) {
            const std::string msg = "an earlier launch gave up waiting (device status " + std::to_string(code) +
                                    "; the status word is sticky: call reset_device_status() once the cause is dealt with)";
            if (backward) throw std::runtime_error("libpa_b200 error " + std::to_string(PA_ETIMEDOUT) + ": " + msg);
            throw PaFailure{PA_ETIMEDOUT, msg};
        }
        a.status = reinterpret_cast<int32_t*>(st.word);
        a.status_host = reinterpret_cast<int32_t*>(st.host);
    }
    const int64_t n = pa_xattn_workspace_bytes(&a, backward ? 1 : 0);
    if (n < 0) raise(static_cast<int>(n), backward);
    Tensor ws;
    if (n > 0) {
        ws = at::empty({n}, q.options().dtype(at::kByte));
        a.workspace = ws.data_ptr();
        a.workspace_bytes = n;
    }
    void* stream = stream_of(q);
    check(backward ? pa_xattn_bwd(&a, stream) : pa_xattn_fwd(&a, stream), backward);
}

std::tuple<Tensor, Tensor> cross_forward(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& rows,
                                         double scale, bool need_lse, Status st) {
    c10::cuda::CUDAGuard guard(query.device());
    Tensor out = bshd(query), lse;
    if (need_lse) lse = at::empty({query.size(0), query.size(1), query.size(2)}, query.options().dtype(at::kFloat));
    if (out.numel() == 0) return {out, lse};
    if (key.size(2) == 0) {
        out.zero_();
        if (need_lse) lse.fill_(-std::numeric_limits<double>::infinity());
        return {out, lse};
    }
    const Tensor q = ready(query), k = ready(key), v = ready(value);
    pa_xattn_args a = cross_args(q, k, v, rows, out, lse, scale);
    launch_cross(a, false, q, st);
    return {out, lse};
}

// First derivatives only: differentiating the result once more raises. The node that raises hangs on everything the
// gradients are functions of (`sources`), not on the gradients alone: where only the way to one input is walked, a node off that
// way is not run, and PyTorch takes the derivative for zero.
variable_list once(variable_list grads, const variable_list& sources, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    std::vector<size_t> at_;
    variable_list defined;
    for (size_t i = 0; i < grads.size(); ++i)
        if (grads[i].defined()) {
            at_.push_back(i);
            defined.push_back(grads[i].requires_grad() ? grads[i] : grads[i].detach().requires_grad_(true));
        }
    if (defined.empty()) return grads;
    for (const Tensor& s : sources)
        if (s.defined() && s.requires_grad()) defined.push_back(s);
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " can be differentiated once only",
                                                                  static_cast<int64_t>(defined.size()));
    variable_list marked = (*error)(std::move(defined));
    for (size_t i = 0; i < at_.size(); ++i) grads[at_[i]] = marked[i];
    return grads;
}

struct CrossAttention : public torch::autograd::Function<CrossAttention> {
    static variable_list forward(AutogradContext* ctx, const Tensor& query, const Tensor& key, const Tensor& value,
                                 const std::optional<Tensor>& rows_, double scale, int64_t word, int64_t host) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor rows = rows_.value_or(Tensor());
        auto [out, lse] = cross_forward(query, key, value, rows, scale, true, Status{word, host});
        ctx->save_for_backward({query, key, value, rows, out, lse});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["word"] = word;
        ctx->saved_data["host"] = host;
        ctx->mark_non_differentiable({lse});
        ctx->set_materialize_grads(false);
        return {out, lse};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list result(7);
        const Tensor dout = grads[0];
        if (!dout.defined()) return result;
        refuse_tangents("the backward pass of cross_attention", {&dout});
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &query = saved[0], &key = saved[1], &value = saved[2], &rows = saved[3], &out = saved[4], &lse = saved[5];
        {
            at::AutoDispatchBelowADInplaceOrView below;
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(query.device());
            // two passes, one for dq and one for dk and dv: each only if something is asked of it
            const bool queries = ctx->needs_input_grad(0), keys = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
            Tensor dq, dk, dv;
            if (queries) dq = bshd(query);
            if (keys) dk = bshd(key), dv = bshd(value);
            if (query.numel() == 0 || key.numel() == 0) {
                for (Tensor* t : {&dq, &dk, &dv})
                    if (t->defined()) t->zero_();
            } else if (queries || keys) {
                // (out may have been saved elsewhere meanwhile and come back with other strides)
                const Tensor q = ready(query), k = ready(key), v = ready(value), g = ready(dout), o = ready(out);
                pa_xattn_args a = cross_args(q, k, v, rows, o, lse, ctx->saved_data["scale"].toDouble());
                a.dout = g.data_ptr();
                strides(g, a.do_stride);
                if (queries) {
                    a.dq = dq.data_ptr();
                    strides(dq, a.dq_stride);
                }
                if (keys) {
                    a.dk = dk.data_ptr();
                    a.dv = dv.data_ptr();
                    strides(dk, a.dk_stride);
                    strides(dv, a.dv_stride);
                }
                launch_cross(a, true, q, Status{ctx->saved_data["word"].toInt(), ctx->saved_data["host"].toInt()});
            }
            result[0] = dq;
            result[1] = dk;
            result[2] = dv;  // (what was not asked for is undefined, or dropped by the engine)
        }
        return once(std::move(result), {dout, query, key, value}, "cross_attention");
    }
};

std::tuple<Tensor, std::optional<Tensor>> cross_attention(const Tensor& query, const Tensor& key, const Tensor& value,
                                                          const std::optional<Tensor>& rows_, double scale, bool need_lse,
                                                          int64_t word, int64_t host) {
    refuse_tangents("cross_attention", {&query, &key, &value});
    if (at::GradMode::is_enabled() && (query.requires_grad() || key.requires_grad() || value.requires_grad())) {
        auto r = CrossAttention::apply(query, key, value, rows_, scale, word, host);
        return {r[0], need_lse ? std::optional<Tensor>(r[1]) : std::nullopt};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor k = key, v = value;
    // an expanded batch is read once
    if (query.size(0) > 1 && key.size(0) == query.size(0) && key.stride(0) == 0 && value.stride(0) == 0) {
        k = key.narrow(0, 0, 1);
        v = value.narrow(0, 0, 1);
    }
    auto [out, lse] = cross_forward(query, k, v, rows_.value_or(Tensor()), scale, need_lse, Status{word, host});
    return {out, need_lse ? std::optional<Tensor>(lse) : std::nullopt};
}

// ---- norm and rotation of queries and keys ----------------------------------------------------------

struct NormPlan {
    int64_t row_offset;
    bool interleaved;
    double eps;
};

pa_qk_norm_args norm_args(const variable_list& xs, const variable_list& ys, const variable_list& ws, const Tensor& cos,
                          const Tensor& sin, const NormPlan& plan) {
    pa_qk_norm_args a = {};
    a.batch = static_cast<int32_t>(xs[0].size(0));
    a.rows = static_cast<int32_t>(xs[0].size(2));
    a.head_dim = static_cast<int32_t>(xs[0].size(3));
    a.dtype = dtype_of(xs[0]);
    a.interleaved = plan.interleaved ? 1 : 0;
    a.eps = static_cast<float>(plan.eps);
    for (size_t i = 0; i < xs.size(); ++i) {
        a.x[i] = xs[i].data_ptr();
        a.y[i] = ys[i].data_ptr();
        a.heads[i] = static_cast<int32_t>(xs[i].size(1));
        if (ws[i].defined()) a.weight[i] = ws[i].data_ptr();
        int64_t s[3];
        strides(xs[i], s);
        a.x_stride[i][0] = s[0], a.x_stride[i][1] = s[2], a.x_stride[i][2] = s[1];
        strides(ys[i], s);
        a.y_stride[i][0] = s[0], a.y_stride[i][1] = s[2], a.y_stride[i][2] = s[1];
    }
    if (cos.defined()) {
        a.cos = cos.data_ptr<float>();
        a.sin = sin.data_ptr<float>();
        a.table_row0 = plan.row_offset;
    }
    return a;
}

variable_list norm_forward(const variable_list& xs_, const variable_list& ws_, const Tensor& cos, const Tensor& sin,
                           const NormPlan& plan) {
    c10::cuda::CUDAGuard guard(xs_[0].device());
    variable_list xs, ys, ws, all;
    for (size_t i = 0; i < xs_.size(); ++i) {
        all.push_back(bshd(xs_[i]));
        if (xs_[i].numel() == 0) continue;
        ys.push_back(all.back());
        xs.push_back(ready(xs_[i]));
        ws.push_back(aligned(ws_[i]));
    }
    if (xs.empty()) return all;
    const Tensor c = aligned(cos), s = aligned(sin);
    pa_qk_norm_args a = norm_args(xs, ys, ws, c, s, plan);
    check(pa_qk_norm_fwd(&a, stream_of(xs[0])), false);
    return all;
}

struct QkNorm : public torch::autograd::Function<QkNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k_,
                                 const std::optional<Tensor>& wq_, const std::optional<Tensor>& wk_, const std::optional<Tensor>& cos_,
                                 const std::optional<Tensor>& sin_, int64_t row_offset, bool interleaved, double eps) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor k = k_.value_or(Tensor()), wq = wq_.value_or(Tensor()), wk = wk_.value_or(Tensor());
        const Tensor cos = cos_.value_or(Tensor()), sin = sin_.value_or(Tensor());
        variable_list xs{q}, ws{wq};
        if (k.defined()) {
            xs.push_back(k);
            ws.push_back(wk);
        }
        variable_list ys = norm_forward(xs, ws, cos, sin, NormPlan{row_offset, interleaved, eps});
        ctx->save_for_backward({q, k, wq, wk, cos, sin});
        ctx->saved_data["row_offset"] = row_offset;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        return ys;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list result(9);
        for (const Tensor& g : grads) refuse_tangents("the backward pass of qk_norm_rotary", {&g});
        const variable_list saved = ctx->get_saved_variables();
        const NormPlan plan{ctx->saved_data["row_offset"].toInt(), ctx->saved_data["interleaved"].toBool(),
                            ctx->saved_data["eps"].toDouble()};
        {
            at::AutoDispatchBelowADInplaceOrView below;
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(saved[0].device());
            // (the node has an edge for each tensor that was given)
            bool asked[4] = {};
            for (int i = 0, edge = 0; i < 4; ++i)
                if (saved[i].defined()) asked[i] = ctx->needs_input_grad(edge++);
            // the tensors something is asked of, and which they are
            variable_list xs, dxs, dys, ws, dws;
            std::vector<int> which;
            for (int i = 0; i < 2; ++i) {
                const Tensor& x = saved[i];
                if (!x.defined() || !(asked[i] || asked[i + 2])) continue;
                const bool weighted = saved[i + 2].defined() && asked[i + 2];
                const Tensor dy = static_cast<size_t>(i) < grads.size() ? grads[i] : Tensor();
                if (!dy.defined() || x.numel() == 0) {  // an output nothing depends on, or without elements
                    if (asked[i]) result[i] = at::zeros_like(x);
                    if (weighted) result[i + 2] = at::zeros_like(saved[i + 2]);
                    continue;
                }
                which.push_back(i);
                xs.push_back(ready(x));
                dys.push_back(ready(dy));
                dxs.push_back(bshd(x));
                ws.push_back(aligned(saved[i + 2]));
                dws.push_back(weighted ? at::empty(saved[i + 2].sizes(), saved[i + 2].options()) : Tensor());
            }
            if (!xs.empty()) {
                bool any_weight = false;
                for (const Tensor& w : dws) any_weight = any_weight || w.defined();
                const Tensor cos = aligned(saved[4]), sin = aligned(saved[5]);
                pa_qk_norm_args a = norm_args(xs, dxs, ws, cos, sin, plan);
                for (size_t i = 0; i < xs.size(); ++i) {
                    a.dy[i] = dys[i].data_ptr();
                    int64_t s[3];
                    strides(dys[i], s);
                    a.dy_stride[i][0] = s[0], a.dy_stride[i][1] = s[2], a.dy_stride[i][2] = s[1];
                    if (dws[i].defined()) a.dweight[i] = dws[i].data_ptr();
                }
                Tensor scratch;
                if (any_weight) {
                    scratch = at::empty({pa_qk_norm_workspace_bytes()}, xs[0].options().dtype(at::kByte));
                    a.workspace = scratch.data_ptr();
                    a.workspace_bytes = scratch.numel();
                }
                check(pa_qk_norm_bwd(&a, stream_of(xs[0])), true);
                for (size_t i = 0; i < which.size(); ++i) {
                    if (asked[which[i]]) result[which[i]] = dxs[i];
                    if (dws[i].defined()) result[which[i] + 2] = dws[i];
                }
            }
        }
        variable_list sources(saved.begin(), saved.begin() + 4);
        sources.insert(sources.end(), grads.begin(), grads.end());
        return once(std::move(result), sources, "qk_norm_rotary");
    }
};

std::tuple<Tensor, std::optional<Tensor>> qk_norm_rotary(const Tensor& q, const std::optional<Tensor>& k_,
                                                         const std::optional<Tensor>& wq_, const std::optional<Tensor>& wk_,
                                                         const std::optional<Tensor>& cos_, const std::optional<Tensor>& sin_,
                                                         int64_t row_offset, bool interleaved, double eps) {
    const Tensor k = k_.value_or(Tensor()), wq = wq_.value_or(Tensor()), wk = wk_.value_or(Tensor());
    const Tensor cos = cos_.value_or(Tensor()), sin = sin_.value_or(Tensor());
    refuse_tangents("qk_norm_rotary", {&q, &k, &wq, &wk, &cos, &sin});
    auto asks = [](const std::optional<Tensor>& t) { return t.has_value() && t->requires_grad(); };
    variable_list ys;
    if (at::GradMode::is_enabled() && (q.requires_grad() || asks(k_) || asks(wq_) || asks(wk_))) {
        ys = QkNorm::apply(q, k_, wq_, wk_, cos_, sin_, row_offset, interleaved, eps);
    } else {
        at::AutoDispatchBelowADInplaceOrView below;
        variable_list xs{q}, ws{wq};
        if (k.defined()) {
            xs.push_back(k);
            ws.push_back(wk);
        }
        ys = norm_forward(xs, ws, cos, sin, NormPlan{row_offset, interleaved, eps});
    }
    return {ys[0], ys.size() > 1 ? std::optional<Tensor>(ys[1]) : std::nullopt};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("cross_attention", &cross_attention);
    m.def("qk_norm_rotary", &qk_norm_rotary);
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const PaFailure& f) {
            const py::object cls = py::module_::import("paraattention_b200._lib").attr("PaError");
            const py::object err = cls(f.code, f.msg);
            PyErr_SetObject(cls.ptr(), err.ptr());
        }
    });
}
