// The torch side of the row norm and the 8-bit product: output tensors, autograd and the calls of sgv_rms_norm, sgv_rms_norm_backward, sgv_dequantize_rows and
// sgv_int8_gemm (include/sgv_ops.h) on the current stream of the tensors' device.
//
// In C++ because at a token or a small batch these operators take less time on the GPU than Python takes to call them: per call of host time, [32, 512] fp32 norm 11.3 -> 6 us
// under autograd, forward and backward 75 -> 43 us (of which 30 are the hand-over to the autograd engine's device thread and back, where a Python backward also starts cold).
//
// Arguments are checked here with one predicate for each operator; `Refused` sends the caller (ops/rms_norm.py, ops/int8.py) to the check that words the reason, `Watched` to
// the formula in torch operations, or to a refusal where the operator has no gradient.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/sgv_ops.h"

#include <limits>
#include <stdexcept>
#include <tuple>

namespace {

using at::Tensor;
using std::optional;

struct Refused : std::runtime_error { using std::runtime_error::runtime_error; };
struct Watched : Refused { using Refused::Refused; };

// the C entry points, as addresses in the loaded libsgv_hip.so
struct {
    decltype(&sgv_rms_norm) rms_norm;
    decltype(&sgv_rms_norm_backward) rms_norm_backward;
    decltype(&sgv_rms_norm_backward_workspace_bytes) workspace_bytes;
    decltype(&sgv_dequantize_rows) dequantize_rows;
    decltype(&sgv_int8_gemm) int8_gemm;
    decltype(&sgv_last_error) last_error;
} lib;

void bind(const std::vector<int64_t>& entries) {
    if (entries.size() != 6) throw std::runtime_error("six entry points");
    lib.rms_norm = (decltype(lib.rms_norm))entries[0];
    lib.rms_norm_backward = (decltype(lib.rms_norm_backward))entries[1];
    lib.workspace_bytes = (decltype(lib.workspace_bytes))entries[2];
    lib.dequantize_rows = (decltype(lib.dequantize_rows))entries[3];
    lib.int8_gemm = (decltype(lib.int8_gemm))entries[4];
    lib.last_error = (decltype(lib.last_error))entries[5];
}

void check(int rc) {
    if (rc != SGV_OK) throw std::runtime_error(lib.last_error());
}
void require(bool ok, const char* what) {
    if (!ok) throw Refused(what);
}

// Whether something follows this tensor that sees torch's operations and no launch: a derivative of forward mode by the tangent it has (a launch's output would come without
// one, and without an error), a function transform or a subclass, whose tensors have no memory of their own; or whether torch records a graph of its operations, which would
// hold the outputs' allocation and not what fills them (torch.jit.trace, make_fx).
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool without_memory(const Tensor& t) {
    using Key = c10::DispatchKey;
    return t.defined() && t.key_set().has_any(c10::DispatchKeySet({Key::Batched, Key::FuncTorchBatched, Key::FuncTorchGradWrapper, Key::Functionalize, Key::Python, Key::ZeroTensor}));
}
bool has_tangent(const optional<Tensor>& t) { return t && has_tangent(*t); }
bool without_memory(const optional<Tensor>& t) { return t && without_memory(*t); }
bool recorded() {
    return torch::jit::tracer::isTracing() ||
           (c10::impl::TorchDispatchModeTLS::any_modes_set() && c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
}
template <typename... Ts> void unwatched(const Ts&... ts) {
    if (recorded()) throw Watched("launches a kernel, which a trace does not record: trace the function without it, or the layer before quantize_int8_()");
    if ((has_tangent(ts) || ...)) throw Watched("serves inference and has no gradient, of forward mode neither: call it with detached tensors");
    if ((without_memory(ts) || ...)) throw Watched("takes tensors in memory: it has no form under a function transform (vmap, grad, jvp) or for a tensor subclass");
}
template <typename... Ts> bool watched(const Ts&... ts) { return recorded() || ((has_tangent(ts) || without_memory(ts)) || ...); }

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int type_code(at::ScalarType t) {
    return t == at::kFloat ? SGV_F32 : t == at::kHalf ? SGV_F16 : t == at::kBFloat16 ? SGV_BF16 : -1;
}
at::ScalarType code_type(int64_t code) {
    require(code == SGV_F32 || code == SGV_F16 || code == SGV_BF16, "unsupported dtype");
    return code == SGV_F32 ? at::kFloat : code == SGV_F16 ? at::kHalf : at::kBFloat16;
}

// t as [rows, columns] with unit stride along a row: a view where t allows one, else a copy.  (A negated view, whose memory holds the values with the other sign, is copied:
// so are dense_or_none's and the gradients that arrive.)
Tensor row_view(const Tensor& t) {
    if (t.is_neg()) return row_view(t.resolve_neg());
    const int64_t cols = t.size(-1);
    if (t.is_contiguous()) return t.dim() == 2 ? t : t.view({-1, cols});
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, cols});
    return cols > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}
Tensor dense_or_none(const Tensor& t) {
    if (!t.defined() || (t.is_contiguous() && !t.is_neg())) return t;
    return t.resolve_neg().contiguous();
}
Tensor dense_or_none(const optional<Tensor>& t) { return t ? dense_or_none(*t) : Tensor(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
int64_t stride(const Tensor& t) { return t.defined() ? t.stride(0) : 0; }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const optional<Tensor>& t) { return t && t->requires_grad(); }

bool rows_fit(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& residual, double eps) {
    if (!x.is_cuda() || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > std::numeric_limits<int32_t>::max() || type_code(x.scalar_type()) < 0 || !(eps >= 0)) return false;
    if (weight && (weight->dim() != 1 || weight->size(0) != x.size(-1) || (weight->scalar_type() != x.scalar_type() && weight->scalar_type() != at::kFloat) ||
                   weight->device() != x.device())) return false;
    return !residual || (residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() && residual->device() == x.device());
}
bool scaled_rows_fit(const Tensor& q, const Tensor& scale) {
    return q.is_cuda() && q.scalar_type() == at::kChar && q.dim() >= 1 && q.size(-1) >= 1 && scale.scalar_type() == at::kFloat && scale.sizes() == q.sizes().slice(0, q.dim() - 1) &&
           scale.device() == q.device();
}

struct Forward { Tensor y, h, inv, scale; };
// y (or q with its scale), h, 1 / rms of rows; x and residual are row_views, the weight is dense
Forward launch_forward(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, bool int8, bool normalize, bool want_inv) {
    const int64_t rows = x.size(0), cols = x.size(1), pitch = int8 ? (cols + 15) / 16 * 16 : cols;
    Forward out;
    if (residual.defined()) out.h = at::empty({rows, cols}, x.options());
    if (want_inv) out.inv = at::empty({rows}, x.options().dtype(at::kFloat));
    out.y = at::empty({rows, pitch}, int8 ? x.options().dtype(at::kChar) : x.options());       // 8 bits: rows on 16 bytes, zeros behind the last column
    if (int8) out.scale = at::empty({rows}, x.options().dtype(at::kFloat));
    if (rows) {
        sgv_rms_norm_params p{};
        p.x = ptr(x); p.residual = ptr(residual); p.weight = ptr(weight); p.h = out_ptr(out.h); p.inv_rms = (float*)out_ptr(out.inv);
        (int8 ? p.q : p.y) = out_ptr(out.y);
        p.q_scale = (float*)out_ptr(out.scale);
        p.rows = rows; p.x_stride = stride(x); p.residual_stride = stride(residual); p.q_stride = pitch; p.cols = (int32_t)cols;
        p.weight_f32 = weight.defined() && weight.scalar_type() == at::kFloat; p.normalize = normalize; p.eps = (float)eps;
        const c10::DeviceGuard guard(x.device());
        check(lib.rms_norm(&p, type_code(x.scalar_type()), stream_of(x)));
    }
    if (pitch != cols) out.y = out.y.narrow(1, 0, cols);
    return out;
}

// (dx, dweight) in torch operations: what the kernel computes, differentiable once more.  The norm is fp64, as the kernel's is where squares leave fp32's range; the
// normalised row, of sqrt(columns) at most, is fp32 again.
std::tuple<Tensor, Tensor> gradient_formula(const Tensor& dy, const Tensor& h, const Tensor& dh, const Tensor& weight, double eps) {
    Tensor dx, dw;
    if (dy.defined()) {
        const Tensor hd = h.to(at::kDouble), inv = (hd.square().mean(-1, true) + eps).rsqrt(), xh = (hd * inv).to(at::kFloat);
        Tensor g = dy.to(at::kFloat);
        if (weight.defined()) {
            dw = (g * xh).sum(0).to(weight.scalar_type());
            g = g * weight.to(at::kFloat);
        }
        dx = inv * (g - xh * (g * xh).mean(-1, true));
    }
    if (dh.defined()) dx = dx.defined() ? dx + dh.to(at::kFloat) : dh.to(at::kFloat);
    return {dx.to(h.scalar_type()), dw};
}

// rows in, rows out: y, or (y, h) with a residual
struct RmsNorm : torch::autograd::Function<RmsNorm> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight_, const optional<Tensor>& residual_, double eps) {
        const at::AutoDispatchBelowADInplaceOrView below;
        const Tensor weight = weight_ ? *weight_ : Tensor(), residual = residual_ ? *residual_ : Tensor();
        const Forward out = launch_forward(x, dense_or_none(weight), residual, eps, false, true, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({residual.defined() ? out.h : x, weight, out.inv});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["needs"] = (int64_t)(wants_grad(x) | wants_grad(weight) << 1 | wants_grad(residual) << 2);
        if (residual.defined()) return {out.y, out.h};
        return {out.y};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &weight = saved[1], &inv = saved[2];
        const int64_t needs = ctx->saved_data["needs"].toInt();
        const bool need_x = needs & 1, need_r = needs & 4;
        Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor(), dx, dw;
        const bool need_w = (needs & 2) && dy.defined();
        if (!dy.defined() && !dh.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        if (at::GradMode::is_enabled() || watched(dy, dh, h, weight)) {
            std::tie(dx, dw) = gradient_formula(dy, h, dh, weight, ctx->saved_data["eps"].toDouble());
        } else if (!dy.defined()) {
            dx = dh;
        } else {
            const int64_t rows = h.size(0), cols = h.size(1);
            if (dy.is_neg()) dy = dy.resolve_neg();
            if (dh.defined() && dh.is_neg()) dh = dh.resolve_neg();
            if (cols > 1 && dy.stride(1) != 1) dy = dy.contiguous();
            if (cols > 1 && dh.defined() && dh.stride(1) != 1) dh = dh.contiguous();
            const Tensor w = dense_or_none(weight);
            if (need_x || need_r) dx = at::empty({rows, cols}, h.options());
            if (need_w) dw = at::empty({cols}, w.options());
            if (rows) {
                const int type = type_code(h.scalar_type());
                sgv_rms_norm_backward_params p{};
                Tensor work;
                if (need_w) {
                    p.workspace_bytes = lib.workspace_bytes(rows, (int32_t)cols, type);
                    work = at::empty({p.workspace_bytes / 4}, inv.options());
                    p.workspace = out_ptr(work);
                }
                p.dy = ptr(dy); p.h = ptr(h); p.dh = ptr(dh); p.weight = ptr(w); p.inv_rms = (const float*)ptr(inv); p.dx = out_ptr(dx); p.dweight = out_ptr(dw);
                p.rows = rows; p.dy_stride = stride(dy); p.h_stride = stride(h); p.dh_stride = stride(dh); p.cols = (int32_t)cols;
                p.weight_f32 = w.defined() && w.scalar_type() == at::kFloat;
                const c10::DeviceGuard guard(h.device());
                check(lib.rms_norm_backward(&p, type, stream_of(h)));
            } else if (need_w) {
                dw.zero_();
            }
        }
        return {need_x ? dx : Tensor(), need_w ? dw : Tensor(), need_r ? dx : Tensor(), Tensor()};
    }
};

std::tuple<Tensor, optional<Tensor>> rms_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& residual, double eps) {
    unwatched(x, weight, residual);
    require(rows_fit(x, weight, residual, eps), "rms_norm: arguments");
    const Tensor rows = row_view(x);
    const optional<Tensor> res = residual ? optional<Tensor>(row_view(*residual)) : optional<Tensor>();
    Tensor y, h;
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(residual))) {
        const auto out = RmsNorm::apply(rows, weight, res, eps);
        y = out[0];
        if (residual) h = out[1];
    } else {
        const Forward out = launch_forward(rows, dense_or_none(weight), res ? *res : Tensor(), eps, false, true, false);
        y = out.y;
        h = out.h;
    }
    if (x.dim() != 2) {
        y = y.view(x.sizes());
        if (residual) h = h.view(x.sizes());
    }
    return {y, residual ? optional<Tensor>(h) : optional<Tensor>()};
}

std::tuple<Tensor, Tensor, optional<Tensor>> rms_norm_int8(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& residual, double eps, bool normalize) {
    unwatched(x, weight, residual);
    require(rows_fit(x, weight, residual, eps) && !(at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(residual))), "rms_norm_int8: arguments");
    Forward out = launch_forward(row_view(x), dense_or_none(weight), residual ? row_view(*residual) : Tensor(), eps, true, normalize, false);
    if (x.dim() != 2) {
        const auto lead = x.sizes().slice(0, x.dim() - 1);
        out.y = lead.empty() ? out.y.select(0, 0) : out.y.unflatten(0, lead);
        out.scale = out.scale.view(lead);
        if (residual) out.h = out.h.view(x.sizes());
    }
    return {out.y, out.scale, residual ? optional<Tensor>(out.h) : optional<Tensor>()};
}

Tensor dequantize_rows(const Tensor& q, const Tensor& scale, int64_t code) {
    unwatched(q, scale);
    require(scaled_rows_fit(q, scale) && q.size(-1) <= std::numeric_limits<int32_t>::max() && !(at::GradMode::is_enabled() && scale.requires_grad()), "dequantize_rows: arguments");
    const Tensor out = at::empty(q.sizes(), q.options().dtype(code_type(code)).memory_format(at::MemoryFormat::Contiguous)), rows = row_view(q), s = dense_or_none(scale);
    if (rows.size(0)) {
        const c10::DeviceGuard guard(q.device());
        check(lib.dequantize_rows(ptr(rows), rows.stride(0), (const float*)ptr(s), out_ptr(out), rows.size(0), (int32_t)rows.size(1), (int)code, stream_of(q)));
    }
    return out;
}

// The rows of q starting on 16 bytes and readable up to the next multiple of 16 columns -- q itself where it is so (what the quantisers return, and any dense
// K % 16 == 0 tensor), else a copy -- and their distance in bytes
std::tuple<Tensor, int64_t> product_rows(const Tensor& t) {
    constexpr int64_t MAX_STRIDE = 1 << 23;          // between two rows that the product takes as they are
    const Tensor q = row_view(t);
    const int64_t rows = q.size(0), cols = q.size(1), pitch = (cols + 15) / 16 * 16, step = rows > 1 ? q.stride(0) : pitch;
    if (step % 16 == 0 && step < MAX_STRIDE && (uintptr_t)ptr(q) % 16 == 0 && (cols == pitch || q.storage_offset() + (rows - 1) * step + pitch <= (int64_t)q.storage().nbytes())) return {q, step};
    Tensor copy = at::empty({rows, pitch}, q.options());
    copy.narrow(1, 0, cols).copy_(q);                // (what lies behind the last column is ignored)
    return {copy, pitch};
}

struct Epilogue { const optional<Tensor>& bias; int act; double alpha, gain; };

bool layer_fits(int64_t cols, c10::Device device, const Tensor& b, const Tensor& b_scale, const Epilogue& e) {
    return scaled_rows_fit(b, b_scale) && b.dim() == 2 && b.size(1) == cols && b.device() == device && cols <= 131071 &&
           (!e.bias || (e.bias->dim() == 1 && e.bias->size(0) == b.size(0) && e.bias->scalar_type() == at::kFloat && e.bias->device() == device)) &&
           !(at::GradMode::is_enabled() && (b_scale.requires_grad() || wants_grad(e.bias)));
}

// out = the product of m rows of a (lda bytes apart, dense scales) with the rows of b
void launch_product(const Tensor& a, int64_t m, int64_t lda, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, const Epilogue& e, const Tensor& out) {
    const auto [br, ldb] = product_rows(b);
    const Tensor sb = dense_or_none(b_scale), bias = dense_or_none(e.bias);
    require(m <= std::numeric_limits<int32_t>::max() && b.size(0) <= std::numeric_limits<int32_t>::max(), "int8 product: too many rows");
    sgv_int8_gemm_params p{};
    p.a = ptr(a); p.b = ptr(br); p.a_scale = (const float*)ptr(a_scale); p.b_scale = (const float*)ptr(sb); p.bias = (const float*)ptr(bias); p.c = out_ptr(out);
    p.lda = lda; p.ldb = ldb; p.ldc = b.size(0); p.m = (int32_t)m; p.n = (int32_t)b.size(0); p.k = (int32_t)b.size(1);
    p.act = e.act; p.alpha = (float)e.alpha; p.gain = (float)e.gain;
    const c10::DeviceGuard guard(out.device());
    check(lib.int8_gemm(&p, type_code(out.scalar_type()), stream_of(out)));
}

at::DimVector layer_shape(const Tensor& x, const Tensor& b) {
    at::DimVector size(x.sizes().begin(), x.sizes().end());
    size.back() = b.size(0);
    return size;
}

Tensor matmul(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, const optional<Tensor>& bias, int act, double alpha, double gain, int64_t code) {
    const Epilogue e{bias, act, alpha, gain};
    unwatched(a, a_scale, b, b_scale, bias);
    require(scaled_rows_fit(a, a_scale) && layer_fits(a.size(-1), a.device(), b, b_scale, e) && !(at::GradMode::is_enabled() && a_scale.requires_grad()), "matmul: arguments");
    const Tensor out = at::empty(layer_shape(a, b), a.options().dtype(code_type(code)));
    if (out.numel()) {
        const auto [rows, lda] = product_rows(a);
        launch_product(rows, rows.size(0), lda, dense_or_none(a_scale), b, b_scale, e, out);
    }
    return out;
}

Tensor dense(const Tensor& x, const Tensor& b, const Tensor& b_scale, const optional<Tensor>& bias, int act, double alpha, double gain, bool normalize, double eps) {
    const Epilogue e{bias, act, alpha, gain};
    unwatched(x, b, b_scale, bias);
    require(rows_fit(x, {}, {}, eps) && layer_fits(x.size(-1), x.device(), b, b_scale, e) && !(at::GradMode::is_enabled() && x.requires_grad()), "dense: arguments");
    const Tensor out = at::empty(layer_shape(x, b), x.options());
    if (out.numel()) {
        const Forward q = launch_forward(row_view(x), Tensor(), Tensor(), eps, true, normalize, false);
        launch_product(q.y, q.y.size(0), q.y.stride(0), q.scale, b, b_scale, e, out);
    }
    return out;
}

}  // namespace

PYBIND11_MODULE(_sgv_row_ops, m) {
    pybind11::register_exception<Refused>(m, "Refused", PyExc_RuntimeError);
    pybind11::register_exception<Watched>(m, "Watched", m.attr("Refused"));
    const pybind11::call_guard<pybind11::gil_scoped_release> no_gil;       // (a launch waits where the queue is full)
    m.def("bind", &bind);
    m.def("rms_norm", &rms_norm, no_gil);
    m.def("rms_norm_int8", &rms_norm_int8, no_gil);
    m.def("dequantize_rows", &dequantize_rows, no_gil);
    m.def("matmul", &matmul, no_gil);
    m.def("dense", &dense, no_gil);
}
