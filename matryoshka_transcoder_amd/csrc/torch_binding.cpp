// Host side of the block norms and of the gradient clipping on torch tensors: argument checks, outputs, workspaces, streams and the
// autograd node, in C++.  The calls are a few microseconds of GPU work for a token or a small list of gradients, where the
// same steps in Python cost 15 us forward, 110 us for a list of 61 tensors and, through a Python autograd node on the
// engine's thread, 150 us forward and backward.  No kernel is here: everything computes in libmtc.so, whose entry
// points are handed over by address (bind), so that this module and ctypes drive the one library that is loaded.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <limits>
#include <sstream>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/mtc.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

namespace {

struct MtcError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

template <typename... A> [[noreturn]] void fail(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    throw MtcError(s.str());
}

struct Lib {
    decltype(&mtc_last_error) last_error = nullptr;
    decltype(&mtc_block_norm_fwd) norm_fwd = nullptr;
    decltype(&mtc_block_norm_bwd) norm_bwd = nullptr;
    decltype(&mtc_block_norm_bwd_workspace_bytes) norm_ws = nullptr;
    decltype(&mtc_grad_norm_workspace_bytes) clip_ws = nullptr;
    decltype(&mtc_grad_norm) grad_norm = nullptr;
    decltype(&mtc_grad_clip) grad_clip = nullptr;
} lib;

void check(int rc, const char* what) {
    if (rc) fail(what, " failed (", rc, "): ", lib.last_error());
}

// What records torch operations (jit.trace, make_fx, export and what builds on them) sees an output's allocation and nothing of the kernel
// that fills it: the record would return memory that nobody wrote.
void refuse_tracing(const char* what) {
    if (at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
        c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value())
        fail(what, " cannot be traced (torch.jit.trace, make_fx): the kernel would be missing from the trace");
}

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int dtype_code(const Tensor& t, const char* what) {
    if (t.scalar_type() == at::kFloat) return MTC_F32;
    if (t.scalar_type() == at::kBFloat16) return MTC_BF16;
    fail(what, " ", t.dtype(), ": libmtc computes in float32 or bfloat16");
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ------------------------------------------------------------------------------------------------ block norms
constexpr int64_t MAX_WIDTH = 8192;

struct Plan {
    int64_t A, rows;
    int dtype, branch, post_kind, pre_kind, gate_kind;
    float post_eps, pre_eps, post_off, pre_off, rs, bs;
    bool need[7];                       // gradients: residual, branch, gate, post w, post b, pre w, pre b

    mtc_block_norm_desc desc(bool pre) const {
        mtc_block_norm_desc d = {};
        d.rows = rows; d.A = (int32_t)A; d.dtype = dtype; d.has_branch = branch; d.gate_kind = gate_kind;
        d.post_kind = post_kind; d.post_eps = post_eps; d.post_offset = post_off;
        if (pre) { d.pre_kind = pre_kind; d.pre_eps = pre_eps; d.pre_offset = pre_off; }
        d.residual_scale = rs; d.branch_scale = bs;
        return d;
    }
};

struct PlanHolder : torch::CustomClassHolder {
    Plan p;
    explicit PlanHolder(const Plan& q) : p(q) {}
};

// [rows, A] with contiguous columns: a view, or a copy where the leading dimensions do not collapse or the columns are
// strided; ld receives its row stride
Tensor rows_of(const Tensor& t, int64_t A, int64_t& ld) {
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, A});
    if (A > 1 && r.stride(1) != 1) r = r.contiguous();
    ld = r.stride(0);
    return r;
}

struct Operands {
    Tensor residual, branch, gate;
    Operands(const Plan& p, const Tensor& r, const Tensor& b, const Tensor& g, mtc_block_norm_desc& d) {
        residual = rows_of(r, p.A, d.ld_residual);
        if (p.branch) branch = rows_of(b, p.A, d.ld_branch);
        if (p.gate_kind == MTC_GATE_CHANNEL) gate = g.contiguous();
        else if (p.gate_kind == MTC_GATE_SCALAR) gate = g;
        else if (p.gate_kind == MTC_GATE_ROW) gate = rows_of(g, 1, d.ld_gate);
        else if (p.gate_kind == MTC_GATE_FULL) gate = rows_of(g, p.A, d.ld_gate);
    }
};

std::tuple<Tensor, Tensor> norm_forward(const Plan& p, const Tensor& residual, const Tensor& branch, const Tensor& gate, const Tensor& post_w,
                                        const Tensor& post_b, const Tensor& pre_w, const Tensor& pre_b, const Tensor& stats) {
    Tensor hidden, normed;
    c10::DeviceGuard guard(residual.device());
    if (p.branch) hidden = at::empty(residual.sizes(), residual.options());
    if (p.pre_kind) normed = at::empty(residual.sizes(), residual.options());
    if (p.rows) {
        mtc_block_norm_desc d = p.desc(true);
        d.ld_hidden = d.ld_normed = p.A;
        const Operands o(p, residual, branch, gate, d);
        check(lib.norm_fwd(&d, ptr(o.residual), ptr(o.branch), ptr(o.gate), ptr(post_w), ptr(post_b), ptr(pre_w), ptr(pre_b), ptr(hidden),
                           ptr(normed), (float*)ptr(stats), stream_of(residual)),
              "mtc_block_norm_fwd");
    }
    return {hidden, normed};
}

Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// The engine adds a leaf's gradient on the stream on which the leaf's accumulation node was made, and an eager graph that is still alive
// keeps that node.  Recorded into a HIP graph, the default stream would have to wait for the recording, which ends the process.
void check_recorded_leaf(const Tensor& t) {
    if (!t.is_leaf()) return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = node ? node->stream() : std::nullopt;
    if (stream && stream->id() == 0)
        fail("a backward of the block norms cannot be recorded into a HIP graph while an eager graph of the same leaf, made on the default "
             "stream, is alive: release it first (its outputs or loss)");
}

struct BlockNormFn : torch::autograd::Function<BlockNormFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& residual, const OptTensor& branch, const OptTensor& gate,
                                 const OptTensor& post_w, const OptTensor& post_b, const OptTensor& pre_w, const OptTensor& pre_b, const Plan& p) {
        const Tensor br = get(branch), g = get(gate), w0 = get(post_w), b0 = get(post_b), w1 = get(pre_w), b1 = get(pre_b);
        const Tensor stats = at::empty({p.rows, 4}, residual.options().dtype(at::kFloat));
        auto [hidden, normed] = norm_forward(p, residual, br, g, w0, b0, w1, b1, stats);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({stats, residual, br, g, w0, b0, w1, b1});
        ctx->saved_data["plan"] = c10::IValue::make_capsule(c10::make_intrusive<PlanHolder>(p));
        if (p.branch && p.pre_kind) return {hidden, normed};
        return {p.branch ? hidden : normed};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (at::GradMode::is_enabled()) fail("the block norms have no second derivative (create_graph = True)");
        const Plan p = static_cast<PlanHolder*>(ctx->saved_data["plan"].toCapsule().get())->p;
        const variable_list s = ctx->get_saved_variables();
        const Tensor &stats = s[0], &residual = s[1], &branch = s[2], &gate = s[3];
        variable_list out(8);
        Tensor dh = p.branch ? grads[0] : Tensor(), dn = p.pre_kind ? grads.back() : Tensor();
        if (!dh.defined() && !dn.defined()) return out;
        const bool pre = dn.defined();
        c10::DeviceGuard guard(residual.device());
        const bool recording = c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
        bool need[7];
        for (int i = 0, edge = 0; i < 7; ++i) {
            need[i] = p.need[i] && ctx->needs_input_grad(edge);      // edges: the operands that are there
            edge += s[1 + i].defined();
            if (!need[i]) continue;
            if (recording) check_recorded_leaf(s[1 + i]);
            // rows of nothing, and a pre norm whose output nobody used, leave zeros
            const bool zero = !p.rows || (i >= 5 && !pre);
            out[i] = zero ? at::zeros(s[1 + i].sizes(), residual.options()) : at::empty(s[1 + i].sizes(), residual.options());
        }
        if (!p.rows) return out;
        mtc_block_norm_desc d = p.desc(pre);
        const Operands o(p, residual, branch, gate, d);
        int64_t ld_dh = 0, ld_dn = 0;
        if (dh.defined()) dh = rows_of(dh, p.A, ld_dh);
        if (pre) dn = rows_of(dn, p.A, ld_dn);
        Tensor ws;
        size_t ws_bytes = 0;
        const bool gate_sum = need[2] && (p.gate_kind == MTC_GATE_CHANNEL || p.gate_kind == MTC_GATE_SCALAR);
        if (need[3] || need[4] || need[5] || need[6] || gate_sum) {
            ws_bytes = lib.norm_ws(&d);
            ws = at::empty({(int64_t)ws_bytes}, residual.options().dtype(at::kByte));
        }
        check(lib.norm_bwd(&d, ptr(o.residual), ptr(o.branch), ptr(o.gate), ptr(s[4]), ptr(s[5]), ptr(s[6]), ptr(s[7]), (const float*)ptr(stats),
                           ptr(dh), ld_dh, ptr(dn), ld_dn, ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(out[3]), ptr(out[4]),
                           pre ? ptr(out[5]) : nullptr, pre ? ptr(out[6]) : nullptr, ptr(ws), ws_bytes, stream_of(residual)),
              "mtc_block_norm_bwd");
        return out;
    }
};

OptTensor norm_vector(const OptTensor& t, int64_t A, const Tensor& like, const char* what, const char* part) {
    if (!t.has_value() || !t->defined()) return std::nullopt;
    if (t->device() != like.device() || t->scalar_type() != like.scalar_type() || t->dim() != 1 || t->size(0) != A)
        fail(what, " ", part, " must be [", A, "] of ", like.dtype(), " on ", like.device(), ", got ", t->sizes(), " of ", t->dtype(), " on ", t->device());
    return t->is_contiguous() ? *t : t->contiguous();
}

int gate_kind(const OptTensor& gate, const Tensor& like) {
    if (!gate.has_value() || !gate->defined()) return MTC_GATE_NONE;
    if (gate->device() != like.device() || gate->scalar_type() != like.scalar_type())
        fail("gate must be ", like.dtype(), " on ", like.device(), ", got ", gate->dtype(), " on ", gate->device());
    const int64_t A = like.size(-1), n = like.dim(), gd = gate->dim();
    if (gd == 1 && gate->size(0) == A) return MTC_GATE_CHANNEL;
    if (gd == 0 || (gd == 1 && gate->size(0) == 1)) return MTC_GATE_SCALAR;
    if (gate->sizes() == like.sizes()) return MTC_GATE_FULL;
    if (gd == n && gate->size(-1) == 1 && gate->sizes().slice(0, n - 1) == like.sizes().slice(0, n - 1)) return MTC_GATE_ROW;
    fail("gate of shape ", gate->sizes(), " fits neither a scalar, [", A, "], ", like.sizes().slice(0, n - 1), " + [1] nor ", like.sizes());
}

// (hidden or None, normed or None)
std::tuple<OptTensor, OptTensor> block_norm(const Tensor& residual, const OptTensor& branch, const OptTensor& gate, int post_kind,
                                            const OptTensor& post_w, const OptTensor& post_b, double post_eps, double post_off,
                                            int64_t post_width, int pre_kind, const OptTensor& pre_w, const OptTensor& pre_b, double pre_eps,
                                            double pre_off, int64_t pre_width, double rs, double bs) {
    refuse_tracing("a block norm");
    if (!residual.is_cuda())
        fail("the block norms run on the GPU only (HIP kernels); got a ", residual.device(), " tensor and there is no CPU fallback");
    if (residual.dim() < 1) fail("a norm needs a tensor with at least one dimension");
    Plan p = {};
    p.dtype = dtype_code(residual, "unsupported model dtype");
    p.A = residual.size(-1);
    if (p.A < 1 || p.A > MAX_WIDTH) fail("norm width ", p.A, " outside 1..", MAX_WIDTH);
    p.rows = residual.numel() / p.A;
    p.branch = branch.has_value() && branch->defined();
    if (p.branch && (branch->sizes() != residual.sizes() || branch->scalar_type() != residual.scalar_type() || branch->device() != residual.device()))
        fail("residual and branch must share shape, dtype and device: ", residual.sizes(), " ", residual.dtype(), " ", residual.device(),
             " against ", branch->sizes(), " ", branch->dtype(), " ", branch->device());
    p.post_kind = post_kind; p.pre_kind = pre_kind;
    if (post_kind && post_width != p.A) fail("post norm of width ", post_width, " on activations of width ", p.A);
    if (pre_kind && pre_width != p.A) fail("pre norm of width ", pre_width, " on activations of width ", p.A);
    p.post_eps = (float)post_eps; p.pre_eps = (float)pre_eps; p.post_off = (float)post_off; p.pre_off = (float)pre_off;
    p.rs = (float)rs; p.bs = (float)bs;
    const OptTensor t[7] = {residual, branch, gate, norm_vector(post_w, p.A, residual, "post", "weight"),
                            norm_vector(post_b, p.A, residual, "post", "bias"), norm_vector(pre_w, p.A, residual, "pre", "weight"),
                            norm_vector(pre_b, p.A, residual, "pre", "bias")};
    p.gate_kind = gate_kind(gate, residual);
    for (const OptTensor& x : t)
        if (x.has_value() && x->defined() && x->_fw_grad(0).defined()) fail("the block norms have no forward-mode derivative");
    bool any = false;
    if (at::GradMode::is_enabled())
        for (int i = 0; i < 7; ++i) any |= p.need[i] = t[i].has_value() && t[i]->defined() && t[i]->requires_grad();
    if (!any) {
        auto [hidden, normed] = norm_forward(p, residual, get(t[1]), get(t[2]), get(t[3]), get(t[4]), get(t[5]), get(t[6]), Tensor());
        return {p.branch ? OptTensor(hidden) : std::nullopt, p.pre_kind ? OptTensor(normed) : std::nullopt};
    }
    const variable_list o = BlockNormFn::apply(residual, t[1], t[2], t[3], t[4], t[5], t[6], p);
    return {p.branch ? OptTensor(o[0]) : std::nullopt, p.pre_kind ? OptTensor(o.back()) : std::nullopt};
}

// ------------------------------------------------------------------------------------------------ gradient clipping
float norm_order(double p) {
    if (p != 1.0 && p != 2.0 && p != std::numeric_limits<double>::infinity()) fail("the norm's order must be 1, 2 or inf, got ", p);
    return (float)p;
}

float norm_limit(double m) {
    if (!(m >= 0.0)) fail("max_norm must not be negative or NaN, got ", m);
    return (float)m;
}

void check_gradients(const std::vector<Tensor>& ts) {
    for (const Tensor& t : ts) {
        if (!t.is_cuda()) fail("gradient clipping runs on the GPU only (HIP kernels); got a ", t.device(), " tensor and there is no CPU fallback");
        if (t.layout() != at::kStrided) fail("gradients must be dense tensors, got ", t.layout());
        if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) fail("gradients must be float32 or bfloat16, got ", t.dtype());
        if (t.device() != ts[0].device()) fail("all gradients must live on one GPU, got ", ts[0].device(), " and ", t.device());
    }
}

// host arrays and workspace of one call over tensors that hold every element once, without gaps
struct ClipCall {
    std::vector<const void*> src;
    std::vector<uint64_t> elems;
    std::vector<int32_t> dtype;
    Tensor ws;
    size_t ws_bytes;
    explicit ClipCall(const std::vector<Tensor>& ts) {
        src.reserve(ts.size()); elems.reserve(ts.size()); dtype.reserve(ts.size());
        for (const Tensor& t : ts) {
            src.push_back(t.numel() ? t.data_ptr() : nullptr);
            elems.push_back((uint64_t)t.numel());
            dtype.push_back(t.scalar_type() == at::kFloat ? MTC_F32 : MTC_BF16);
        }
        ws_bytes = lib.clip_ws((int32_t)ts.size(), elems.data(), dtype.data());
        ws = at::empty({(int64_t)ws_bytes}, ts[0].options().dtype(at::kByte));
    }
    void norm(float p, double* total, float max_norm, float* norm_coef) const {
        check(lib.grad_norm((int32_t)src.size(), src.data(), elems.data(), dtype.data(), p, ws.data_ptr(), ws_bytes, total, max_norm, norm_coef,
                            stream_of(ws)),
              "mtc_grad_norm");
    }
};

std::vector<Tensor> dense(const std::vector<Tensor>& ts) {
    std::vector<Tensor> out;
    out.reserve(ts.size());
    for (const Tensor& t : ts) out.push_back(t.is_non_overlapping_and_dense() ? t : t.contiguous());
    return out;
}

// {norm, coef} (fp32), or with `raw` the sum before the root (fp64)
Tensor norm_of(const std::vector<Tensor>& ts, double order, double max_norm, bool raw) {
    refuse_tracing("a gradient norm");
    const float p = norm_order(order), limit = norm_limit(max_norm);
    check_gradients(ts);
    if (ts.empty()) fail("no gradients to take a norm of");
    c10::DeviceGuard guard(ts[0].device());
    at::NoGradGuard no_grad;
    const std::vector<Tensor> d = dense(ts);
    const ClipCall call(d);
    const Tensor out = raw ? at::empty({}, ts[0].options().dtype(at::kDouble)) : at::empty({2}, ts[0].options().dtype(at::kFloat));
    if (raw) call.norm(p, out.data_ptr<double>(), limit, nullptr);
    else call.norm(p, nullptr, limit, out.data_ptr<float>());
    return out;
}

// mtc_grad_clip refuses outputs that share memory; those written by a copy after it are held to the same, by the ranges they span
void check_copied_outputs(const std::vector<Tensor>& dst, const std::vector<Tensor>& copied) {
    struct Span { uintptr_t a, b; size_t i; };
    std::vector<Span> s;
    bool any = false;
    for (size_t i = 0; i < dst.size(); ++i) {
        if (!dst[i].numel()) continue;
        uintptr_t elems = 1;
        for (int64_t k = 0; k < dst[i].dim(); ++k) elems += (uintptr_t)((dst[i].size(k) - 1) * dst[i].stride(k));
        const uintptr_t a = (uintptr_t)dst[i].data_ptr();
        s.push_back({a, a + elems * dst[i].element_size(), i});
        any |= copied[i].defined();
    }
    if (!any) return;
    std::sort(s.begin(), s.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
    for (size_t k = 1, last = 0; k < s.size(); ++k) {                // last: the furthest end so far
        if (s[k].a < s[last].b && (copied[s[k].i].defined() || copied[s[last].i].defined()))
            fail("outputs ", s[last].i, " and ", s[k].i, " span the same memory");
        if (s[k].b > s[last].b) last = k;
    }
}

Tensor clip(const std::vector<Tensor>& src, const std::optional<std::vector<Tensor>>& out, double order, double max_norm) {
    refuse_tracing("gradient clipping");
    const float p = norm_order(order), limit = norm_limit(max_norm);
    const std::vector<Tensor>& dst = out.has_value() ? *out : src;
    check_gradients(src);
    if (out.has_value()) {
        if (src.empty() && !dst.empty()) fail("out has tensors but there are none to clip");
        if (dst.size() != src.size()) fail(src.size(), " tensors but ", dst.size(), " outputs");
        for (size_t i = 0; i < src.size(); ++i)
            if (src[i].sizes() != dst[i].sizes() || src[i].scalar_type() != dst[i].scalar_type() || src[i].device() != dst[i].device())
                fail("output ", i, " must be ", src[i].sizes(), " of ", src[i].dtype(), " on ", src[i].device(), ", got ", dst[i].sizes(), " of ",
                     dst[i].dtype(), " on ", dst[i].device());
    }
    for (const Tensor& o : dst)
        for (int64_t k = 0; k < o.dim(); ++k)
            if (o.stride(k) == 0 && o.size(k) > 1) fail("a tensor that repeats its memory (expanded) cannot be written");
    if (src.empty()) return at::zeros({});
    c10::DeviceGuard guard(src[0].device());
    at::NoGradGuard no_grad;
    // the kernel walks over memory: inputs with gaps, and outputs laid out another way, go through a dense copy
    const std::vector<Tensor> a = dense(src);
    std::vector<Tensor> back(src.size());
    std::vector<void*> to(src.size());
    for (size_t i = 0; i < src.size(); ++i) {
        if (a[i].numel() && dst[i].strides() != a[i].strides()) back[i] = at::empty_like(a[i]);
        to[i] = !a[i].numel() ? nullptr : back[i].defined() ? back[i].data_ptr() : dst[i].data_ptr();
    }
    if (out.has_value()) check_copied_outputs(dst, back);
    const ClipCall call(a);
    const Tensor norm = at::empty({}, src[0].options().dtype(at::kFloat));
    check(lib.grad_clip((int32_t)a.size(), call.src.data(), to.data(), call.elems.data(), call.dtype.data(), p, limit, call.ws.data_ptr(),
                        call.ws_bytes, norm.data_ptr<float>(), stream_of(norm)),
          "mtc_grad_clip");
    for (size_t i = 0; i < src.size(); ++i) {
        if (back[i].defined()) dst[i].copy_(back[i]);
        else if (!dst[i].is_inference()) dst[i].unsafeGetTensorImpl()->bump_version();       // written behind autograd's back
    }
    return norm;
}

PyObject* error_class = nullptr;

template <typename F> void bind_one(const py::dict& addresses, const char* name, F& f) {
    f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

}  // namespace

PYBIND11_MODULE(_torch_binding, m) {
    m.doc() = "libmtc's block norms and gradient clipping on torch tensors";
    m.def("bind", [](const py::dict& addresses, const py::object& error) {
        bind_one(addresses, "mtc_last_error", lib.last_error);
        bind_one(addresses, "mtc_block_norm_fwd", lib.norm_fwd);
        bind_one(addresses, "mtc_block_norm_bwd", lib.norm_bwd);
        bind_one(addresses, "mtc_block_norm_bwd_workspace_bytes", lib.norm_ws);
        bind_one(addresses, "mtc_grad_norm_workspace_bytes", lib.clip_ws);
        bind_one(addresses, "mtc_grad_norm", lib.grad_norm);
        bind_one(addresses, "mtc_grad_clip", lib.grad_clip);
        error_class = error.inc_ref().ptr();
    });
    py::register_exception_translator([](std::exception_ptr e) {
        try {
            if (e) std::rethrow_exception(e);
        } catch (const MtcError& x) {
            PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, x.what());
        }
    });
    m.def("block_norm", &block_norm, py::call_guard<py::gil_scoped_release>());
    m.def("norm_of", &norm_of, py::call_guard<py::gil_scoped_release>());
    m.def("refuse_tracing", &refuse_tracing);
    m.def("clip", &clip, py::call_guard<py::gil_scoped_release>());
}
