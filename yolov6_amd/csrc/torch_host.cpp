// torch_host.cpp - the host side of the training operators that walk torch objects on every call: linear_cross_entropy's autograd node
// and the gradient lists of grad_norm / clip_grad_norm_.  Host code only; the kernels are behind libyolov6_hip.so's C ABI, whose
// entry points `bind` receives from the process's loaded library.
//
// Why C++.  A Python attribute of a tensor costs 0.13 us: a list of 489 gradients (YOLOv6-L) took 368 us of host time in front of 60 us of
// kernels.  A Python autograd node costs the engine's thread the interpreter twice: 64 rows x 1000 classes took 206 us a step, of which
// the kernels were 60.
#include <Python.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/variable.h>

#include <cmath>
#include <unordered_set>
#include <vector>

#include "../../include/yolov6_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
    decltype(&y6_last_error) last_error;
    decltype(&y6_linear_ce_saved_bytes) ce_saved;
    decltype(&y6_linear_ce_workspace_bytes) ce_workspace;
    decltype(&y6_linear_ce_forward) ce_forward;
    decltype(&y6_linear_ce_backward) ce_backward;
    decltype(&y6_grad_norm_workspace_bytes) norm_workspace;
    decltype(&y6_grad_norm) norm;
    decltype(&y6_grad_clip) clip;
} lib = {};

void check(int rc, const char* what) { TORCH_CHECK(rc == Y6_OK, "yolov6_hip ", what, " failed (code ", rc, "): ", lib.last_error()); }
void* stream_of(const c10::Device& d) { return (void*)c10::hip::getCurrentHIPStream(d.index()).stream(); }

int type_code(at::ScalarType t) {
    return t == at::kHalf ? Y6_F16 : t == at::kBFloat16 ? Y6_BF16 : t == at::kFloat ? Y6_F32 : -1;
}
void require_gpu(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), "yolov6_amd: ", name, " must live on a ROCm device (got ", t.device(), "); the hot path has no CPU fallback");
}
std::string shape(const Tensor& t) {
    std::ostringstream s;
    s << t.sizes();
    return s.str();
}
// A dual tensor does not require a gradient, and its tangent would be lost without a word.  (Outside a dual level there is none, and
// asking each of 489 gradients took 7 us.)
bool dual_level() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
void refuse_dual(const Tensor& t, const char* what) {
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "yolov6_amd: ", what, " has no forward mode derivative (a dual tensor was given)");
}
Tensor bytes_on(const Tensor& like, size_t n) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false)); }

// ---------------------------------------------------------------------------------------------------------- linear cross entropy
struct Options {
    int64_t ignore;
    double smoothing;
    int64_t reduction;
    bool recompute;
};

// all but features and labels
y6_linear_ce_desc describe(int64_t rows, const Tensor& w, const Tensor& b, const Options& o) {
    y6_linear_ce_desc d = {};
    d.weight = w.data_ptr(), d.bias = b.defined() ? b.data_ptr() : nullptr;
    d.rows = rows, d.width = (int32_t)w.size(1), d.classes = (int32_t)w.size(0), d.dtype = type_code(w.scalar_type());
    d.w_pitch = d.classes > 1 ? w.stride(0) : d.width;
    d.ignore_index = o.ignore, d.smoothing = (float)o.smoothing, d.reduction = (int32_t)o.reduction;
    d.flags = o.recompute ? Y6_CE_RECOMPUTE : 0;
    return d;
}

// whether the kernels read such a weight where it lies; others are copied, row by row
bool in_place(const Tensor& w) {
    const int64_t rows = w.size(0), width = w.size(1), size = w.element_size();
    return (width == 1 || w.stride(1) == 1) && (rows == 1 || (w.stride(0) >= width && w.stride(0) <= (1 << 21) && w.stride(0) * size % 16 == 0)) &&
           (uintptr_t)w.data_ptr() % 16 == 0;
}

std::tuple<Tensor, Tensor> ce_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& t, const Options& o, bool want_saved) {
    const auto f32 = x.options().dtype(at::kFloat).requires_grad(false);
    const int64_t n = x.size(0);
    const bool rows = o.reduction == Y6_REDUCE_NONE;
    if (n == 0) return {rows ? at::empty({0}, f32) : at::zeros({}, f32), bytes_on(x, 0)};
    const c10::DeviceGuard guard(x.device());
    Tensor loss = rows ? at::empty({n}, f32) : at::empty({}, f32), saved;
    y6_linear_ce_desc d = describe(n, w, b, o);
    d.x = x.data_ptr(), d.x_pitch = n > 1 ? x.stride(0) : d.width, d.target = t.data_ptr<int64_t>();
    d.loss = loss.data_ptr<float>();
    if (want_saved) {
        d.saved_bytes = lib.ce_saved(&d);
        if (d.saved_bytes == 0) check(Y6_EINVAL, "linear_ce_forward");
        saved = bytes_on(x, d.saved_bytes);
        d.saved = saved.data_ptr();
    }
    d.workspace_bytes = lib.ce_workspace(&d, 0);
    if (d.workspace_bytes == 0) check(Y6_EINVAL, "linear_ce_forward");
    const Tensor ws = bytes_on(x, d.workspace_bytes);
    d.workspace = ws.data_ptr();
    check(lib.ce_forward(&d, stream_of(x.device())), "linear_ce_forward");
    return {loss, saved};
}

std::tuple<Tensor, Tensor, Tensor> ce_backward(const Tensor& grad, int64_t n, const Tensor& w, const Tensor& b, const Tensor& saved, const Options& o, bool want_x,
                                               bool want_w, bool want_b) {
    // (saved-tensor hooks, or a caller of the op, may hand over anything: what the kernels would read by its address is looked at here)
    require_gpu(w, "weight");
    TORCH_CHECK(w.dim() == 2 && type_code(w.scalar_type()) >= 0 && w.layout() == at::kStrided, "yolov6_amd: linear_cross_entropy's backward is given a weight ", shape(w));
    const int64_t width = w.size(1), classes = w.size(0);
    for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"gradient", grad}, {"saved bytes", saved}, {"bias", b}})
        TORCH_CHECK(!t.defined() || (t.device() == w.device() && t.layout() == at::kStrided), "yolov6_amd: linear_cross_entropy's backward is given ", name, " on ",
                    t.device(), ", the weight on ", w.device());
    TORCH_CHECK(grad.numel() == (o.reduction == Y6_REDUCE_NONE ? n : 1) && saved.scalar_type() == at::kByte && saved.is_contiguous() &&
                    (!b.defined() || (b.dim() == 1 && b.size(0) == classes && b.scalar_type() == w.scalar_type())),
                "yolov6_amd: linear_cross_entropy's backward of ", n, " rows is given a gradient ", shape(grad), ", saved bytes ", shape(saved), " of ",
                saved.scalar_type(), b.defined() ? ", a bias " + shape(b) : std::string());
    want_b = want_b && b.defined();
    const auto like = w.options().requires_grad(false);
    const c10::DeviceGuard guard(w.device());
    if (n == 0) {
        return {want_x ? at::zeros({0, width}, like) : Tensor(), want_w ? at::zeros({classes, width}, like) : Tensor(),
                want_b ? at::zeros({classes}, like) : Tensor()};
    }
    const Tensor dx = want_x ? at::empty({n, width}, like) : Tensor(), dw = want_w ? at::empty({classes, width}, like) : Tensor(),
                 db = want_b ? at::empty({classes}, like) : Tensor();
    if (!want_x && !want_w && !want_b) return {dx, dw, db};
    const Tensor g = grad.detach().to(at::kFloat).contiguous(), bias = b.defined() ? b.contiguous() : b;
    // Whether the forward took a copy of the weight went by where it lay; saved-tensor hooks may hand it back elsewhere.  The size of
    // `saved` tells: with a copy (16 bytes at least) it is larger.
    y6_linear_ce_desc d = describe(n, w, bias, o);
    d.x = saved.data_ptr(), d.x_pitch = width, d.target = (const int64_t*)saved.data_ptr();           // (the backward reads neither)
    d.flags |= Y6_CE_COPY_WEIGHT;
    d.weight = saved.data_ptr(), d.w_pitch = width;          // (not read then)
    Tensor moved;
    if ((size_t)saved.numel() != lib.ce_saved(&d)) {
        moved = in_place(w) ? w : w.clone(at::MemoryFormat::Contiguous);
        const auto at = describe(n, moved, bias, o);
        d.flags = at.flags, d.weight = at.weight, d.w_pitch = at.w_pitch;
        TORCH_CHECK((size_t)saved.numel() == lib.ce_saved(&d), "yolov6_amd: linear_cross_entropy's backward is given other operands than its forward");
    }
    d.saved = saved.data_ptr(), d.saved_bytes = (size_t)saved.numel(), d.grad_out = g.data_ptr<float>();
    d.dx = want_x ? dx.data_ptr() : nullptr, d.dw = want_w ? dw.data_ptr() : nullptr, d.dbias = want_b ? db.data_ptr() : nullptr;
    d.workspace_bytes = lib.ce_workspace(&d, 1);
    if (d.workspace_bytes == 0) check(Y6_EINVAL, "linear_ce_backward");
    const Tensor ws = bytes_on(w, d.workspace_bytes);
    d.workspace = ws.data_ptr();
    check(lib.ce_backward(&d, stream_of(w.device())), "linear_ce_backward");
    return {dx, dw, db};
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, const Tensor& t, int64_t ignore,
                          double smoothing, int64_t reduction, bool recompute) {
        const Tensor b = bias.has_value() ? *bias : Tensor();
        const Options o = {ignore, smoothing, reduction, recompute};
        auto [loss, saved] = ce_forward(x, w, b, t, o, true);
        // (neither features nor labels: the backward reads what the forward gathered of them, and they may go)
        ctx->save_for_backward({w, b, saved});
        ctx->saved_data["rows"] = x.size(0);
        ctx->saved_data["width"] = w.size(1);
        ctx->saved_data["classes"] = w.size(0);
        ctx->saved_data["type"] = (int64_t)w.scalar_type();
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["smoothing"] = smoothing;
        ctx->saved_data["reduction"] = reduction;
        ctx->saved_data["recompute"] = recompute;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Options o = {ctx->saved_data["ignore"].toInt(), ctx->saved_data["smoothing"].toDouble(), ctx->saved_data["reduction"].toInt(),
                           ctx->saved_data["recompute"].toBool()};
        variable_list out;
        {
            const at::AutoGradMode off(false);
            TORCH_CHECK(s[0].dim() == 2 && s[0].size(0) == ctx->saved_data["classes"].toInt() && s[0].size(1) == ctx->saved_data["width"].toInt() &&
                            (int64_t)s[0].scalar_type() == ctx->saved_data["type"].toInt(),
                        "yolov6_amd: linear_cross_entropy's weight comes back from a saved-tensor hook as ", shape(s[0]), " of ", s[0].scalar_type());
            auto [dx, dw, db] = ce_backward(grads[0], ctx->saved_data["rows"].toInt(), s[0], s[1], s[2], o, ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                            s[1].defined() && ctx->needs_input_grad(2));
            out = {dx, dw, db};
        }
        if (at::GradMode::is_enabled()) {       // create_graph: once differentiable
            const auto stop = std::make_shared<torch::autograd::DelayedError>("yolov6_amd: linear_cross_entropy is differentiable once", 3);
            variable_list marked;
            for (auto& g : out) marked.push_back(g.defined() ? g.set_requires_grad(true) : g);
            out = (*stop)(std::move(marked));
        }
        return {out[0], out[1], out[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// While a stream is captured, a leaf's gradient accumulator must not be one that a living eager graph made on the default stream: the
// engine would make that stream wait for the captured one, which it cannot join, and the capture's end brings the process down.  (Another
// stream joins the capture: a warm-up on a side stream may keep its loss.)
void refuse_outer_graph(const std::initializer_list<const Tensor*>& operands) {
    for (const Tensor* t : operands) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto stream = c10::hip::getCurrentHIPStream(t->device().index());
        hipStreamCaptureStatus state = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(stream.stream(), &state) != hipSuccess || state == hipStreamCaptureStatusNone) return;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        // (by their ids: the two carry different device types, and the streams themselves are never equal)
        TORCH_CHECK(!node || node->input_metadata(0).stream().id() != c10::hip::getDefaultHIPStream(t->device().index()).id(),
                    "yolov6_amd: linear_cross_entropy is captured into a graph while an eager graph over one of its operands, made on the default stream, is "
                    "alive (drop the loss that holds it before the capture, make it on another stream, or capture with a detached operand)");
    }
}

struct Operands {
    Tensor x, w, b, t;
    Options o;
};
// Operands as the kernels take them: features [rows, width], weight [classes, width], target [rows]
Operands operands(const Tensor& features, const Tensor& weight, const Tensor& target, const std::optional<Tensor>& bias_in, int64_t ignore, double smoothing,
                  const std::string& reduction, bool recompute) {
    const Tensor bias = bias_in.has_value() ? *bias_in : Tensor();
    if (dual_level())
        for (const Tensor* t : {&features, &weight, &bias}) refuse_dual(*t, "linear_cross_entropy");
    const int64_t code = reduction == "none" ? Y6_REDUCE_NONE : reduction == "sum" ? Y6_REDUCE_SUM : reduction == "mean" ? Y6_REDUCE_MEAN : -1;
    TORCH_CHECK(code >= 0, "yolov6_amd: linear_cross_entropy reduction '", reduction, "' ('mean', 'sum' or 'none')");
    TORCH_CHECK(smoothing >= 0.0 && smoothing <= 1.0, "yolov6_amd: linear_cross_entropy label_smoothing ", smoothing, " is not in [0, 1]");
    TORCH_CHECK(type_code(features.scalar_type()) >= 0 && weight.scalar_type() == features.scalar_type() &&
                    (!bias.defined() || bias.scalar_type() == features.scalar_type()),
                "yolov6_amd: linear_cross_entropy takes features, weight and bias of one type, fp16, bf16 or fp32 (got ", features.scalar_type(), ", ",
                weight.scalar_type(), bias.defined() ? std::string(", ") + c10::toString(bias.scalar_type()) : std::string(), ")");
    TORCH_CHECK(target.scalar_type() == at::kLong, "yolov6_amd: linear_cross_entropy labels are int64 (got ", target.scalar_type(), ")");
    TORCH_CHECK(features.dim() >= 1 && weight.dim() == 2 && features.size(-1) == weight.size(1) && target.dim() == features.dim() - 1 &&
                    target.sizes() == features.sizes().slice(0, features.dim() - 1) && (!bias.defined() || (bias.dim() == 1 && bias.size(0) == weight.size(0))),
                "yolov6_amd: linear_cross_entropy features ", shape(features), ", weight ", shape(weight), ", target ", shape(target),
                bias.defined() ? ", bias " + shape(bias) : std::string(), " do not fit together");
    TORCH_CHECK(weight.size(0) >= 1 && weight.size(1) >= 1, "yolov6_amd: linear_cross_entropy weight ", shape(weight), " has no class or no column");
    TORCH_CHECK(weight.size(0) <= (1 << 30) && weight.size(1) <= (1 << 20), "yolov6_amd: linear_cross_entropy weight ", shape(weight), " is too large");
    for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"features", features}, {"weight", weight}, {"target", target}, {"bias", bias}}) {
        if (!t.defined()) continue;
        TORCH_CHECK(t.layout() == at::kStrided, "yolov6_amd: linear_cross_entropy ", name, " is not a dense tensor");
        require_gpu(t, name);
        TORCH_CHECK(t.device() == features.device(), "yolov6_amd: linear_cross_entropy ", name, " on ", t.device(), ", features on ", features.device());
    }
    Tensor x = features.dim() == 2 ? features : features.reshape({target.numel(), features.size(-1)}), w = weight;
    if (x.size(1) > 1 && x.stride(1) != 1) x = x.contiguous();
    if ((w.size(1) > 1 && w.stride(1) != 1) || (w.size(0) > 1 && (w.stride(0) < w.size(1) || w.stride(0) > (1 << 21)))) w = w.contiguous();   // (an expanded weight)
    return {x, w, bias.defined() ? bias.contiguous() : bias, target.reshape({-1}).contiguous(), {ignore, smoothing, code, recompute}};
}

Tensor linear_cross_entropy(const Tensor& features, const Tensor& weight, const Tensor& target, const std::optional<Tensor>& bias, int64_t ignore,
                            double smoothing, const std::string& reduction, bool recompute) {
    // (here and not in operands(): the dispatcher's ops take their operands as they are, cast in front of them)
    const bool cast = at::autocast::is_autocast_enabled(at::kCUDA);
    const auto as = [&](const Tensor& t) { return cast ? t.to(at::autocast::get_autocast_dtype(at::kCUDA)) : t; };
    const Operands p = operands(as(features), as(weight), target, bias.has_value() ? std::optional<Tensor>(as(*bias)) : bias, ignore, smoothing, reduction,
                                recompute);
    Tensor loss;
    if (at::GradMode::is_enabled()) {
        const Tensor given = bias.has_value() ? *bias : Tensor();
        refuse_outer_graph({&features, &weight, &given});
    }
    if (at::GradMode::is_enabled() && (p.x.requires_grad() || p.w.requires_grad() || (p.b.defined() && p.b.requires_grad())))
        loss = LinearCrossEntropy::apply(p.x, p.w, p.b.defined() ? std::optional<Tensor>(p.b) : std::nullopt, p.t, p.o.ignore, p.o.smoothing, p.o.reduction,
                                         p.o.recompute);
    else
        loss = std::get<0>(ce_forward(p.x, p.w, p.b, p.t, p.o, false));
    return p.o.reduction == Y6_REDUCE_NONE && target.dim() != 1 ? loss.reshape(target.sizes()) : loss;
}

// -------------------------------------------------------------------------------------------------------------------- gradient lists
std::vector<Tensor> tensors_of(PyObject* seq, bool grads) {
    PyObject* const fast = PySequence_Fast(seq, "a sequence of tensors");
    if (!fast) throw py::error_already_set();
    const py::object keep = py::reinterpret_steal<py::object>(fast);
    std::vector<Tensor> out;
    std::unordered_set<const void*> seen;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    out.reserve((size_t)n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* const o = PySequence_Fast_GET_ITEM(fast, i);
        TORCH_CHECK(THPVariable_Check(o), "yolov6_amd: gradients are taken from tensors");
        const Tensor& t = THPVariable_Unpack(o);
        if (!grads) {
            out.push_back(t);
        } else if (seen.insert(t.unsafeGetTensorImpl()).second) {      // a parameter that comes twice counts once
            const Tensor& g = t.grad();
            if (g.defined()) out.push_back(g);
        }
    }
    return out;
}

struct List {
    std::vector<Tensor> dense;         // outlive the call
    std::vector<void*> at;
    std::vector<int64_t> n;
    std::vector<int32_t> type;
    y6_grad_list c;
    int64_t elements = 0;
    List(const std::vector<Tensor>& grads, int norm) {
        const auto device = grads[0].device();
        const bool dual = dual_level();
        for (const Tensor& g : grads) {
            if (dual) refuse_dual(g, "the gradients' norm");
            const int code = g.layout() == at::kStrided ? type_code(g.scalar_type()) : -1;
            TORCH_CHECK(code >= 0, "yolov6_amd: gradients must be dense fp16, bf16 or fp32 tensors (got ", g.scalar_type(), ", ", g.layout(), ")");
            TORCH_CHECK(g.device() == device, "yolov6_amd: gradients on ", device, " and ", g.device(), ": one norm is taken on one device");
            require_gpu(g, "gradients");
            dense.push_back(g.is_non_overlapping_and_dense() ? g : g.contiguous());
            at.push_back(dense.back().data_ptr());
            n.push_back(g.numel());
            elements += g.numel();
            type.push_back(code);
        }
        c = {at.data(), n.data(), type.data(), (int32_t)at.size(), norm};
    }
};

Tensor norm_of(const List& l) {
    const c10::DeviceGuard guard(l.dense[0].device());
    const size_t size = lib.norm_workspace(l.c.count, l.elements);
    const Tensor ws = bytes_on(l.dense[0], size), out = at::empty({}, l.dense[0].options().dtype(at::kFloat).requires_grad(false));
    check(lib.norm(&l.c, ws.data_ptr(), size, out.data_ptr<float>(), stream_of(ws.device())), "grad_norm");
    return out;
}

Tensor grad_norm(const py::object& grads, int norm) {
    const at::NoGradGuard off;
    const auto list = tensors_of(grads.ptr(), false);
    if (list.empty()) return at::zeros({});
    return norm_of(List(list, norm));
}

Tensor clip_grad_norm(const py::object& parameters, double max_norm, int norm, bool error_if_nonfinite) {
    const at::NoGradGuard off;
    const auto grads = tensors_of(parameters.ptr(), true);
    if (grads.empty()) return at::zeros({});
    // (y6_grad_clip refuses dense ones that overlap; those with gaps are scaled as copies, and it does not see them)
    bool gaps = false;
    for (const Tensor& g : grads) {
        TORCH_CHECK(!g.requires_grad(), "yolov6_amd: gradients that carry a graph (create_graph=True) are not scaled in place");
        if (g.layout() != at::kStrided || g.is_non_overlapping_and_dense()) continue;            // (List refuses the former)
        gaps = true;
        TORCH_CHECK(at::has_internal_overlap(g) != at::MemOverlap::Yes, "yolov6_amd: a gradient whose elements share memory is not scaled in place");
    }
    std::unordered_set<const void*> starts;
    if (gaps)
        for (const Tensor& g : grads)
            TORCH_CHECK(g.numel() == 0 || starts.insert(g.data_ptr()).second, "yolov6_amd: clip_grad_norm_: two gradients share memory");
    const List l(grads, norm);
    TORCH_CHECK(!error_if_nonfinite || std::isfinite(norm_of(l).item<float>()), "yolov6_amd: the norm of the gradients is not finite, so they cannot be clipped");
    const c10::DeviceGuard guard(l.dense[0].device());
    const size_t size = lib.norm_workspace(l.c.count, l.elements);
    const Tensor ws = bytes_on(l.dense[0], size), out = at::empty({}, l.dense[0].options().dtype(at::kFloat).requires_grad(false));
    check(lib.clip(&l.c, max_norm, ws.data_ptr(), size, out.data_ptr<float>(), stream_of(ws.device())), "grad_clip");
    for (size_t i = 0; i < grads.size(); ++i) {
        // (autograd has to see the write: a graph that saved the gradient would use it as it is now.  Inference tensors have no counter)
        if (!l.dense[i].is_same(grads[i])) const_cast<Tensor&>(grads[i]).copy_(l.dense[i]);
        else if (!grads[i].is_inference()) grads[i].unsafeGetTensorImpl()->bump_version();
    }
    return out;
}

}  // namespace

PYBIND11_MODULE(_y6_torch, m) {
    m.def("bind", [](const std::vector<uintptr_t>& f) {
        TORCH_CHECK(f.size() == 8, "eight entry points");
        lib = {(decltype(lib.last_error))f[0], (decltype(lib.ce_saved))f[1], (decltype(lib.ce_workspace))f[2], (decltype(lib.ce_forward))f[3],
               (decltype(lib.ce_backward))f[4], (decltype(lib.norm_workspace))f[5], (decltype(lib.norm))f[6], (decltype(lib.clip))f[7]};
    });
    m.def("linear_cross_entropy", &linear_cross_entropy);
    m.def("linear_cross_entropy_refuse_outer_graph", [](const Tensor& x, const Tensor& w, const std::optional<Tensor>& b) {
        const Tensor given = b.has_value() ? *b : Tensor();
        refuse_outer_graph({&x, &w, &given});
    });
    m.def("linear_cross_entropy_forward", [](const Tensor& x, const Tensor& w, const Tensor& t, const std::optional<Tensor>& b, int64_t ignore, double smoothing,
                                             const std::string& reduction, bool recompute) {
        const at::NoGradGuard off;
        const Operands p = operands(x, w, t, b, ignore, smoothing, reduction, recompute);
        auto [loss, saved] = ce_forward(p.x, p.w, p.b, p.t, p.o, true);
        return std::make_tuple(p.o.reduction == Y6_REDUCE_NONE ? loss.reshape(t.sizes()) : loss, saved);
    });
    m.def("linear_cross_entropy_backward", [](const Tensor& grad, const Tensor& x, const Tensor& w, const Tensor& t, const std::optional<Tensor>& b, const Tensor& saved,
                                              int64_t ignore, double smoothing, const std::string& reduction, bool recompute) {
        const at::NoGradGuard off;
        const Operands p = operands(x, w, t, b, ignore, smoothing, reduction, recompute);
        auto [dx, dw, db] = ce_backward(grad.reshape({-1}), p.x.size(0), p.w, p.b, saved, p.o, true, true, p.b.defined());
        return std::make_tuple(dx.reshape(x.sizes()), dw, p.b.defined() ? db : at::empty({0}, dw.options()));
    });
    m.def("grad_norm", &grad_norm);
    m.def("clip_grad_norm", &clip_grad_norm);
}
