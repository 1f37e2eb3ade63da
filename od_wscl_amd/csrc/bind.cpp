// bind.cpp -- torch-side glue of the optimiser and the row norm (od_wscl_amd/_bind.so): argument checks over tensor lists, workspaces,
// and the norm's autograd node, in front of the C-ABI of libodwscl.so.
//
// The other operators are bound by ctypes; these are called with lists of a hundred small tensors, or once a layer on a few rows, where
// Python's look at each tensor (0.35 us for its device, type, size, layout and address) was most of the call.  From Python / from here,
// us: 8-bit AdamW over 120 tensors 200 / 38 (its kernels 28), clipping 16 tensors 29 / 17.5, the norm of one row 13.7 / 6.8, forward and
// backward of 447 x 1373 53 to 108 / 58 to 60 (the autograd engine hands over to its own thread: 33 for a node without a kernel).  No
// kernel lives here.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>

#include "../../include/odwscl.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

std::string format(const char* fmt, va_list ap) {
    char text[512];
    vsnprintf(text, sizeof(text), fmt, ap);
    return text;
}
[[noreturn]] void value_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    const std::string s = format(fmt, ap);
    va_end(ap);
    throw py::value_error(s);
}
[[noreturn]] void type_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    const std::string s = format(fmt, ap);
    va_end(ap);
    throw py::type_error(s);
}
void need_gpu(const Tensor& t) {
    if (!t.is_cuda()) throw std::runtime_error("od_wscl_amd: tensor is not on the GPU -- the hot path has no CPU implementation");
    // (the stand-ins of torch.func's transforms)
    if (t.layout() == at::kStrided && !t.has_storage())
        throw std::runtime_error("od_wscl_amd: tensor has no memory of its own -- a transform's stand-in");
}
void check(int code, const char* what) {
    if (code != 0) throw std::runtime_error(std::string(what) + " failed (" + std::to_string(code) + "): " + odw_last_error());
}
// (a trace would record the empty outputs and not the launches that fill them)
void not_traced(const char* what) {
    if (torch::jit::tracer::isTracing()) throw std::runtime_error(std::string(what) + ": cannot be traced");
}
std::string name_of(at::ScalarType t) { return std::string("torch.") + at::toString(t); }
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// The tensors were written: autograd's saved copies of them are stale (those made in inference mode have no version to count).
void changed(const std::vector<Tensor>& list) {
    for (const Tensor& t : list)
        if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---- the optimiser ----------------------------------------------------------------------------------------------------------------

typedef std::vector<at::ScalarType> Types;

std::string names_of(const Types& types) {
    std::string s;
    for (at::ScalarType t : types) s += (s.empty() ? "" : " | ") + name_of(t);
    return s;
}

// `list` beside the first one: as many, on its GPU, contiguous, of one of `types` and of `sizes`; their addresses.  What is written must
// not be in a list twice (two workgroups would update it at once).  `alone` (a norm, a scaling): elements go with no other list's, so
// that any order without gaps will do, and a lazily negated view too, whose memory holds the other sign.
std::vector<void*> addresses(const char* what, const char* name, const std::vector<Tensor>& list, int device, const std::vector<int64_t>& sizes,
                             const Types& types, bool written, bool alone = false) {
    if (list.size() != sizes.size()) value_error("%s: %zu %s for %zu tensors", what, list.size(), name, sizes.size());
    std::vector<void*> at;
    at.reserve(list.size());
    for (size_t i = 0; i < list.size(); ++i) {
        const Tensor& t = list[i];
        need_gpu(t);
        if (t.get_device() != device)
            value_error("%s: %s[%zu] is on cuda:%d, tensor 0 on cuda:%d", what, name, i, (int)t.get_device(), device);
        bool known = false;
        for (at::ScalarType k : types) known |= t.scalar_type() == k;
        if (!known || t.layout() != at::kStrided)
            type_error("%s: %s[%zu] is %s%s (%s)", what, name, i, t.layout() != at::kStrided ? "sparse " : "", name_of(t.scalar_type()).c_str(),
                       names_of(types).c_str());
        if (t.numel() != sizes[i])
            value_error("%s: %s[%zu] has %lld elements, %lld wanted", what, name, i, (long long)t.numel(), (long long)sizes[i]);
        if (alone ? !t.is_non_overlapping_and_dense() : !t.is_contiguous()) value_error("%s: %s[%zu] is not contiguous", what, name, i);
        if (!alone && t.is_neg()) value_error("%s: %s[%zu] is a negated view (resolve_neg)", what, name, i);
        at.push_back(t.numel() ? t.data_ptr() : nullptr);
    }
    if (written) {
        std::vector<void*> seen = at;
        std::sort(seen.begin(), seen.end());
        for (size_t i = 1; i < seen.size(); ++i)
            if (seen[i] && seen[i] == seen[i - 1]) value_error("%s: the same tensor is in `%s` twice", what, name);
    }
    return at;
}

std::vector<int64_t> sizes_of(const std::vector<Tensor>& list) {
    std::vector<int64_t> n;
    n.reserve(list.size());
    for (const Tensor& t : list) n.push_back(t.numel());
    return n;
}

const Types kFloats = {at::kFloat, at::kBFloat16};

// out[0] = the norm, out[1] = the factor that clips it.
Tensor norm_of(const char* what, const std::vector<Tensor>& grads, double max_norm, bool written) {
    not_traced(what);
    if (grads.empty()) value_error("%s: no gradients", what);
    need_gpu(grads[0]);
    const std::vector<int64_t> n = sizes_of(grads);
    const std::vector<void*> at = addresses(what, "grads", grads, grads[0].get_device(), n, kFloats, written, true);
    if (!(max_norm > 0.0)) value_error("%s: max_norm = %g", what, max_norm);
    std::vector<int> types;
    for (const Tensor& g : grads) types.push_back(g.scalar_type() == at::kBFloat16 ? 2 : 0);
    const c10::DeviceGuard guard(grads[0].device());
    const int count = (int)grads.size();
    const int64_t bytes = odw_grad_norm_workspace(count, n.data());
    const Tensor ws = at::empty({bytes}, grads[0].options().dtype(at::kByte)), out = at::empty({2}, grads[0].options().dtype(at::kFloat));
    void* stream = stream_of(out);
    check(odw_grad_norm(count, at.data(), n.data(), types.data(), max_norm, out.data_ptr<float>(), bytes ? ws.data_ptr() : nullptr, bytes, stream),
          "grad_norm");
    if (written) {
        check(odw_scale_tensors(count, at.data(), n.data(), types.data(), out.data_ptr<float>() + 1, stream), "scale_tensors");
        changed(grads);
    }
    return out;
}

// Gradients out of tensors and / or parameters: a leaf that requires grad stands for its .grad.
std::vector<Tensor> grads_of(const char* what, const std::vector<Tensor>& items, bool any_layout) {
    std::vector<Tensor> grads;
    for (const Tensor& t : items) {
        const Tensor g = t.requires_grad() && t.is_leaf() ? t.grad() : t.detach();
        if (!g.defined()) continue;
        if (g.layout() != at::kStrided) type_error("%s: gradient %zu is sparse", what, grads.size());
        grads.push_back(any_layout && !g.is_non_overlapping_and_dense() ? g.contiguous() : g);
    }
    return grads;
}

py::object grad_norm(const std::vector<Tensor>& items, std::optional<double> max_norm) {
    const at::NoGradGuard no_grad;
    const Tensor out = norm_of("grad_norm", grads_of("grad_norm", items, true), max_norm ? *max_norm : INFINITY, false);
    if (!max_norm) return py::cast(out.select(0, 0));
    return py::make_tuple(out.select(0, 0), out.select(0, 1));
}

Tensor clip_grad_norm(const std::vector<Tensor>& items, double max_norm) {
    const at::NoGradGuard no_grad;
    const std::vector<Tensor> grads = grads_of("clip_grad_norm_", items, false);
    if (grads.empty() && max_norm > 0.0) return at::zeros({}, (items.empty() ? at::TensorOptions() : items[0].options()).dtype(at::kFloat));
    return norm_of("clip_grad_norm_", grads, max_norm, true).select(0, 0);
}

std::vector<float> scalars(const char* what, const char* name, const py::object& value, size_t n) {
    std::vector<float> out;
    out.reserve(n);
    auto push = [&](double x) {
        if (!(x >= 0.0 && std::isfinite((float)x))) value_error("%s: %s = %g", what, name, x);
        out.push_back((float)x);
    };
    if (PyFloat_Check(value.ptr()) || PyLong_Check(value.ptr())) {
        push(value.cast<double>());
        out.resize(n, out[0]);
    } else {
        for (const py::handle& x : py::reinterpret_borrow<py::sequence>(value)) push(x.cast<double>());
        if (out.size() != n) value_error("%s: %zu values of %s for %zu tensors", what, out.size(), name, n);
    }
    return out;
}

void device_scalar(const char* what, const char* name, const Tensor& t, int device, at::ScalarType type) {
    if (t.numel() != 1 || t.scalar_type() != type || !t.is_cuda() || t.get_device() != device)
        value_error("%s: %s has to be one %s on cuda:%d (got %s of %lld elements)", what, name, name_of(type).c_str(), device,
                    name_of(t.scalar_type()).c_str(), (long long)t.numel());
}

void adamw(bool bits8, const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& m, const std::vector<Tensor>& v,
           const std::optional<std::vector<Tensor>>& scales, const py::object& step, const std::vector<int64_t>& key, const py::object& lr,
           const std::vector<double>& betas, double eps, const py::object& weight_decay, const OptTensor& grad_scale,
           const std::optional<std::vector<OptTensor>>& copies, double grad_mult, int64_t max_workgroups, bool hold_v) {
    const char* what = bits8 ? "adamw8_step" : "adamw_step";
    not_traced(what);
    const at::NoGradGuard no_grad;
    if (bits8 && (key.size() != 2 || key[0] < 0 || key[1] < 0 || key[0] >> 32 || key[1] >> 32))
        value_error("%s: key has to be two 32-bit integers", what);
    if (params.empty()) return;
    need_gpu(params[0]);
    const int device = params[0].get_device();
    const size_t count = params.size();
    const std::vector<int64_t> n = sizes_of(params);
    const std::vector<void*> ap = addresses(what, "params", params, device, n, kFloats, true),
                             ag = addresses(what, "grads", grads, device, n, kFloats, false),
                             am = addresses(what, "exp_avgs", m, device, n, {bits8 ? at::kFloat8_e4m3fn : at::kFloat}, true),
                             av = addresses(what, "exp_avg_sqs", v, device, n, {bits8 ? at::kFloat8_e5m2 : at::kFloat}, true);
    std::vector<void*> ae, ac;
    if (bits8) {
        std::vector<int64_t> blocks;
        for (int64_t k : n) blocks.push_back(2 * ((k + 255) / 256));
        if (!scales) value_error("%s: no scales", what);
        ae = addresses(what, "scales", *scales, device, blocks, {at::kByte}, true);
    }
    std::vector<Tensor> have;
    if (copies) {
        if (copies->size() != count) value_error("%s: %zu copies for %zu tensors", what, copies->size(), count);
        std::vector<int64_t> k;
        for (size_t i = 0; i < count; ++i)
            if ((*copies)[i]) {
                have.push_back(*(*copies)[i]);
                k.push_back(n[i]);
            }
        const std::vector<void*> at = addresses(what, "copies", have, device, k, {at::kBFloat16}, true);
        size_t j = 0;
        for (size_t i = 0; i < count; ++i) ac.push_back((*copies)[i] ? at[j++] : nullptr);
    }
    if (betas.size() != 2 || !(betas[0] >= 0.0 && betas[0] < 1.0) || !(betas[1] >= 0.0 && betas[1] < 1.0))
        value_error("%s: betas have to be two numbers in [0, 1)", what);
    // (a gradient whose square is nothing in fp32, below 1e-21, then moves p by at most lr * 1e-6, not by lr * g / eps of any size)
    if (!(eps >= 1e-15 && std::isfinite((float)eps))) value_error("%s: eps = %g", what, eps);
    if (!std::isfinite((float)grad_mult)) value_error("%s: grad_mult = %g", what, grad_mult);
    // (all refusals come before the step's number on the GPU moves)
    if (max_workgroups < 0) throw std::runtime_error(std::string(what) + ": max_workgroups = " + std::to_string(max_workgroups));
    const std::vector<float> lrs = scalars(what, "lr", lr, count), wds = scalars(what, "weight_decay", weight_decay, count);
    if (grad_scale) device_scalar(what, "grad_scale", *grad_scale, device, at::kFloat);
    std::vector<int> types;
    for (size_t i = 0; i < count; ++i)
        types.push_back((params[i].scalar_type() == at::kBFloat16 ? 1 : 0) + (grads[i].scalar_type() == at::kBFloat16 ? 2 : 0) +
                        (bits8 && !hold_v ? 4 : 0));
    const c10::DeviceGuard guard(params[0].device());
    void* stream = stream_of(params[0]);
    Tensor bias;
    int64_t number = 0;
    if (THPVariable_Check(step.ptr())) {
        const Tensor counter = THPVariable_Unpack(step.ptr());
        device_scalar(what, "step", counter, device, at::kLong);
        bias = at::empty({4}, params[0].options().dtype(at::kFloat));
        check(odw_adamw_advance(counter.data_ptr<int64_t>(), betas[0], betas[1], bias.data_ptr<float>(), stream), "adamw_advance");
        changed({counter});
    } else {
        const double x = step.cast<double>();
        number = (int64_t)x;
        if (!(x >= 1.0) || (double)number != x) value_error("%s: step = %g (the first one is 1)", what, x);
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
            throw std::runtime_error(std::string(what) + ": a captured step would replay step " + std::to_string(number) +
                                     " for ever: pass `step` as an int64 tensor on the GPU");
    }
    const float* bp = bias.defined() ? bias.data_ptr<float>() : nullptr;
    const float* gs = grad_scale ? grad_scale->data_ptr<float>() : nullptr;
    void* const* cp = ac.empty() ? nullptr : ac.data();
    const int wide = (int)std::min<int64_t>(max_workgroups, INT32_MAX);
    if (bits8)
        check(odw_adamw8((int)count, ap.data(), ag.data(), am.data(), av.data(), (uint8_t* const*)ae.data(), cp, n.data(), types.data(), lrs.data(),
                         wds.data(), betas[0], betas[1], eps, number, bp, gs, (float)grad_mult, (uint32_t)key[0], (uint32_t)key[1], wide, stream), what);
    else
        check(odw_adamw((int)count, ap.data(), ag.data(), am.data(), av.data(), cp, n.data(), types.data(), lrs.data(), wds.data(), betas[0], betas[1], eps,
                        number, bp, gs, (float)grad_mult, wide, stream), what);
    changed(params);
    changed(m);
    changed(v);
    if (bits8) changed(*scales);
    changed(have);
}

// ---- the norm of rows ---------------------------------------------------------------------------------------------------------------

// (rows, D) view with dense columns; a copy only where there is none (or its negation is not in memory yet).
Tensor rows(const Tensor& any, int64_t D) {
    const Tensor t = any.resolve_neg(), r = t.dim() == 2 ? t : t.reshape({-1, D});
    return r.stride(1) == 1 || D == 1 ? r : r.contiguous();
}
bool is_bf16(at::ScalarType t) { return t == at::kBFloat16; }
void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

void check_rows(const char* what, const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
    not_traced(what);
    need_gpu(x);
    if (x.dim() < 1 || x.size(-1) < 1) value_error("%s: x has no columns", what);
    if (x.size(-1) > INT32_MAX) value_error("%s: x has %lld columns", what, (long long)x.size(-1));
    const std::pair<const char*, const Tensor*> all[3] = {
        {"x", &x}, {"weight", weight ? &*weight : nullptr}, {"residual", residual ? &*residual : nullptr}};
    for (const auto& [name, t] : all) {
        if (!t) continue;
        need_gpu(*t);
        if (t->scalar_type() != at::kFloat && t->scalar_type() != at::kBFloat16)
            type_error("%s: %s is %s (torch.float32 | torch.bfloat16)", what, name, name_of(t->scalar_type()).c_str());
        if (t->get_device() != x.get_device())
            value_error("%s: %s is on cuda:%d, x on cuda:%d", what, name, (int)t->get_device(), (int)x.get_device());
    }
    if (weight && (weight->dim() != 1 || weight->size(0) != x.size(-1)))
        value_error("%s: weight has %lld elements in %lld dimensions, x %lld columns", what, (long long)weight->numel(),
                    (long long)weight->dim(), (long long)x.size(-1));
    if (residual && residual->sizes() != x.sizes()) value_error("%s: residual has another shape than x", what);
    if (residual && residual->scalar_type() != x.scalar_type() && residual->scalar_type() != at::kFloat)
        type_error("%s: residual is %s beside x in %s (x's type or torch.float32)", what, name_of(residual->scalar_type()).c_str(),
                   name_of(x.scalar_type()).c_str());
    if (!(eps >= 0.0 && std::isfinite((float)eps))) value_error("%s: eps = %g", what, eps);
}

int types_of(at::ScalarType x, at::ScalarType h, const Tensor& w) {
    return is_bf16(x) + 2 * is_bf16(h) + (w.defined() && is_bf16(w.scalar_type()) ? 4 : 0);
}

// The forward launch into `out` (y, or with `scale` the 8-bit codes); h is undefined without a residual.
Tensor norm_rows(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps, const Tensor& out, const Tensor& rstd,
                 const Tensor& scale) {
    const int64_t D = x.size(-1);
    const Tensor x2 = rows(x, D), r2 = residual ? rows(*residual, D) : Tensor(), w = weight ? weight->resolve_neg().contiguous() : Tensor();
    const Tensor h = residual ? at::empty(x.sizes(), residual->options()) : Tensor();
    const int types = types_of(x.scalar_type(), (residual ? *residual : x).scalar_type(), w);
    const int64_t R = x2.size(0), ldx = x2.stride(0), ldr = residual ? r2.stride(0) : 0;
    if (scale.defined())
        check(odw_rms_norm_fp8(ptr(x2), ldx, ptr(r2), ldr, ptr(w), R, (int)D, (float)eps, ptr(out), (float*)ptr(scale), ptr(h), types,
                               stream_of(x)), "rms_norm_fp8");
    else
        check(odw_rms_norm(ptr(x2), ldx, ptr(r2), ldr, ptr(w), R, (int)D, (float)eps, ptr(out), ptr(h), (float*)ptr(rstd), types,
                           stream_of(x)), "rms_norm");
    return h;
}

// A captured backward pass hands its gradients on: to a leaf's accumulator that an eager graph, still alive, has made on the default
// stream (or to any node of that stream), the engine would make that stream wait for the capture, which it cannot, and the process ends.
// Refused before it does.
void no_default_stream_behind_a_capture() {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    for (size_t i = 0; i < node->num_outputs(); ++i) {
        const auto& edge = node->next_edge(i);
        if (!edge.is_valid() || !node->task_should_compute_output(i)) continue;
        const auto stream = edge.function->stream();
        if (stream && stream->id() == 0)
            throw std::runtime_error("rms_norm: a captured backward pass would reach a node of the default stream: a graph made there before, of the "
                                     "same leaves or of the input, is still alive (let it go, or make it on the capture's stream)");
    }
}

enum { kNeedX = 1, kNeedW = 2, kNeedR = 4, kHasR = 8, kXIsBf16 = 16 };

struct RMSNorm : torch::autograd::Function<RMSNorm> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& residual,
                                                  double eps) {
        const c10::DeviceGuard guard(x.device());
        const Tensor y = at::empty(x.sizes(), x.options()),
                     rstd = at::empty({x.numel() / x.size(-1)}, x.options().dtype(at::kFloat));
        const Tensor h = norm_rows(x, weight, residual, eps, y, rstd, Tensor());
        ctx->save_for_backward({h.defined() ? h : x, weight ? *weight : Tensor(), rstd});
        ctx->set_materialize_grads(false);
        ctx->saved_data["flags"] = (int64_t)((x.requires_grad() ? kNeedX : 0) | (weight && weight->requires_grad() ? kNeedW : 0) |
                                             (residual && residual->requires_grad() ? kNeedR : 0) | (residual ? kHasR : 0) |
                                             (is_bf16(x.scalar_type()) ? kXIsBf16 : 0));
        if (h.defined()) return {y, h};
        return {y};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        no_default_stream_behind_a_capture();
        const int64_t flags = ctx->saved_data["flags"].toInt();
        const auto saved = ctx->get_saved_variables();
        torch::autograd::variable_list out;
        {
            const at::NoGradGuard no_grad;
            out = gradients(flags, saved[0], saved[1], saved[2], grads[0], grads.size() > 1 ? grads[1] : Tensor());
        }
        if (at::GradMode::is_enabled()) {
            // (create_graph: a derivative of these gradients is not to be had, and must not be taken for zero)
            auto error = std::make_shared<torch::autograd::DelayedError>("rms_norm: the gradients cannot be differentiated again", (int64_t)out.size());
            torch::autograd::variable_list held;
            for (const Tensor& t : out) held.push_back(t.defined() ? t.detach().set_requires_grad(true) : t);
            out = (*error)(std::move(held));
        }
        return {out[0], out[1], out[2], Tensor()};
    }

    static torch::autograd::variable_list gradients(int64_t flags, const Tensor& h, const Tensor& weight, const Tensor& rstd,
                                                    const Tensor& dy, const Tensor& dh) {
        const bool need_x = flags & kNeedX, need_w = flags & kNeedW, need_r = flags & kNeedR;
        const at::ScalarType x_type = flags & kXIsBf16 ? at::kBFloat16 : at::kFloat, h_type = flags & kHasR ? h.scalar_type() : x_type;
        if (!dy.defined()) {             // only h was used
            return {need_x && dh.defined() ? dh.to(x_type) : Tensor(), need_w ? at::zeros_like(weight) : Tensor(), need_r ? dh : Tensor()};
        }
        const c10::DeviceGuard guard(h.device());
        const int64_t D = h.size(-1);
        const Tensor h2 = rows(h, D), g2 = rows(dy, D), d2 = dh.defined() ? rows(dh, D) : Tensor(),
                     w = weight.defined() ? weight.resolve_neg().contiguous() : Tensor();
        const int64_t R = h2.size(0);
        const bool mixed = h_type != x_type;
        const Tensor dx = need_x || (need_r && !mixed) ? at::empty(h.sizes(), h.options().dtype(x_type)) : Tensor();
        const Tensor dres = need_r && mixed ? at::empty(h.sizes(), h.options().dtype(h_type)) : Tensor();
        const Tensor dw = need_w ? at::empty({D}, w.options()) : Tensor();
        const int64_t bytes = need_w ? odw_rms_norm_bwd_workspace(R, (int)D) : 0;
        const Tensor ws = bytes ? at::empty({bytes}, h.options().dtype(at::kByte)) : Tensor();
        check(odw_rms_norm_bwd(ptr(g2), g2.stride(0), ptr(d2), d2.defined() ? d2.stride(0) : 0, ptr(h2), h2.stride(0), ptr(w), (const float*)ptr(rstd), R, (int)D,
                               ptr(dx), ptr(dres), ptr(dw), types_of(x_type, h_type, w), ptr(ws), bytes, stream_of(h)), "rms_norm_bwd");
        return {need_x ? dx : Tensor(), dw, need_r ? (mixed ? dres : dx) : Tensor()};
    }
};

py::object rms_norm(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
    check_rows("rms_norm", x, weight, residual, eps);
    // (outputs without a tangent would be taken for constant; no_grad does not end forward mode)
    for (const Tensor* t : {&x, weight ? &*weight : nullptr, residual ? &*residual : nullptr})
        if (t && t->_fw_grad(0).defined()) throw std::runtime_error("rms_norm: has no forward-mode derivative");
    if (at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (residual && residual->requires_grad()))) {
        const auto out = RMSNorm::apply(x, weight, residual, eps);
        return residual ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
    }
    const c10::DeviceGuard guard(x.device());
    const Tensor y = at::empty(x.sizes(), x.options());
    const Tensor h = norm_rows(x, weight, residual, eps, y, Tensor(), Tensor());
    return residual ? py::object(py::make_tuple(y, h)) : py::cast(y);
}

py::object rms_norm_fp8(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
    const at::NoGradGuard no_grad;
    check_rows("rms_norm_fp8", x, weight, residual, eps);
    const c10::DeviceGuard guard(x.device());
    const Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)),
                 scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    const Tensor h = norm_rows(x, weight, residual, eps, q, Tensor(), scale);
    return residual ? py::make_tuple(q, scale, h) : py::make_tuple(q, scale);
}

}  // namespace

PYBIND11_MODULE(_bind, mod) {
    mod.def("adamw", &adamw);
    mod.def("grad_norm", &grad_norm);
    mod.def("clip_grad_norm", &clip_grad_norm);
    mod.def("rms_norm", &rms_norm);
    mod.def("rms_norm_fp8", &rms_norm_fp8);
}
