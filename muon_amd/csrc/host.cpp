// The host side of the operators that run many times a step, as a Python module (muon_amd._native): what bounds a call
// over few or small tensors is the interpreter, not the GPU.  From Python, an AdamW step over 49 vectors took 117 us
// of host time, a routing of 64 tokens forward and backward 115 us; the kernels of either take a few.
//
// Each function takes the common case and says so when it does not: the caller then goes the general way, which
// makes the copies that other strides need and raises what there is to raise.  The kernels are reached through the
// addresses of the C ABI's entry points (bind), so that another build of the library can stand behind them.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/Event.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <array>
#include <cstring>
#include <list>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/muon_amd.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct Api {
    decltype(&muon_amd_last_error) last_error;
    decltype(&muon_amd_residual_norm) residual_norm;
    decltype(&muon_amd_residual_norm_backward) residual_norm_backward;
    decltype(&muon_amd_residual_norm_partials) residual_norm_partials;
    decltype(&muon_amd_route) route;
    decltype(&muon_amd_route_backward) route_backward;
    decltype(&muon_amd_route_partials) route_partials;
    decltype(&muon_amd_validate_grads) validate_grads;
    decltype(&muon_amd_grad_norm) grad_norm;
    decltype(&muon_amd_grad_clip) grad_clip;
    decltype(&muon_amd_validate_adamw_values) validate_adamw_values;
    decltype(&muon_amd_adamw_values) adamw_values;
    decltype(&muon_amd_adamw) adamw;
    int max_width, max_experts, max_k, shared_elems, block_elems, norm_partials;
} api{};

struct LibraryError : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void check(int rc, const char* what) {
    if (rc != MUON_AMD_OK)
        throw LibraryError(std::string(what) + " failed (code " + std::to_string(rc) + "): " + api.last_error());
}

void* current_stream(const c10::Device& device) {
    return c10::hip::getCurrentHIPStream(device.index()).stream();
}

// The current stream as torch's device-independent interface names it.
c10::Stream stream_of(const c10::Device& device) { return c10::impl::VirtualGuardImpl(device.type()).getStream(device); }

bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? MUON_AMD_SRC_BF16 : MUON_AMD_SRC_F32; }
bool taken(const Tensor& t) { return t.is_cuda() && (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16); }

// `t` as rows of `width` elements next to each other (any distance between rows): a view where its strides allow that,
// else a copy.
Tensor rows_of(const Tensor& t, int64_t width) {
    if (t.dim() == 2 && (width == 1 || t.stride(1) == 1)) return t;
    const Tensor r = t.reshape({width ? t.numel() / width : 0, width});
    return width == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

// Gradients of a function whose gradients are not differentiable themselves: asked for a graph, they carry the error.
variable_list once(variable_list grads, const char* message) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = torch::autograd::DelayedError(message, 1)({g})[0];
    return grads;
}

// ---- residual_norm -------------------------------------------------------------------------------------------
struct ResidualTensors {
    Tensor x, block, post, pre, gate, scale;           // the last two may be undefined
};

// The arguments of both directions; `keep` holds the tensors behind the addresses in them.
MuonResidualNorm residual_args(const ResidualTensors& t, double eps, std::vector<Tensor>& keep) {
    const int64_t width = t.x.size(-1);
    const auto hold = [&](Tensor r) -> const Tensor& {
        keep.push_back(std::move(r));
        return keep.back();
    };
    keep.reserve(8);
    MuonResidualNorm a{};
    const Tensor& x = hold(rows_of(t.x, width));
    const Tensor& b = hold(rows_of(t.block, width));
    a.x = x.data_ptr();
    a.b = b.data_ptr();
    a.rows = x.size(0);
    a.ld_x = x.stride(0);
    a.ld_b = b.stride(0);
    a.width = static_cast<int32_t>(width);
    a.post_weight = hold(t.post.contiguous()).data_ptr();
    a.pre_weight = hold(t.pre.contiguous()).data_ptr();
    a.stream_dtype = dtype_of(t.x);
    a.block_dtype = dtype_of(t.block);
    a.weight_dtype = dtype_of(t.post);
    a.eps = static_cast<float>(eps);
    if (t.gate.defined()) {
        const Tensor& g = hold(rows_of(t.gate, t.gate.size(-1)));
        a.gate = g.data_ptr();
        a.ld_gate = g.stride(0);
        a.gate_is_token = t.gate.size(-1) != width;
    }
    if (t.scale.defined()) {
        a.scale = hold(t.scale.contiguous()).data_ptr();
        a.scale_is_one = t.scale.numel() != width;
    }
    return a;
}

std::tuple<Tensor, Tensor, Tensor> residual_forward(const ResidualTensors& t, double eps, bool needed) {
    Tensor h = at::empty(t.x.sizes(), t.x.options()), y = at::empty(t.x.sizes(), t.block.options()), rstd;
    if (t.x.numel() == 0) return {h, y, rstd};
    std::vector<Tensor> keep;
    MuonResidualNorm a = residual_args(t, eps, keep);
    if (needed) rstd = at::empty({a.rows, 2}, t.x.options().dtype(at::kFloat));
    a.h = h.data_ptr();
    a.y = y.data_ptr();
    a.rstd = needed ? rstd.data_ptr<float>() : nullptr;
    const c10::DeviceGuard guard(t.x.device());
    check(api.residual_norm(&a, current_stream(t.x.device())), "residual_norm");
    return {h, y, rstd};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& block, const Tensor& post, const Tensor& pre,
                                 const std::optional<Tensor>& gate, const std::optional<Tensor>& scale, double eps) {
        const ResidualTensors t{x, block, post, pre, gate.value_or(Tensor()), scale.value_or(Tensor())};
        auto [h, y, rstd] = residual_forward(t, eps, true);
        ctx->set_materialize_grads(false);
        ctx->saved_data["eps"] = eps;
        ctx->save_for_backward({t.x, t.block, t.post, t.pre, t.gate, t.scale, rstd});
        return {h, y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list douts) {
        const variable_list saved = ctx->get_saved_variables();
        const ResidualTensors t{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5]};
        const Tensor& rstd = saved[6];
        variable_list grads(7);
        // (edges are counted over the inputs that are tensors)
        const bool nothing = !rstd.defined() || (!douts[0].defined() && !douts[1].defined());
        size_t edge = 0;
        for (int i = 0; i < 6; ++i)
            if (saved[i].defined() && ctx->needs_input_grad(edge++))
                grads[i] = nothing ? at::zeros(saved[i].sizes(), saved[i].options()) : at::empty(saved[i].sizes(), saved[i].options());
        if (!nothing) {
            std::vector<Tensor> keep;
            MuonResidualNorm a = residual_args(t, ctx->saved_data["eps"].toDouble(), keep);
            Tensor dh, dy, partials;
            if (douts[0].defined()) {
                dh = rows_of(douts[0], a.width);
                a.dh = dh.data_ptr();
                a.ld_dh = dh.stride(0);
            }
            if (douts[1].defined()) {
                dy = rows_of(douts[1], a.width);
                a.dy = dy.data_ptr();
                a.ld_dy = dy.stride(0);
            }
            const auto address = [&](int i) { return grads[i].defined() ? grads[i].data_ptr() : nullptr; };
            a.rstd = rstd.data_ptr<float>();
            a.dx = address(0);
            a.db = address(1);
            a.dpost_weight = address(2);
            a.dpre_weight = address(3);
            a.dgate = address(4);
            a.dscale = address(5);
            if (a.dpost_weight || a.dpre_weight || a.dscale) {
                partials = at::empty({api.residual_norm_partials(a.rows, a.width)}, rstd.options());
                a.partials = partials.data_ptr<float>();
            }
            const c10::DeviceGuard guard(t.x.device());
            check(api.residual_norm_backward(&a, current_stream(t.x.device())), "residual_norm_backward");
        }
        return once(std::move(grads), "the gradients of residual_norm are not differentiable");
    }
};

// Whether one of them carries a forward-mode derivative: these functions have none, and must not drop it.
bool any_tangent(std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t && t->_fw_grad(0).defined()) return true;
    return false;
}

bool residual_taken(const Tensor& x, const Tensor& block, const Tensor& post, const Tensor& pre, const std::optional<Tensor>& gate,
                    const std::optional<Tensor>& scale, double eps) {
    if (!taken(x) || x.dim() < 1 || !(eps >= 0.)) return false;
    const int64_t width = x.size(-1);
    for (const Tensor* t : {&block, &post, &pre})
        if (!taken(*t) || t->device() != x.device()) return false;
    if (width > api.max_width || block.sizes() != x.sizes() || (x.scalar_type() == at::kBFloat16 && block.scalar_type() != at::kBFloat16))
        return false;
    if (post.dim() != 1 || pre.dim() != 1 || post.size(0) != width || pre.size(0) != width || post.scalar_type() != pre.scalar_type())
        return false;
    if (scale && (!taken(*scale) || scale->device() != x.device() || scale->dim() > 1 || (scale->numel() != 1 && scale->numel() != width) ||
                  scale->scalar_type() != post.scalar_type()))
        return false;
    if (gate) {
        if (!taken(*gate) || gate->device() != x.device() || gate->scalar_type() != block.scalar_type() || gate->dim() != x.dim()) return false;
        if (gate->size(-1) != width && gate->size(-1) != 1) return false;
        for (int64_t d = 0; d + 1 < x.dim(); ++d)
            if (gate->size(d) != x.size(d)) return false;
    }
    return !any_tangent({&x, &block, &post, &pre, gate ? &*gate : nullptr, scale ? &*scale : nullptr});
}

bool any_requires_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t && t->requires_grad()) return true;
    return false;
}

// None where the arguments are not taken.
std::optional<std::tuple<Tensor, Tensor>> residual_norm(const Tensor& x, const Tensor& block, const Tensor& post, const Tensor& pre,
                                                        const std::optional<Tensor>& gate, const std::optional<Tensor>& scale, double eps) {
    if (!residual_taken(x, block, post, pre, gate, scale, eps)) return std::nullopt;
    const py::gil_scoped_release released;
    if (any_requires_grad({&x, &block, &post, &pre, gate ? &*gate : nullptr, scale ? &*scale : nullptr})) {
        const variable_list out = ResidualNorm::apply(x, block, post, pre, gate, scale, eps);
        return std::make_tuple(out[0], out[1]);
    }
    auto [h, y, rstd] = residual_forward({x, block, post, pre, gate.value_or(Tensor()), scale.value_or(Tensor())}, eps, false);
    return std::make_tuple(h, y);
}

// ---- route_topk ------------------------------------------------------------------------------------------------
struct RouteOut {
    Tensor weights, indices, counts, balance, z, part, lse;
};

MuonRoute route_args(const Tensor& logits, const Tensor& mask, const RouteOut& o, bool normalize, std::vector<Tensor>& keep) {
    keep.push_back(rows_of(logits, logits.size(-1)));
    const Tensor& rows = keep.back();
    MuonRoute a{};
    a.logits = rows.data_ptr();
    a.tokens = rows.size(0);
    a.ld_logits = rows.stride(0);
    a.experts = static_cast<int32_t>(rows.size(1));
    a.dtype = dtype_of(logits);
    if (mask.defined()) {
        keep.push_back(mask.contiguous());
        a.mask = static_cast<const uint8_t*>(keep.back().data_ptr());
    }
    a.weights = o.weights.data_ptr<float>();
    a.indices = o.indices.data_ptr<int32_t>();
    a.counts = o.counts.data_ptr<int32_t>();
    a.part = o.part.data_ptr<float>();
    a.lse = o.lse.data_ptr<float>();
    a.lse_rest = a.lse + a.tokens;
    a.k = static_cast<int32_t>(o.weights.size(-1));
    a.normalize = normalize;
    return a;
}

RouteOut route_forward(const Tensor& logits, int64_t k, const Tensor& mask, bool normalize) {
    const int64_t experts = logits.size(-1), tokens = logits.numel() / experts;
    const auto f32 = logits.options().dtype(at::kFloat), i32 = logits.options().dtype(at::kInt);
    std::vector<int64_t> shape = logits.sizes().vec();
    shape.back() = k;
    RouteOut o;
    o.weights = at::empty(shape, f32);
    o.indices = at::empty(shape, i32);
    if (tokens == 0) {
        o.counts = at::zeros({experts}, i32);
        o.balance = at::zeros({}, f32);
        o.z = at::zeros({}, f32);
        return o;
    }
    o.counts = at::empty({experts}, i32);
    o.balance = at::empty({}, f32);
    o.z = at::empty({}, f32);
    o.part = at::empty({}, f32);
    o.lse = at::empty({2, tokens}, f32);              // and what rounding it left out
    const Tensor partials = at::empty({api.route_partials(tokens, static_cast<int>(experts))}, f32);
    std::vector<Tensor> keep;
    keep.reserve(2);
    MuonRoute a = route_args(logits, mask, o, normalize, keep);
    a.balance = o.balance.data_ptr<float>();
    a.z = o.z.data_ptr<float>();
    a.partials = partials.data_ptr<float>();
    const c10::DeviceGuard guard(logits.device());
    check(api.route(&a, current_stream(logits.device())), "route");
    return o;
}

struct RouteTopk : torch::autograd::Function<RouteTopk> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t k, const std::optional<Tensor>& mask, bool normalize) {
        const Tensor m = mask.value_or(Tensor());
        const RouteOut o = route_forward(logits, k, m, normalize);
        ctx->set_materialize_grads(false);
        ctx->saved_data["normalize"] = normalize;
        ctx->save_for_backward({logits, m, o.weights, o.indices, o.counts, o.part, o.lse});
        ctx->mark_non_differentiable({o.indices, o.counts});
        return {o.weights, o.indices, o.counts, o.balance, o.z};
    }
    static variable_list backward(AutogradContext* ctx, variable_list douts) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor& logits = saved[0];
        const RouteOut o{saved[2], saved[3], saved[4], Tensor(), Tensor(), saved[5], saved[6]};
        Tensor dlogits = at::empty(logits.sizes(), logits.options());
        if (o.lse.defined()) {
            std::vector<Tensor> keep;
            keep.reserve(2);
            MuonRoute a = route_args(logits, saved[1], o, ctx->saved_data["normalize"].toBool(), keep);
            a.dlogits = dlogits.data_ptr();
            Tensor dweights;
            if (douts[0].defined()) {
                dweights = rows_of(douts[0], a.k);
                a.dweights = dweights.data_ptr<float>();
                a.ld_dweights = dweights.stride(0);
            }
            a.dbalance = douts[3].defined() ? douts[3].data_ptr<float>() : nullptr;
            a.dz = douts[4].defined() ? douts[4].data_ptr<float>() : nullptr;
            const c10::DeviceGuard guard(logits.device());
            check(api.route_backward(&a, current_stream(logits.device())), "route_backward");
        }
        return once({dlogits, Tensor(), Tensor(), Tensor()}, "the gradients of route_topk are not differentiable");
    }
};

std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>> route_topk(const Tensor& logits, int64_t k, const std::optional<Tensor>& mask,
                                                                             bool normalize) {
    if (!taken(logits) || logits.dim() < 1 || logits.size(-1) < 1 || logits.size(-1) > api.max_experts || k < 1 ||
        k > std::min<int64_t>(logits.size(-1), api.max_k))
        return std::nullopt;
    if (mask && (mask->scalar_type() != at::kBool || mask->device() != logits.device() ||
                 mask->sizes() != logits.sizes().slice(0, logits.dim() - 1)))
        return std::nullopt;
    if (any_tangent({&logits})) return std::nullopt;
    const py::gil_scoped_release released;
    if (any_requires_grad({&logits})) {
        const variable_list out = RouteTopk::apply(logits, k, mask, normalize);
        return std::make_tuple(out[0], out[1], out[2], out[3], out[4]);
    }
    const RouteOut o = route_forward(logits, k, mask.value_or(Tensor()), normalize);
    return std::make_tuple(o.weights, o.indices, o.counts, o.balance, o.z);
}

// ---- addresses of an optimizer's tensors -------------------------------------------------------------------------
// A parameter that the kernels take as it is: fp32 or bf16 in row-major memory on a GPU, with a gradient alike.
const Tensor* plain_parameter(PyObject* p) {
    if (!THPVariable_Check(p)) return nullptr;
    const Tensor& t = THPVariable_Unpack(p);
    return taken(t) && t.is_contiguous() && t.numel() > 0 ? &t : nullptr;
}
bool plain_gradient(const Tensor& g, const Tensor& p) {
    return g.defined() && g.layout() == at::kStrided && g.scalar_type() == p.scalar_type() && g.device() == p.device() &&
           g.sizes() == p.sizes() && g.is_contiguous();
}

// The state of parameter `p`, or null where it has none or one that is empty.  `at` walks along: states are in the order
// of their first step, as a rule that of the parameters.
PyObject* state_of(const py::dict& state, PyObject* p, Py_ssize_t& at) {
    PyObject *key, *s;
    if (!(PyDict_Next(state.ptr(), &at, &key, &s) && key == p)) {
        s = PyDict_GetItemWithError(state.ptr(), p);
        if (!s) PyErr_Clear();
    }
    return s && PyDict_Check(s) && PyDict_GET_SIZE(s) > 0 ? s : nullptr;
}
// The names of a state's tensors, in the order of a launch's table.
const py::str& state_name(int i) {
    static const py::str* const names = new py::str[4]{py::str("exp_avg"), py::str("exp_avg_sq"), py::str("exp_avg_exponent"),
                                                       py::str("exp_avg_sq_exponent")};
    return names[i];
}
// Tensor i of parameter t's state of `bits` bits, or null where it is not what the kernels take.
const Tensor* state_tensor(PyObject* s, int i, const Tensor& t, int bits) {
    PyObject* const v = PyDict_GetItemWithError(s, state_name(i).ptr());
    if (!v || !THPVariable_Check(v)) {
        PyErr_Clear();
        return nullptr;
    }
    const Tensor& x = THPVariable_Unpack(v);
    if (x.scalar_type() != (bits == 8 ? at::kByte : at::kFloat) || x.device() != t.device() || !x.is_contiguous()) return nullptr;
    if (i < 2) return x.sizes() == t.sizes() ? &x : nullptr;
    return x.dim() == 1 && x.size(0) == (t.numel() + api.shared_elems - 1) / api.shared_elems ? &x : nullptr;
}

// The rows of an AdamW launch over a fixed list of parameters.  collect() reads the addresses of parameters, gradients and
// states as they are now; nothing is taken from an earlier step but the answer to whether they are the same.
class AdamWTable {
   public:
    // device: the index of the GPU that the launch runs on (-1: whichever the tensors are on).
    AdamWTable(std::vector<int64_t> numels, std::vector<int> dtypes, int bits, int device)
        : numels_(std::move(numels)), dtypes_(std::move(dtypes)), bits_(bits), device_(device), columns_(bits == 8 ? 6 : 4),
          rows_(numels_.size() * columns_), now_(rows_.size()) {}

    // The step these parameters are about to take (one for all), or -1: not the common case.
    int64_t collect(const py::list& params, const py::dict& state) {
        dicts_.clear();
        const size_t n = numels_.size();
        if (static_cast<size_t>(PyList_GET_SIZE(params.ptr())) != n) return -1;
        int64_t step = -1;
        std::optional<c10::Device> device;
        Py_ssize_t at = 0;
        for (size_t i = 0; i < n; ++i) {
            PyObject* const p = PyList_GET_ITEM(params.ptr(), i);
            const Tensor* const t = plain_parameter(p);
            if (!t || t->numel() != numels_[i] || dtype_of(*t) != dtypes_[i]) return -1;
            if (!device) device = t->device();
            if (t->device() != *device || (device_ >= 0 && device->index() != device_) || !plain_gradient(t->grad(), *t)) return -1;
            PyObject* const s = state_of(state, p, at);
            if (!s) return -1;
            int64_t* const row = &now_[i * columns_];
            row[0] = reinterpret_cast<int64_t>(t->data_ptr());
            row[1] = reinterpret_cast<int64_t>(t->grad().data_ptr());
            for (int c = 2; c < columns_; ++c) {
                const Tensor* const x = state_tensor(s, c - 2, *t, bits_);
                if (!x) return -1;
                row[c] = reinterpret_cast<int64_t>(x->data_ptr());
            }
            PyObject* const count = PyDict_GetItemWithError(s, step_.ptr());
            if (!count || !PyLong_Check(count)) {
                PyErr_Clear();
                return -1;
            }
            const int64_t next = PyLong_AsLongLong(count) + 1;
            if (step >= 0 && next != step) return -1;
            step = next;
            dicts_.push_back(py::reinterpret_borrow<py::dict>(s));
        }
        if (now_ != rows_) {
            rows_ = now_;
            ++version_;
        }
        return step;
    }
    // Puts the addresses into the rows of the launch's table, which begin with them (valid after collect).
    void write(const py::buffer& table) const {
        const py::buffer_info rows = table.request(/*writable=*/true);
        const size_t size = columns_ * sizeof(int64_t), stride = static_cast<size_t>(rows.itemsize);
        if (rows.ndim != 1 || static_cast<size_t>(rows.size) != numels_.size() || stride < size || rows.strides[0] != rows.itemsize)
            throw py::value_error("not this list's table");
        for (size_t i = 0; i < numels_.size(); ++i)
            std::memcpy(static_cast<char*>(rows.ptr) + i * stride, &rows_[i * columns_], size);
    }
    int64_t version() const { return version_; }
    // Writes the new step count to the states that collect() saw.
    void bump(int64_t step) {
        const py::int_ value(step);
        for (const py::dict& d : dicts_)
            if (PyDict_SetItem(d.ptr(), step_.ptr(), value.ptr()) != 0) throw py::error_already_set();
        dicts_.clear();
    }

   private:
    const std::vector<int64_t> numels_;
    const std::vector<int> dtypes_;
    const int bits_, device_, columns_;
    std::vector<int64_t> rows_, now_;
    int64_t version_ = 0;
    std::vector<py::dict> dicts_;
    const py::str step_{"step"};
};

// The AdamW launch on the current stream of a device (addresses as numbers; hyper: lr, 1 - lr weight_decay, 1 - beta1,
// 1 - beta2, eps, 1 - beta1^t, 1 - beta2^t, t).  Whether a HIP graph records it.
bool adamw_launch(int device, uintptr_t descs, uintptr_t prefix, int n, int blocks, int dtype, int bits, const std::array<double, 8>& hyper,
                  uintptr_t grad_scale, uintptr_t scalars) {
    const auto f = [&](int i) { return static_cast<float>(hyper[i]); };
    check(api.adamw(reinterpret_cast<const MuonAdamWDesc*>(descs), reinterpret_cast<const int32_t*>(prefix), n, blocks, dtype, bits, f(0), f(1),
                    f(2), f(3), f(4), f(5), f(6), static_cast<uint32_t>(hyper[7]), reinterpret_cast<const float*>(grad_scale),
                    reinterpret_cast<const float*>(scalars), c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(device)).stream()),
          "adamw");
    return capturing();
}

// The memory of tables that a captured HIP graph reads: a replay holds their addresses for as long as the program keeps it,
// whatever becomes of the tables' owners.  (Never destroyed: the process ends with it.)
std::vector<Tensor>& tables_of_graphs() {
    static auto* const kept = new std::vector<Tensor>;
    return *kept;
}

// A table of descriptors and its block prefix on the device.  A table is never rewritten: other contents get memory of
// their own, so a launch on one stream cannot see what a call on another stream uploads.
class Table {
   public:
    template <typename D>
    void upload(const std::vector<D>& descs, const c10::Device& device) {
        if (capturing()) throw LibraryError("tensors that no call has seen before cannot be uploaded while a HIP graph is captured: make the call once before");
        captured_ = false;
        std::vector<int32_t> prefix(descs.size() + 1, 0);
        for (size_t i = 0; i < descs.size(); ++i)
            prefix[i + 1] = prefix[i] + static_cast<int32_t>((descs[i].numel + api.block_elems - 1) / api.block_elems);
        check(validator<D>()(descs.data(), static_cast<int>(descs.size()), prefix.data()), "validate");
        const size_t first = descs.size() * sizeof(D), size = first + prefix.size() * sizeof(int32_t);
        Tensor host = at::empty({static_cast<int64_t>(size)}, at::TensorOptions().dtype(at::kByte).pinned_memory(true));
        std::memcpy(host.data_ptr(), descs.data(), first);
        std::memcpy(static_cast<char*>(host.data_ptr()) + first, prefix.data(), prefix.size() * sizeof(int32_t));
        memory_ = host.to(device, /*non_blocking=*/true);
        prefix_ = first;
        n_ = static_cast<int>(descs.size());
        blocks_ = prefix.back();
        uploaded_ = c10::Event(device.type());
        uploaded_.record(stream_of(device));
    }
    // Before a launch on the current stream: its table is there, and stays while it runs.
    // (What a HIP graph records cannot wait for an event from outside of it: a caller that captures has made the call
    // before.  The graph keeps the table's address: from then on its memory is not given back.)
    void use(const c10::Device& device) {
        if (capturing()) {
            if (!captured_) tables_of_graphs().push_back(memory_);
            captured_ = true;
            return;
        }
        const c10::Stream stream = stream_of(device);
        uploaded_.block(stream);
        memory_.record_stream(stream);
    }
    template <typename D>
    const D* descs() const { return static_cast<const D*>(memory_.data_ptr()); }
    const int32_t* prefix() const { return reinterpret_cast<const int32_t*>(static_cast<const char*>(memory_.data_ptr()) + prefix_); }
    int size() const { return n_; }
    int blocks() const { return blocks_; }
    bool captured() const { return captured_; }

   private:
    template <typename D>
    static auto validator() {
        if constexpr (std::is_same_v<D, MuonGradDesc>) return api.validate_grads;
        else return api.validate_adamw_values;
    }
    Tensor memory_;
    size_t prefix_ = 0;
    int n_ = 0, blocks_ = 0;
    bool captured_ = false;
    c10::Event uploaded_{c10::DeviceType::CUDA};
};

struct GradTable {
    c10::Device device;
    std::vector<MuonGradDesc> descs;
    bool overlap;                          // of gradients with each other
    Table table;
};
bool overlapping(const std::vector<MuonGradDesc>& descs) {
    std::vector<std::pair<uintptr_t, uintptr_t>> ranges;
    for (const MuonGradDesc& d : descs) {
        const uintptr_t begin = reinterpret_cast<uintptr_t>(d.grad);
        ranges.emplace_back(begin, begin + d.numel * (d.dtype == MUON_AMD_SRC_BF16 ? 2 : 4));
    }
    std::sort(ranges.begin(), ranges.end());
    for (size_t i = 1; i < ranges.size(); ++i)
        if (ranges[i].first < ranges[i - 1].second) return true;
    return false;
}
// The tables of the last gradient lists, newest first (calls hold the interpreter's lock).
std::list<GradTable>& grad_tables() {
    static std::list<GradTable> tables;
    return tables;
}
constexpr size_t GRAD_TABLES = 16;

// (norm, coefficient) of these gradients (dense fp32 or bf16 tensors of one device, row-major, not empty).
std::tuple<Tensor, Tensor> clip_tensors(const std::vector<const Tensor*>& grads, double max_norm, bool in_place) {
    const c10::Device device = grads[0]->device();
    std::vector<MuonGradDesc> descs(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) descs[i] = {grads[i]->data_ptr(), grads[i]->numel(), dtype_of(*grads[i]), 0};
    const c10::DeviceGuard guard(device);
    auto& tables = grad_tables();
    const auto same = [&](const GradTable& t) {
        return t.device == device && t.descs.size() == descs.size() &&
               std::memcmp(t.descs.data(), descs.data(), descs.size() * sizeof(MuonGradDesc)) == 0;
    };
    const auto found = std::find_if(tables.begin(), tables.end(), same);
    if (found != tables.end()) {
        tables.splice(tables.begin(), tables, found);
    } else {
        const bool overlap = overlapping(descs);
        GradTable fresh{device, std::move(descs), overlap, {}};
        fresh.table.upload(fresh.descs, device);
        tables.push_front(std::move(fresh));
        size_t others = 0;
        for (auto i = tables.begin(); i != tables.end();)
            i = !i->table.captured() && ++others > GRAD_TABLES ? tables.erase(i) : std::next(i);
    }
    if (in_place && tables.front().overlap) throw py::value_error("gradients that share memory cannot be scaled in place");
    Table& table = tables.front().table;
    const auto options = at::TensorOptions().device(device);
    const Tensor out = at::empty({2}, options.dtype(at::kFloat));
    const Tensor partials = at::empty({std::min(table.blocks(), api.norm_partials)}, options.dtype(at::kDouble));
    table.use(device);
    check((in_place ? api.grad_clip : api.grad_norm)(table.descs<MuonGradDesc>(), table.prefix(), table.size(), table.blocks(),
                                                     partials.data_ptr<double>(), static_cast<float>(max_norm), out.data_ptr<float>(),
                                                     current_stream(device)),
          in_place ? "grad_clip" : "grad_norm");
    return {out.select(0, 0), out.select(0, 1)};
}

// The same for the gradients of a list of parameters; None: not the common case (other strides, types or devices, a
// parameter that is in the list twice, no gradient at all).
std::optional<std::tuple<Tensor, Tensor>> clip(const py::list& params, double max_norm, bool in_place) {
    std::vector<const Tensor*> grads;
    std::vector<const void*> seen;
    const Py_ssize_t n = PyList_GET_SIZE(params.ptr());
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* const p = PyList_GET_ITEM(params.ptr(), i);
        if (!THPVariable_Check(p)) return std::nullopt;
        const Tensor& g = THPVariable_Unpack(p).grad();
        if (!g.defined()) continue;
        if (!taken(g) || g.layout() != at::kStrided || !g.is_contiguous() || g.numel() == 0 ||
            (!grads.empty() && g.device() != grads[0]->device()))
            return std::nullopt;
        grads.push_back(&g);
        seen.push_back(p);
    }
    std::sort(seen.begin(), seen.end());
    if (grads.empty() || std::adjacent_find(seen.begin(), seen.end()) != seen.end()) return std::nullopt;
    return clip_tensors(grads, max_norm, in_place);
}
std::tuple<Tensor, Tensor> clip_list(const std::vector<Tensor>& grads, double max_norm, bool in_place) {
    std::vector<const Tensor*> pointers;
    for (const Tensor& g : grads) {
        TORCH_CHECK(taken(g) && g.is_contiguous() && g.numel() > 0 && g.device() == grads[0].device(), "not a plain gradient");
        pointers.push_back(&g);
    }
    return clip_tensors(pointers, max_norm, in_place);
}

// The launch that turns 8-bit states into numbers, for tensors of one device: rows of {exp_avg, exp_avg_sq, their
// exponents, the two bf16 tensors that take the values}, whose sizes and types the caller has checked.
class ValueTable {
   public:
    void run(const std::vector<std::vector<Tensor>>& rows) {
        std::vector<MuonAdamWValuesDesc> descs;
        for (const auto& r : rows) add(descs, {&r[0], &r[1], &r[2], &r[3], &r[4], &r[5]});
        launch(std::move(descs), rows[0][0].device());
    }
    // The same for the parameters that have a state, into `out` (pairs, in their order); false: not the common case.
    bool run_plain(const py::list& params, const py::dict& state, const py::list& out) {
        std::vector<MuonAdamWValuesDesc> descs;
        std::optional<c10::Device> device;
        Py_ssize_t at = 0;
        const Py_ssize_t n = PyList_GET_SIZE(params.ptr());
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* const p = PyList_GET_ITEM(params.ptr(), i);
            PyObject* const s = state_of(state, p, at);
            if (!s) continue;
            const Tensor* const t = plain_parameter(p);
            if (!t || (device && t->device() != *device) || static_cast<Py_ssize_t>(descs.size()) >= PyList_GET_SIZE(out.ptr())) return false;
            device = t->device();
            PyObject* const pair = PyList_GET_ITEM(out.ptr(), descs.size());
            if (!PyTuple_Check(pair) || PyTuple_GET_SIZE(pair) != 2) return false;
            std::array<const Tensor*, 6> row;
            for (int c = 0; c < 4; ++c)
                if (!(row[c] = state_tensor(s, c, *t, 8))) return false;
            for (int c = 0; c < 2; ++c) {
                PyObject* const v = PyTuple_GET_ITEM(pair, c);
                if (!THPVariable_Check(v)) return false;
                const Tensor& x = THPVariable_Unpack(v);
                if (x.scalar_type() != at::kBFloat16 || x.numel() != t->numel() || x.device() != *device || !x.is_contiguous()) return false;
                row[4 + c] = &x;
            }
            add(descs, row);
        }
        if (descs.empty() || static_cast<Py_ssize_t>(descs.size()) != PyList_GET_SIZE(out.ptr())) return false;
        launch(std::move(descs), *device);
        return true;
    }

   private:
    static void add(std::vector<MuonAdamWValuesDesc>& descs, const std::array<const Tensor*, 6>& r) {
        const auto bytes = [&](int c) { return static_cast<const uint8_t*>(r[c]->data_ptr()); };
        descs.push_back({bytes(0), bytes(1), bytes(2), bytes(3), static_cast<uint16_t*>(r[4]->data_ptr()),
                         static_cast<uint16_t*>(r[5]->data_ptr()), r[0]->numel()});
    }
    void launch(std::vector<MuonAdamWValuesDesc> descs, const c10::Device& device) {
        const c10::DeviceGuard guard(device);
        if (descs.size() != descs_.size() || std::memcmp(descs.data(), descs_.data(), descs.size() * sizeof(descs[0])) != 0) {
            table_.upload(descs, device);
            descs_ = std::move(descs);
        }
        table_.use(device);
        check(api.adamw_values(table_.descs<MuonAdamWValuesDesc>(), table_.prefix(), table_.size(), table_.blocks(), current_stream(device)),
              "adamw_values");
    }
    std::vector<MuonAdamWValuesDesc> descs_;
    Table table_;
};

void bind(const py::dict& addresses, const py::object& error) {
    const auto get = [&](auto& f, const char* name) {
        f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(addresses[name].cast<uintptr_t>());
    };
    get(api.last_error, "muon_amd_last_error");
    get(api.residual_norm, "muon_amd_residual_norm");
    get(api.residual_norm_backward, "muon_amd_residual_norm_backward");
    get(api.residual_norm_partials, "muon_amd_residual_norm_partials");
    get(api.route, "muon_amd_route");
    get(api.route_backward, "muon_amd_route_backward");
    get(api.route_partials, "muon_amd_route_partials");
    get(api.validate_grads, "muon_amd_validate_grads");
    get(api.grad_norm, "muon_amd_grad_norm");
    get(api.grad_clip, "muon_amd_grad_clip");
    get(api.validate_adamw_values, "muon_amd_validate_adamw_values");
    get(api.adamw_values, "muon_amd_adamw_values");
    get(api.adamw, "muon_amd_adamw");
    const auto number = [&](const char* name) {
        int (*f)(void);
        get(f, name);
        return f();
    };
    api.max_width = number("muon_amd_residual_norm_max_width");
    api.max_experts = number("muon_amd_route_max_experts");
    api.max_k = number("muon_amd_route_max_k");
    api.shared_elems = number("muon_amd_adamw_shared_elems");
    api.block_elems = number("muon_amd_elementwise_block_elems");
    api.norm_partials = number("muon_amd_grad_norm_partials");
    const auto same = [&](const char* name, size_t size) {
        size_t (*f)(void);
        get(f, name);
        if (f() != size) throw std::runtime_error(std::string(name) + " differs between the library and this module: build both again");
    };
    same("muon_amd_sizeof_residual_norm", sizeof(MuonResidualNorm));
    same("muon_amd_sizeof_route", sizeof(MuonRoute));
    same("muon_amd_sizeof_grad_desc", sizeof(MuonGradDesc));
    same("muon_amd_sizeof_adamw_values_desc", sizeof(MuonAdamWValuesDesc));
    static PyObject* raised;
    raised = error.inc_ref().ptr();
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const LibraryError& e) {
            PyErr_SetString(raised, e.what());
        }
    });
}

}  // namespace

PYBIND11_MODULE(_native, m) {
    m.def("bind", &bind);
    m.def("abi_version", [] { return MUON_AMD_ABI_VERSION; });
    m.def("residual_norm", &residual_norm);
    m.def("route_topk", &route_topk);
    m.def("adamw_launch", &adamw_launch);
    m.def("clip", &clip);
    m.def("clip_list", &clip_list);
    m.def("clear_tables", [] { grad_tables().clear(); });
    m.def("tables_of_graphs", [] { return tables_of_graphs().size(); });
    py::class_<ValueTable>(m, "ValueTable").def(py::init<>()).def("run", &ValueTable::run).def("run_plain", &ValueTable::run_plain);
    py::class_<AdamWTable>(m, "AdamWTable")
        .def(py::init<std::vector<int64_t>, std::vector<int>, int, int>(), py::arg("numels"), py::arg("dtypes"), py::arg("bits"), py::arg("device") = -1)
        .def("collect", &AdamWTable::collect)
        .def("write", &AdamWTable::write)
        .def_property_readonly("version", &AdamWTable::version)
        .def("bump", &AdamWTable::bump);
}
