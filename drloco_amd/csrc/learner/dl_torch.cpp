// dl_torch.cpp -- the learner's operators on torch tensors: argument checks, allocation from torch's allocator, the current
// stream, autograd; everything else is the C-ABI of include/drloco_learner.h.  A rollout's backward pass runs on autograd's own
// thread: here it needs no interpreter lock (in Python the same pass took 60 us longer than its kernels).
//
// A function returns None where its arguments are not what it takes; the Python wrappers say what is wrong with them.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "drloco_learner.h"

namespace {

using at::Tensor;
typedef std::optional<Tensor> Maybe;

int type_of(at::ScalarType t) { return t == at::kFloat ? DL_F32 : t == at::kBFloat16 ? DL_BF16 : t == at::kHalf ? DL_F16 : -1; }
const void* ptr(const Maybe& t) { return t ? t->data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
struct Failed : std::runtime_error { using std::runtime_error::runtime_error; };          // DrlocoError in Python
int64_t check(int64_t rc) {
    if (rc < 0) throw Failed("drloco_learner error " + std::to_string(rc) + ": " + dl_learner_last_error());
    return rc;
}
Tensor floats(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor bytes(const Tensor& like, int64_t n) { return at::empty({n}, like.options().dtype(at::kByte)); }
void written(const Tensor& t) { if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }          // behind torch's back: its version counter has to move

// ---- gated memory ----
bool memory_takes(const Tensor& x, const Tensor& gate, const Maybe& starts, const Maybe& state, int64_t axes) {
    if (!x.is_cuda() || x.dim() != axes || type_of(x.scalar_type()) < 0) return false;
    if (gate.scalar_type() != x.scalar_type() || gate.sizes() != x.sizes() || gate.device() != x.device()) return false;
    if (starts && ((starts->scalar_type() != at::kByte && starts->scalar_type() != at::kBool) || starts->sizes() != x.sizes().slice(0, axes - 1) || starts->device() != x.device())) return false;
    return !state || (state->scalar_type() == at::kFloat && state->sizes() == x.sizes().slice(axes - 2) && state->device() == x.device());
}

// A forward-mode derivative would be lost without a word: there is no rule for it.
bool has_tangent(const Tensor& t) { return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined(); }

// The last axis contiguous, walkers near enough for the kernels' 32-bit row offsets.
Tensor rows(const Tensor& t) {
    const int64_t D = t.size(-1), N = t.size(-2);
    if (t.stride(-1) != 1 && D > 1) return t.contiguous();
    if (N > 1 && t.stride(-2) > 2000000 && t.stride(-2) >= ((int64_t)1 << 29) / std::min<int64_t>(N, 256 / D + 2)) return t.contiguous();
    return t;
}

dl_memory_shape memory_shape(const Tensor& x, const Tensor& gate, const Maybe& starts, const Maybe& grad) {
    dl_memory_shape s{};
    s.T = x.size(0); s.N = x.size(1); s.D = x.size(2);
    s.x_t = x.stride(0); s.x_n = x.stride(1);
    s.gate_t = gate.stride(0); s.gate_n = gate.stride(1);
    if (starts) { s.starts_t = starts->stride(0); s.starts_n = starts->stride(1); }
    if (grad) { s.grad_t = grad->stride(0); s.grad_n = grad->stride(1); }
    s.dtype = type_of(x.scalar_type());
    return s;
}

std::tuple<Tensor, Tensor, Tensor> memory_forward(const Tensor& x, const Tensor& gate, const Maybe& starts, const Maybe& state, bool marked) {
    const c10::DeviceGuard guard(x.device());
    const dl_memory_shape s = memory_shape(x, gate, starts, std::nullopt);
    Tensor h = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)), last = floats(x, {s.N, s.D}), marks, work;
    if (marked) marks = floats(x, {(s.T + DL_MEMORY_MARK - 1) / DL_MEMORY_MARK, s.N, s.D});
    const int64_t size = check(dl_memory_workspace_bytes(&s));
    if (size) work = bytes(x, size);
    check(dl_memory_forward(&s, x.data_ptr(), gate.data_ptr(), (const uint8_t*)ptr(starts), (const float*)ptr(state), h.data_ptr(), last.data_ptr<float>(),
                            marked ? marks.data_ptr<float>() : nullptr, size ? work.data_ptr() : nullptr, stream_of(x)));
    return {h, last, marks};
}

struct GatedMemory : torch::autograd::Function<GatedMemory> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Maybe& starts, const Maybe& state) {
        auto [h, last, marks] = memory_forward(x, gate, starts, state, true);
        ctx->save_for_backward({x, gate, starts ? *starts : Tensor(), marks});
        ctx->saved_data["dstate"] = state && state->requires_grad();
        ctx->set_materialize_grads(false);
        return {h, last};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &gate = saved[1], &marks = saved[3];
        const Maybe starts = saved[2].defined() ? Maybe(saved[2]) : std::nullopt;
        std::vector<Tensor> out;
        {
            const at::NoGradGuard no_grad;
            const c10::DeviceGuard guard(x.device());
            const Maybe gh = grads[0].defined() ? Maybe(rows(grads[0])) : std::nullopt, gl = grads[1].defined() ? Maybe(grads[1].contiguous()) : std::nullopt;
            const dl_memory_shape s = memory_shape(x, gate, starts, gh);
            const auto plain = x.options().memory_format(at::MemoryFormat::Contiguous);
            out = {at::empty(x.sizes(), plain), at::empty(x.sizes(), plain)};
            if (ctx->saved_data["dstate"].toBool()) out.push_back(floats(x, {s.N, s.D}));
            const int64_t size = check(dl_memory_workspace_bytes(&s));
            Tensor work;
            if (size) work = bytes(x, size);
            check(dl_memory_backward(&s, x.data_ptr(), gate.data_ptr(), (const uint8_t*)ptr(starts), marks.data_ptr<float>(), ptr(gh), (const float*)ptr(gl), out[0].data_ptr(), out[1].data_ptr(),
                                     out.size() > 2 ? out[2].data_ptr<float>() : nullptr, size ? work.data_ptr() : nullptr, stream_of(x)));
        }
        if (at::GradMode::is_enabled())          // create_graph: a second differentiation is an error, not a zero
            out = (*std::make_shared<torch::autograd::DelayedError>("gated_memory can be differentiated once only", (int64_t)out.size()))(std::move(out));
        return {out[0], out[1], Tensor(), out.size() > 2 ? out[2] : Tensor()};
    }
};

py::object gated_memory(const Tensor& x_, const Tensor& gate_, Maybe starts, Maybe state) {
    if (!memory_takes(x_, gate_, starts, state, 3) || has_tangent(x_) || has_tangent(gate_) || (state && has_tangent(*state))) return py::none();
    if (x_.numel() == 0) return py::cast(std::make_tuple(x_.clone(), state ? state->clone() : at::zeros({x_.size(1), x_.size(2)}, x_.options().dtype(at::kFloat))));
    const Tensor x = rows(x_), gate = rows(gate_);
    if (starts && starts->scalar_type() == at::kBool) starts = starts->view(at::kByte);
    if (state) state = state->contiguous();
    if (at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || (state && state->requires_grad()))) {
        auto out = GatedMemory::apply(x, gate, starts, state);
        return py::cast(std::make_tuple(out[0], out[1]));
    }
    auto [h, last, marks] = memory_forward(x, gate, starts, state, false);
    return py::cast(std::make_tuple(h, last));
}

std::pair<const char*, const char*> extent(const Tensor& t) {
    int64_t reach = 0;
    for (int64_t d = 0; d < t.dim(); ++d) reach += (t.size(d) - 1) * t.stride(d);
    const char* p = (const char*)t.data_ptr();
    return {p, p + (reach + 1) * t.element_size()};
}
bool apart(const Tensor& a, const Tensor& b) {
    if (!a.numel() || !b.numel()) return true;
    const auto p = extent(a), q = extent(b);
    return p.second <= q.first || q.second <= p.first;
}
bool destination(const Tensor& t, const Tensor& like, at::ScalarType type) { return t.scalar_type() == type && t.sizes() == like.sizes() && t.device() == like.device() && t.is_contiguous(); }

py::object gated_memory_step(const Tensor& x_, const Tensor& gate_, const Tensor& state_, const Maybe& starts, const Maybe& out_, const Maybe& state_out_) {
    const at::NoGradGuard no_grad;
    if (!memory_takes(x_, gate_, starts, state_, 2)) return py::none();
    Tensor h, last;
    if (out_) {
        h = *out_;
        if (!destination(h, x_, x_.scalar_type()) || !apart(h, x_) || !apart(h, gate_) || !apart(h, state_) || (starts && !apart(h, *starts))) return py::none();
    } else h = at::empty(x_.sizes(), x_.options().memory_format(at::MemoryFormat::Contiguous));
    if (state_out_) {
        last = *state_out_;
        const bool same = last.data_ptr() == state_.data_ptr() && state_.is_contiguous();
        if (!destination(last, x_, at::kFloat) || !apart(last, x_) || !apart(last, gate_) || !apart(last, h) || (starts && !apart(last, *starts)) || !(same || apart(last, state_))) return py::none();
    } else last = floats(x_, x_.sizes());
    if (x_.numel()) {
        const c10::DeviceGuard guard(x_.device());
        const Tensor x = rows(x_), gate = rows(gate_), state = state_.contiguous();
        dl_memory_shape s{};
        s.T = 1; s.N = x.size(0); s.D = x.size(1);
        s.x_n = x.stride(0); s.gate_n = gate.stride(0);
        if (starts) s.starts_n = starts->stride(0);
        s.dtype = type_of(x.scalar_type());
        check(dl_memory_step(&s, x.data_ptr(), gate.data_ptr(), (const uint8_t*)ptr(starts), state.data_ptr<float>(), h.data_ptr(), last.data_ptr<float>(), stream_of(x)));
        if (out_) written(h);
        if (state_out_) written(last);
    }
    return py::cast(std::make_tuple(h, last));
}

// ---- orthogonalised updates: the wrappers have checked everything; out and momentum_out are contiguous ----
Tensor stacked(const Tensor& t_) {
    const Tensor t = t_.stride(-1) != 1 && t_.size(-1) > 1 ? t_.contiguous() : t_;
    return t.dim() == 2 ? t.unsqueeze(0) : t.dim() == 3 ? t : t.reshape({-1, t.size(-2), t.size(-1)});
}

void orth_update(const Tensor& grad, const Maybe& momentum, const Maybe& momentum_out, const Maybe& weight, const Tensor& out, int64_t steps, double a, double b, double c, double beta, bool nesterov,
                 double keep, double gain) {
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(grad.device());
    const Tensor g = stacked(grad), o = stacked(out);
    Tensor m, mo, w;
    dl_orth_shape s{};
    s.batch = g.size(0); s.rows = g.size(1); s.cols = g.size(2);
    s.grad_b = g.stride(0); s.grad_r = g.stride(1); s.grad_type = type_of(g.scalar_type());
    s.out_b = o.stride(0); s.out_r = o.stride(1); s.out_type = type_of(o.scalar_type());
    if (momentum) {
        m = stacked(*momentum); mo = stacked(*momentum_out);
        s.momentum_b = m.stride(0); s.momentum_r = m.stride(1);
        s.momentum_out_b = mo.stride(0); s.momentum_out_r = mo.stride(1);
    }
    if (weight) {
        w = stacked(*weight);
        s.weight_b = w.stride(0); s.weight_r = w.stride(1); s.weight_type = type_of(w.scalar_type());
    }
    s.a = a; s.b = b; s.c = c; s.beta = beta; s.weight_keep = keep; s.gain = gain;
    s.steps = (int32_t)steps; s.nesterov = nesterov;
    const int64_t size = check(dl_orth_workspace_bytes(&s));
    Tensor work;
    if (size) work = bytes(g, size);
    check(dl_orth_update(&s, g.data_ptr(), momentum ? m.data_ptr<float>() : nullptr, momentum ? mo.data_ptr<float>() : nullptr, weight ? w.data_ptr() : nullptr, o.data_ptr(), size ? work.data_ptr() : nullptr, stream_of(g)));
    written(out);
    if (momentum) written(*momentum_out);
}

}  // namespace

PYBIND11_MODULE(dl_learner_torch, m) {
    py::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failed& e) {
            PyErr_SetString(py::module_::import("drloco_amd.lib").attr("DrlocoError").ptr(), e.what());
        }
    });
    m.def("gated_memory", &gated_memory);
    m.def("gated_memory_step", &gated_memory_step);
    m.def("orth_update", &orth_update);
}
