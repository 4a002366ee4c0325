// Binding of the memory operators (include/nesle_memory.h) to PyTorch tensors
// and autograd: argument checks, output allocation and the backward nodes of
// nesle_amd/memory.py, which documents the calls.  In C++ because acting calls
// them for one token at a time and autograd runs a backward on a thread of its
// own: the same work in Python took 15 us a call and 80 us a backward, several
// times the kernels.
#include <ATen/ATen.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <limits>
#include <optional>
#include <sstream>
#include <string>

#include "../../include/nesle_memory.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

namespace {

// ---- refusals ------------------------------------------------------------------

std::string shown(const Tensor& t) {
    std::ostringstream s;
    s << "shape " << t.sizes() << ", " << t.scalar_type() << " on " << t.device() << ", strides " << t.strides();
    return s.str();
}

[[noreturn]] void refuse(const char* who, const char* name, const std::string& want, const Tensor& got) {
    throw py::value_error(std::string(who) + ": " + name + " must be " + want + ", got " + shown(got));
}

bool given(const MaybeTensor& t) { return t.has_value() && t->defined(); }
Tensor some(const MaybeTensor& t) { return t.value_or(Tensor()); }

// What a call's tensors have in common: the first of them says it.
struct Common {
    const char* who;
    at::ScalarType type;
    at::Device device;
    int64_t lead;              // leading dimensions: [N] or [T, N]
    at::IntArrayRef sizes;     // of the first tensor
    int64_t steps() const { return lead == 2 ? sizes[0] : 1; }
    int64_t batch() const { return sizes[lead - 1]; }
};

// The C entries take sizes of 32 bits, and have limits of their own below that.
void check_sizes(const char* who, const char* name, const Tensor& t) {
    for (const int64_t n : t.sizes())
        if (n > std::numeric_limits<uint32_t>::max()) refuse(who, name, "of sizes below 2^32", t);
}

Common common_of(const char* who, const Tensor& q, int64_t least, int64_t most) {
    check_sizes(who, "q", q);
    const int64_t lead = q.dim() - 2;
    if (!q.is_cuda() || (q.scalar_type() != at::kFloat && q.scalar_type() != at::kBFloat16) || lead < least ||
        lead > most || q.stride(-1) != 1)
        refuse(who, "q", std::string("a float32 or bfloat16 GPU tensor ") +
               (least == most ? (least == 1 ? "[N, heads, dim]" : "[T, N, heads, dim]") : "[N, heads, dim] or [T, N, heads, dim]") +
               ", elements of a head next to each other", q);
    return {who, q.scalar_type(), q.device(), lead, q.sizes()};
}

// [lead..., heads, dim], elements of a head next to each other.
void check_heads(const Common& c, const Tensor& t, const char* name) {
    check_sizes(c.who, name, t);
    bool ok = t.scalar_type() == c.type && t.device() == c.device && t.dim() == c.lead + 2 && t.stride(-1) == 1;
    for (int64_t i = 0; ok && i < c.lead; ++i) ok = t.size(i) == c.sizes[i];
    if (!ok) {
        std::ostringstream want;
        want << "a tensor of q's type, device and leading sizes " << c.sizes.slice(0, c.lead)
             << ", elements of a head next to each other";
        refuse(c.who, name, want.str(), t);
    }
}

bool on_16_bytes(const Tensor& t) { return reinterpret_cast<std::uintptr_t>(t.const_data_ptr()) % 16 == 0; }

void check_plain(const Common& c, const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef sizes,
                 bool aligned = false) {
    if (t.scalar_type() != type || t.device() != c.device || t.sizes() != sizes || !t.is_contiguous()) {
        std::ostringstream want;
        want << "a contiguous " << type << " tensor of shape " << sizes << " on " << c.device;
        refuse(c.who, name, want.str(), t);
    }
    if (aligned && !on_16_bytes(t))
        refuse(c.who, name, "on a 16-byte boundary", t);
}

void check(int rc) {
    if (rc == NESLE_OK) return;
    if (rc == NESLE_EINVAL) throw py::value_error(nesle_last_error());
    throw std::runtime_error(nesle_last_error());
}

// ---- arguments -------------------------------------------------------------------

nesle_heads heads(const Tensor& t) {
    const int64_t d = t.dim();
    return {t.const_data_ptr(), d == 4 ? t.stride(0) : 0, t.stride(d - 3), t.stride(d - 2)};
}

template <typename T = void>
T* ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

Tensor like(const Tensor& t) { return at::empty_like(t, t.options(), at::MemoryFormat::Contiguous); }

Tensor floats(const Tensor& beside, uint64_t n) {
    return n == 0 ? Tensor() : at::empty({static_cast<int64_t>(n)}, beside.options().dtype(at::kFloat));
}

// Gradients as autograd hands them over, made readable where they are not: of
// heads, and of states (a slice of a longer gradient may start anywhere).
Tensor unit_last(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }
Tensor whole(const Tensor& t) {
    const Tensor c = t.contiguous();
    return on_16_bytes(c) ? c : c.clone();
}
Tensor zeros(const Tensor& t) { return at::zeros_like(t, t.options(), at::MemoryFormat::Contiguous); }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

uint32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? NESLE_MEM_F32 : NESLE_MEM_BF16; }

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Forward-mode derivatives are not there either: a tangent would be lost.
void refuse_tangents(const char* who, std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        if (t->defined() && t->_fw_grad(/*level=*/0).defined())
            throw py::value_error(std::string(who) + " has no forward-mode derivative");
}

// A trace records the allocation of the outputs but no launch: what it replays
// would be memory that nobody wrote.
void refuse_tracing(const char* who) {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    if (torch::jit::tracer::isTracing() || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY).has_value())
        throw py::value_error(std::string(who) + " cannot be traced");
}

// The gradients of a node whose own gradient is not there: asking for it is an
// error, where it is asked for.  They depend on the inputs whatever gradient came
// in, also one that requires none.
variable_list first_order(const char* who, const variable_list& outputs) {
    if (!at::GradMode::is_enabled()) return outputs;
    variable_list fakes;
    for (const Tensor& t : outputs) fakes.push_back(t.defined() ? t.detach().requires_grad_() : t);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string(who) + " has no second derivative", static_cast<int64_t>(fakes.size()));
    return (*error)(std::move(fakes));
}

// ---- norm and rotation -------------------------------------------------------------

nesle_qk_args qk_args(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& positions,
                      const Tensor& table, double eps, bool unit, bool interleaved) {
    nesle_qk_args a{};
    const int64_t d = q.dim();
    a.dtype = dtype_of(q);
    a.steps = d == 4 ? static_cast<uint32_t>(q.size(0)) : 1u;
    a.batch = static_cast<uint32_t>(q.size(d - 3));
    a.q_heads = static_cast<uint32_t>(q.size(d - 2));
    a.k_heads = static_cast<uint32_t>(k.size(d - 2));
    a.dim = static_cast<uint32_t>(q.size(d - 1));
    a.unit = unit;
    a.interleaved = interleaved;
    a.eps = static_cast<float>(eps);
    a.q = heads(q);
    a.k = heads(k);
    a.q_weight = ptr<float>(wq);
    a.k_weight = ptr<float>(wk);
    if (table.defined()) {
        a.rotated = static_cast<uint32_t>(table.size(1));
        a.table_rows = static_cast<uint32_t>(table.size(0));
        a.positions = ptr<int32_t>(positions);
        a.table = ptr<float>(table);
    }
    return a;
}

struct QkNormRotate : torch::autograd::Function<QkNormRotate> {
    static variable_list run(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk,
                             const Tensor& positions, const Tensor& table, double eps, bool unit, bool interleaved) {
        const c10::OptionalDeviceGuard guard(q.device());
        nesle_qk_args a = qk_args(q, k, wq, wk, positions, table, eps, unit, interleaved);
        Tensor q_out = like(q), k_out = like(k);
        a.q_out = ptr(q_out);
        a.k_out = ptr(k_out);
        check(nesle_qk_norm_rotate(&a, stream_of(q)));
        return {q_out, k_out};
    }
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const MaybeTensor& q_weight,
                                 const MaybeTensor& k_weight, const MaybeTensor& steps, const MaybeTensor& turns,
                                 double eps, bool unit, bool interleaved) {
        const Tensor wq = some(q_weight), wk = some(k_weight), positions = some(steps), table = some(turns);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({q, k, wq, wk, positions, table});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["how"] = static_cast<int64_t>(unit) | static_cast<int64_t>(interleaved) << 1;
        return run(q, k, wq, wk, positions, table, eps, unit, interleaved);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &wq = saved[2], &wk = saved[3];
        const int64_t how = ctx->saved_data["how"].toInt();
        const c10::OptionalDeviceGuard guard(q.device());
        variable_list out;
        {
            const at::AutoGradMode none(false);
            nesle_qk_args a = qk_args(q, k, wq, wk, saved[4], saved[5], ctx->saved_data["eps"].toDouble(), how & 1, how & 2);
            const Tensor dq_out = grads[0].defined() ? unit_last(grads[0]) : zeros(q);
            const Tensor dk_out = grads[1].defined() ? unit_last(grads[1]) : zeros(k);
            a.dq_out = heads(dq_out);
            a.dk_out = heads(dk_out);
            const Tensor dq = like(q), dk = like(k), dwq = wq.defined() ? like(wq) : Tensor(),
                         dwk = wk.defined() ? like(wk) : Tensor(), scratch = floats(q, nesle_qk_scratch_floats(&a));
            a.dq = ptr(dq);
            a.dk = ptr(dk);
            a.dq_weight = ptr<float>(dwq);
            a.dk_weight = ptr<float>(dwk);
            a.scratch = ptr<float>(scratch);
            check(nesle_qk_norm_rotate_grad(&a, stream_of(q)));
            out = {dq, dk, dwq, dwk};
        }
        out = first_order("qk_norm_rotate", out);
        out.resize(9);
        return out;
    }
};

py::tuple qk_norm_rotate(const Tensor& q, const Tensor& k, const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                         const MaybeTensor& positions, const MaybeTensor& table, double eps, bool unit, bool interleaved) {
    const Tensor wq = some(q_weight), wk = some(k_weight), turns = some(table);
    refuse_tracing("qk_norm_rotate");
    refuse_tangents("qk_norm_rotate", {&q, &k, &wq, &wk, &turns});
    const Common c = common_of("qk_norm_rotate", q, 1, 2);
    check_heads(c, k, "k");
    const int64_t dim = q.size(-1);
    if (k.size(-1) != dim) refuse(c.who, "k", "of q's head dimension " + std::to_string(dim), k);
    if (wq.defined()) check_plain(c, wq, "q_weight", at::kFloat, {dim}, true);
    if (wk.defined()) check_plain(c, wk, "k_weight", at::kFloat, {dim}, true);
    Tensor at_step;
    if (turns.defined()) {
        check_sizes(c.who, "table", turns);
        if (turns.dim() != 2 || turns.size(0) < 1 || turns.size(1) < 8 || turns.size(1) % 8 != 0 || turns.size(1) > dim)
            refuse(c.who, "table", "a float32 tensor [rows, R], R a multiple of 8 up to " + std::to_string(dim), turns);
        check_plain(c, turns, "table", at::kFloat, turns.sizes(), true);
        if (!given(positions)) throw py::value_error("qk_norm_rotate: a table needs positions");
        at_step = *positions;
        check_plain(c, at_step, "positions", at::kInt, c.sizes.slice(0, c.lead));
    } else if (given(positions)) {
        throw py::value_error("qk_norm_rotate: positions need a table");
    }
    const variable_list out = wants_grad({&q, &k, &wq, &wk})
        ? QkNormRotate::apply(q, k, q_weight, k_weight, positions, table, eps, unit, interleaved)
        : QkNormRotate::run(q, k, wq, wk, at_step, turns, eps, unit, interleaved);
    return py::make_tuple(out[0], out[1]);
}

// ---- the gated delta rule -------------------------------------------------------------

nesle_delta_args delta_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                            const Tensor& state, const Tensor& resets, double scale) {
    nesle_delta_args a{};
    const int64_t d = q.dim();
    a.dtype = dtype_of(q);
    a.steps = d == 4 ? static_cast<uint32_t>(q.size(0)) : 1u;
    a.batch = static_cast<uint32_t>(q.size(d - 3));
    a.k_heads = static_cast<uint32_t>(q.size(d - 2));
    a.v_heads = static_cast<uint32_t>(v.size(d - 2));
    a.k_dim = static_cast<uint32_t>(q.size(d - 1));
    a.v_dim = static_cast<uint32_t>(v.size(d - 1));
    a.scale = static_cast<float>(scale);
    a.q = heads(q);
    a.k = heads(k);
    a.v = heads(v);
    a.g = ptr<float>(g);
    a.beta = ptr<float>(beta);
    a.resets = ptr<uint8_t>(resets);
    a.state = ptr<float>(state);
    return a;
}

void check_delta(const Common& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                 const Tensor& beta, const Tensor& state, const Tensor& resets) {
    check_heads(c, k, "k");
    check_heads(c, v, "v");
    if (k.sizes() != q.sizes()) refuse(c.who, "k", "of q's shape", k);
    const int64_t hk = q.size(-2), dk = q.size(-1), hv = v.size(-2), dv = v.size(-1);
    if (hk == 0 || hv == 0 || hv % hk != 0) refuse(c.who, "v", "of a multiple of " + std::to_string(hk) + " heads", v);
    constexpr int64_t most = NESLE_DELTA_MAX_DIM;
    if (dk % 8 != 0 || dv % 8 != 0 || dk < 8 || dv < 8 || dk > most || dv > most)
        throw py::value_error(std::string(c.who) + ": head dimensions must be multiples of 8 up to " + std::to_string(most) +
                              ", got " + std::to_string(dk) + " and " + std::to_string(dv));
    c10::SmallVector<int64_t, 3> gates(c.sizes.slice(0, c.lead).begin(), c.sizes.slice(0, c.lead).end());
    gates.push_back(hv);
    check_plain(c, g, "g", at::kFloat, gates);
    check_plain(c, beta, "beta", at::kFloat, gates);
    if (state.defined()) check_plain(c, state, "state", at::kFloat, {c.batch(), hv, dk, dv}, true);
    if (resets.defined())
        check_plain(c, resets, "resets", resets.scalar_type() == at::kByte ? at::kByte : at::kBool, c.sizes.slice(0, c.lead));
}

double scale_or_default(const std::optional<double>& scale, const Tensor& q) {
    return scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(-1)));
}

struct GatedDelta : torch::autograd::Function<GatedDelta> {
    // Output, state after it and, to keep for the gradient, the states before
    // the chunks.
    static variable_list run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                             const Tensor& state, const Tensor& resets, double scale, bool keep) {
        const c10::OptionalDeviceGuard guard(q.device());
        nesle_delta_args a = delta_args(q, k, v, g, beta, state, resets, scale);
        const Tensor out = like(v), after = at::empty({v.size(1), v.size(2), q.size(3), v.size(3)}, g.options());
        const Tensor saved = floats(q, keep ? nesle_delta_saved_floats(&a) : 0);
        const Tensor scratch = floats(q, nesle_delta_forward_scratch_floats(&a));
        a.out = ptr(out);
        a.state_out = ptr<float>(after);
        a.saved = ptr<float>(saved);
        a.scratch = ptr<float>(scratch);
        check(nesle_delta_forward(&a, stream_of(q)));
        return {out, after, saved};
    }
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& g, const Tensor& beta, const MaybeTensor& start, const MaybeTensor& ends,
                                 double scale) {
        const Tensor state = some(start), resets = some(ends);
        variable_list out = run(q, k, v, g, beta, state, resets, scale, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({q, k, v, g, beta, state, resets, out[2]});
        ctx->saved_data["scale"] = scale;
        out.pop_back();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &v = saved[2], &state = saved[5];
        const c10::OptionalDeviceGuard guard(q.device());
        variable_list out;
        {
            const at::AutoGradMode none(false);
            nesle_delta_args a = delta_args(q, saved[1], v, saved[3], saved[4], state, saved[6],
                                            ctx->saved_data["scale"].toDouble());
            const Tensor dout = grads[0].defined() ? unit_last(grads[0]) : zeros(v);
            const Tensor dafter = grads[1].defined() ? whole(grads[1]) : Tensor();
            const Tensor dq = like(q), dk = like(q), dv = like(v), dg = like(saved[3]), dbeta = like(saved[4]);
            const Tensor dstate = state.defined() && state.requires_grad() ? like(state) : Tensor();
            const Tensor scratch = floats(q, nesle_delta_scratch_floats(&a));
            a.saved = ptr<float>(saved[7]);
            a.dout = heads(dout);
            a.dstate_out = ptr<float>(dafter);
            a.dq = ptr(dq);
            a.dk = ptr(dk);
            a.dv = ptr(dv);
            a.dg = ptr<float>(dg);
            a.dbeta = ptr<float>(dbeta);
            a.dstate = ptr<float>(dstate);
            a.scratch = ptr<float>(scratch);
            check(nesle_delta_backward(&a, stream_of(q)));
            out = {dq, dk, dv, dg, dbeta, dstate};
        }
        out = first_order("gated_delta", out);
        out.resize(8);
        return out;
    }
};

py::tuple gated_delta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                      const MaybeTensor& state, const MaybeTensor& resets, const std::optional<double>& scale) {
    const Tensor start = some(state), ends = some(resets);
    refuse_tracing("gated_delta");
    refuse_tangents("gated_delta", {&q, &k, &v, &g, &beta, &start});
    const Common c = common_of("gated_delta", q, 2, 2);
    check_delta(c, q, k, v, g, beta, start, ends);
    const double s = scale_or_default(scale, q);
    const variable_list out = wants_grad({&q, &k, &v, &g, &beta, &start})
        ? GatedDelta::apply(q, k, v, g, beta, state, resets, s)
        : GatedDelta::run(q, k, v, g, beta, start, ends, s, false);
    return py::make_tuple(out[0], out[1]);
}

Tensor gated_delta_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                        const MaybeTensor& state, const MaybeTensor& resets, const std::optional<double>& scale) {
    if (!given(state)) throw py::value_error("gated_delta_step: state must be a tensor");
    refuse_tracing("gated_delta_step");
    refuse_tangents("gated_delta_step", {&q, &k, &v, &g, &beta, &*state});
    const Common c = common_of("gated_delta_step", q, 1, 1);
    const Tensor ends = some(resets);
    check_delta(c, q, k, v, g, beta, *state, ends);
    if (wants_grad({&q, &k, &v, &g, &beta, &*state}))
        throw py::value_error("gated_delta_step has no gradient: use gated_delta, or torch.no_grad()");
    const c10::OptionalDeviceGuard guard(q.device());
    nesle_delta_args a = delta_args(q, k, v, g, beta, *state, ends, scale_or_default(scale, q));
    const Tensor out = like(v);
    a.out = ptr(out);
    a.state_out = ptr<float>(*state);
    state->unsafeGetTensorImpl()->bump_version();          // autograd sees the state change
    check(nesle_delta_step(&a, stream_of(q)));
    return out;
}

}  // namespace

PYBIND11_MODULE(_memory_native, m) {
    m.doc() = "Tensor and autograd binding of the memory operators (see nesle_amd.memory)";
    m.def("qk_norm_rotate", &qk_norm_rotate);
    m.def("gated_delta", &gated_delta);
    m.def("gated_delta_step", &gated_delta_step);
}
