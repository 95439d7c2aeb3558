// The temporal operators as torch functions: argument checks, allocation, autograd nodes and launches (through the C ABI of libsrvp_hip.so, whose
// entry points the host side passes in).  In C++ because the small calls are host-bound: with the same checks and autograd nodes in Python a training pass of
// the norm over 2304 x 256 took 124 us (now 69, of which 40 are the engine's hand-over to its thread and 14 the kernels), a single-frame step 10.6 us (4.8).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <string>

#include "../../include/srvp_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

namespace {

// ---- entry points
#define ENTRIES(X)                                                                                        \
    X(srvp_last_error) X(srvp_stream_is_capturing) X(srvp_linear_attention_ws_bytes) X(srvp_linear_attention_fwd) X(srvp_linear_attention_bwd) \
    X(srvp_linear_attention_step) X(srvp_rotary) X(srvp_rms_norm) X(srvp_rms_norm_bwd_ws_bytes) X(srvp_rms_norm_bwd) X(srvp_linear_int8)
struct Entries {
#define X(name) decltype(&::name) name = nullptr;
    ENTRIES(X)
#undef X
} lib;
PyObject *hip_error = nullptr, *memory_error = nullptr;      // srvp_amd._lib.SrvpHipError, torch.OutOfMemoryError

void bind(const py::dict& addresses, const py::object& error, const py::object& no_memory) {
#define X(name) lib.name = reinterpret_cast<decltype(&::name)>(addresses[#name].cast<uintptr_t>());
    ENTRIES(X)
#undef X
    Py_INCREF(error.ptr());
    Py_INCREF(no_memory.ptr());
    hip_error = error.ptr();
    memory_error = no_memory.ptr();
}

// ---- errors
[[noreturn]] void value_error(const std::string& m) { throw py::value_error(m); }
[[noreturn]] void type_error(const std::string& m) { throw py::type_error(m); }
struct HipError : std::runtime_error { using std::runtime_error::runtime_error; };
void check(int rc, const char* what) {
    if (rc) throw HipError(std::string(what) + " failed (code " + std::to_string(rc) + "): " + lib.srvp_last_error());
}
std::string shape(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + (t.dim() == 1 ? ",)" : ")");
}
std::string dtype(const Tensor& t) { return c10::toString(t.scalar_type()); }

// ---- arguments
void on_device(const char* what, const Tensor& x) {
    if (!x.is_cuda()) throw HipError(std::string(what) + ": srvp_amd runs on an MI355X only: move the tensors to the GPU; there is no CPU compute path");
}
void same_device(const char* what, const Tensor& x, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t && t->defined() && t->device() != x.device()) value_error(std::string(what) + ": all tensors on one device");
}
void floats(const char* what, std::initializer_list<const Tensor*> ts) {
    const at::ScalarType d = (*ts.begin())->scalar_type();
    if (d != at::kFloat && d != at::kBFloat16) type_error(std::string(what) + ": float32 or bfloat16 tensors, got " + dtype(**ts.begin()));
    for (const Tensor* t : ts)
        if (t->defined() && t->scalar_type() != d) type_error(std::string(what) + ": tensors of one type, got " + c10::toString(d) + " and " + dtype(*t));
}
Tensor inner(const Tensor& x) { return !x.defined() || x.size(-1) <= 1 || x.stride(-1) == 1 ? x : x.contiguous(); }
// (rows, features), features contiguous
Tensor matrix(const Tensor& x) { return !x.defined() ? x : x.dim() == 2 ? inner(x) : inner(x.reshape({-1, x.size(-1)})); }
Tensor whole(const char* what, const char* name, const Tensor& x) {
    if (x.scalar_type() == at::kLong) return x;
    if (x.scalar_type() == at::kInt) return x.to(at::kLong);
    type_error(std::string(what) + ": " + name + " is an int64 or int32 tensor, got " + dtype(x));
}
Tensor decays(const char* what, const Tensor& l, int64_t H) {
    if (l.scalar_type() != at::kFloat || l.dim() != 1 || l.size(0) != H)
        value_error(std::string(what) + ": log_decay is a float32 tensor of one value a head (" + std::to_string(H) + "), got " + shape(l) + " " + dtype(l));
    if (at::GradMode::is_enabled() && l.requires_grad()) value_error(std::string(what) + ": the decays are constants: log_decay must not require a gradient");
    return l.contiguous();
}
bool any_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// (a launch would come back without the tangent, whether or not the tensors ask for a gradient)
void no_tangent(const char* what, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->defined() && t->_fw_grad(0).defined()) throw std::runtime_error(std::string(what) + ": forward-mode derivatives are not supported");
}
void* stream_of(const Tensor& x) { return (void*)c10::hip::getCurrentHIPStream(x.get_device()).stream(); }
// whether the call is to be recorded for autograd.  Not inside a capture: leaves whose eager graph is still alive would pull its stream into the captured
// backward pass, which ends the process.
bool records(const char* what, const Tensor& x, std::initializer_list<const Tensor*> ts) {
    if (!any_grad(ts)) return false;
    int on = 0;
    const c10::DeviceGuard guard(x.device());
    check(lib.srvp_stream_is_capturing(stream_of(x), &on), "srvp_stream_is_capturing");
    if (on) throw std::runtime_error(std::string(what) + ": no gradient is recorded inside a stream capture; detach the inputs and call the backward function itself");
    return true;
}
void no_gradient(const char* what, std::initializer_list<const Tensor*> ts) {
    if (any_grad(ts)) value_error(std::string(what) + ": records no gradient: call it under torch.no_grad() or with detached tensors");
}
void once() {
    // (a backward pass that is itself recorded would come back without the kernels' part)
    if (at::GradMode::is_enabled()) throw std::runtime_error("srvp_amd.temporal: the operators are differentiable once (create_graph=True is not supported)");
}
Tensor get(const Maybe& t) { return t ? *t : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }
void strides3(int64_t* s, const Tensor& t) {
    for (int i = 0; i < 3; ++i) s[i] = t.defined() ? t.stride(i) : 0;
}
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// =============================================================================================================== linear attention
struct Attention {
    Tensor q, k, v, log_decay, state, lengths;
    double scale;
};
Attention attention_args(const char* what, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& state, const Maybe& lengths,
                         std::optional<double> scale) {
    on_device(what, q);
    if (q.dim() != 4 || k.sizes() != q.sizes() || v.dim() != 4 || v.size(0) != q.size(0) || v.size(1) != q.size(1) || v.size(2) != q.size(2))
        value_error(std::string(what) + ": q, k (T, B, H, Dk) and v (T, B, H, Dv), got " + shape(q) + ", " + shape(k) + ", " + shape(v));
    floats(what, {&q, &k, &v});
    const int64_t B = q.size(1), H = q.size(2), Dk = q.size(3), Dv = v.size(3);
    if (Dk < 1 || Dk > 256 || Dv < 1 || Dv > 256) value_error(std::string(what) + ": heads of 1 to 256 features, got " + std::to_string(Dk) + " and " + std::to_string(Dv));
    if (q.size(0) >= (1 << 30) || B >= (1 << 20) || H >= (1 << 20) || B * H >= (1 << 20)) value_error(std::string(what) + ": fewer than 2^30 tokens and 2^20 (sequence, head) pairs");
    Attention a;
    a.log_decay = decays(what, log_decay, H);
    if (state) {
        if (state->scalar_type() != at::kFloat || state->sizes() != at::IntArrayRef({B, H, Dk, Dv}))
            value_error(std::string(what) + ": state is a float32 tensor (" + std::to_string(B) + ", " + std::to_string(H) + ", " + std::to_string(Dk) + ", " +
                        std::to_string(Dv) + "), got " + shape(*state) + " " + dtype(*state));
        a.state = state->contiguous();
    }
    if (lengths) {
        if (lengths->dim() != 1 || lengths->size(0) != B) value_error(std::string(what) + ": one length a sequence (" + std::to_string(B) + "), got " + shape(*lengths));
        a.lengths = whole(what, "lengths", *lengths).contiguous();
    }
    same_device(what, q, {&k, &v, &a.log_decay, &a.state, &a.lengths});
    a.scale = scale ? *scale : 1.0 / std::sqrt((double)Dk);
    if (!(std::abs(a.scale) >= 1e-30 && std::abs(a.scale) <= 1e30)) value_error(std::string(what) + ": scale of 1e-30 to 1e30, got " + std::to_string(a.scale));
    a.q = inner(q);
    a.k = inner(k);
    a.v = inner(v);
    return a;
}
srvp_linear_attention_desc describe(const Attention& a, const Tensor& o, const Tensor& new_state) {
    srvp_linear_attention_desc d = {};
    d.q = ptr(a.q); d.k = ptr(a.k); d.v = ptr(a.v); d.o = ptr(o);
    strides3(d.qs, a.q); strides3(d.ks, a.k); strides3(d.vs, a.v); strides3(d.os, o);
    d.log_decay = (const float*)ptr(a.log_decay);
    d.state_in = (const float*)ptr(a.state);
    d.state_out = (float*)ptr(new_state);
    d.lengths = (const int64_t*)ptr(a.lengths);
    d.T = a.q.size(0); d.B = a.q.size(1); d.H = a.q.size(2); d.Dk = a.q.size(3); d.Dv = a.v.size(3);
    d.scale = (float)a.scale;
    d.elem_f32 = f32(a.q);
    return d;
}
Tensor workspace(srvp_linear_attention_desc& d, int backward, const Tensor& like) {
    const int64_t n = lib.srvp_linear_attention_ws_bytes(&d, backward);
    if (n < 0) check(1, "srvp_linear_attention_ws_bytes");
    Tensor ws;
    if (n) {
        ws = bytes(n, like);
        d.ws = ptr(ws);
        d.ws_bytes = n;
    }
    return ws;
}
variable_list attention_fwd(const Attention& a, bool want_state) {
    const c10::DeviceGuard guard(a.q.device());
    const int64_t B = a.q.size(1), H = a.q.size(2), Dk = a.q.size(3), Dv = a.v.size(3);
    Tensor o = at::empty(a.v.sizes(), a.v.options()), s;
    if (want_state) s = at::empty({B, H, Dk, Dv}, a.v.options().dtype(at::kFloat));
    auto d = describe(a, o, s);
    const Tensor ws = workspace(d, 0, o);
    check(lib.srvp_linear_attention_fwd(&d, stream_of(o)), "srvp_linear_attention_fwd");
    if (want_state) return {o, s};
    return {o};
}
variable_list attention_bwd(const Attention& a, Tensor d_out, Tensor d_new, bool want_state) {
    const c10::DeviceGuard guard(a.q.device());
    const int64_t B = a.q.size(1), H = a.q.size(2), Dk = a.q.size(3), Dv = a.v.size(3);
    d_out = inner(d_out);
    if (d_new.defined()) d_new = d_new.contiguous();
    Tensor dq = at::empty(a.q.sizes(), a.q.options()), dk = at::empty(a.q.sizes(), a.q.options()), dv = at::empty(a.v.sizes(), a.v.options()), ds;
    if (want_state) ds = at::empty({B, H, Dk, Dv}, a.v.options().dtype(at::kFloat));
    srvp_linear_attention_bwd_desc d = {};
    d.f = describe(a, Tensor(), Tensor());
    const Tensor ws = workspace(d.f, 1, dq);
    d.d_o = ptr(d_out); d.dq = ptr(dq); d.dk = ptr(dk); d.dv = ptr(dv);
    strides3(d.d_os, d_out); strides3(d.dqs, dq); strides3(d.dks, dk); strides3(d.dvs, dv);
    d.d_state_out = (const float*)ptr(d_new);
    d.d_state_in = (float*)ptr(ds);
    check(lib.srvp_linear_attention_bwd(&d, stream_of(dq)), "srvp_linear_attention_bwd");
    return {dq, dk, dv, ds};
}
struct AttentionNode : torch::autograd::Function<AttentionNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& state,
                                 const Maybe& lengths, double scale, bool want_state) {
        const Attention a{q, k, v, log_decay, get(state), get(lengths), scale};
        ctx->save_for_backward({q, k, v, log_decay, a.state, a.lengths});
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        return attention_fwd(a, want_state);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once();
        const auto s = ctx->get_saved_variables();
        const Attention a{s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["scale"].toDouble()};
        const Tensor d_out = g[0].defined() ? g[0] : at::zeros(a.v.sizes(), a.v.options());
        const auto r = attention_bwd(a, d_out, g.size() > 1 ? g[1] : Tensor(), a.state.defined() && ctx->needs_input_grad(4));
        return {r[0], r[1], r[2], Tensor(), r[3], Tensor(), Tensor(), Tensor()};
    }
};
py::object linear_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& state, const Maybe& lengths,
                            std::optional<double> scale, bool return_state) {
    const Attention a = attention_args("linear_attention", q, k, v, log_decay, state, lengths, scale);
    no_tangent("linear_attention", {&a.q, &a.k, &a.v, &a.log_decay, &a.state});
    variable_list r;
    if (records("linear_attention", a.q, {&a.q, &a.k, &a.v, &a.state}))
        r = AttentionNode::apply(a.q, a.k, a.v, a.log_decay, a.state.defined() ? Maybe(a.state) : Maybe(), a.lengths.defined() ? Maybe(a.lengths) : Maybe(), a.scale, return_state);
    else
        r = attention_fwd(a, return_state);
    return return_state ? (py::object)py::make_tuple(r[0], r[1]) : py::cast(r[0]);
}
py::tuple linear_attention_backward(const Tensor& d_out, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& state,
                                    const Maybe& lengths, std::optional<double> scale, const Maybe& d_state) {
    const char* what = "linear_attention_backward";
    const Attention a = attention_args(what, q, k, v, log_decay, state, lengths, scale);
    const Tensor dn = get(d_state);
    no_tangent(what, {&d_out, &a.q, &a.k, &a.v, &a.log_decay, &a.state, &dn});
    no_gradient(what, {&d_out, &a.q, &a.k, &a.v, &a.state, &dn});
    if (d_out.sizes() != a.v.sizes()) value_error(std::string(what) + ": d_out " + shape(a.v) + ", got " + shape(d_out));
    floats(what, {&a.q, &d_out});
    if (dn.defined() && (dn.scalar_type() != at::kFloat || dn.sizes() != at::IntArrayRef({a.q.size(1), a.q.size(2), a.q.size(3), a.v.size(3)})))
        value_error(std::string(what) + ": d_state is a float32 tensor of the state's shape, got " + shape(dn) + " " + dtype(dn));
    same_device(what, a.q, {&d_out, &dn});
    const auto r = attention_bwd(a, d_out, dn, a.state.defined());
    return py::make_tuple(r[0], r[1], r[2], r[3].defined() ? py::cast(r[3]) : py::none());
}
Tensor linear_attention_step(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& log_decay, const Tensor& state, const Maybe& slots,
                             std::optional<double> scale) {
    const char* what = "linear_attention_step";
    on_device(what, q0);
    if (q0.dim() != 3 || k0.sizes() != q0.sizes() || v0.dim() != 3 || v0.size(0) != q0.size(0) || v0.size(1) != q0.size(1))
        value_error(std::string(what) + ": q, k (B, H, Dk) and v (B, H, Dv), got " + shape(q0) + ", " + shape(k0) + ", " + shape(v0));
    floats(what, {&q0, &k0, &v0});
    no_tangent(what, {&q0, &k0, &v0, &log_decay, &state});
    no_gradient(what, {&q0, &k0, &v0, &state});
    const int64_t B = q0.size(0), H = q0.size(1), Dk = q0.size(2), Dv = v0.size(2);
    if (Dk < 1 || Dk > 256 || Dv < 1 || Dv > 256) value_error(std::string(what) + ": heads of 1 to 256 features, got " + std::to_string(Dk) + " and " + std::to_string(Dv));
    if (B >= (1 << 24) || H >= (1 << 24) || B * H >= (1 << 24) || (state.dim() == 4 && state.size(0) >= (1LL << 31))) value_error(std::string(what) + ": fewer than 2^24 (row, head) pairs and 2^31 states");
    const Tensor ld = decays(what, log_decay, H);
    if (state.scalar_type() != at::kFloat || state.dim() != 4 || state.size(1) != H || state.size(2) != Dk || state.size(3) != Dv || !state.is_contiguous() ||
        (state.numel() && (uintptr_t)state.data_ptr() % 16))
        value_error(std::string(what) + ": state is a contiguous, 16-byte aligned float32 tensor (slots, " + std::to_string(H) + ", " + std::to_string(Dk) + ", " +
                    std::to_string(Dv) + "), got " + shape(state) + " " + dtype(state));
    Tensor sl;
    if (slots) {
        if (B > 65536) value_error(std::string(what) + ": at most 65536 rows with slots, got " + std::to_string(B));
        if (slots->dim() != 1 || slots->size(0) != B) value_error(std::string(what) + ": one slot a row (" + std::to_string(B) + "), got " + shape(*slots));
        sl = whole(what, "slots", *slots).contiguous();
    } else if (B > state.size(0)) {
        value_error(std::string(what) + ": " + std::to_string(B) + " rows for " + std::to_string(state.size(0)) + " states");
    }
    same_device(what, q0, {&k0, &v0, &ld, &state, &sl});
    const c10::DeviceGuard guard(q0.device());
    const Tensor q = inner(q0), k = inner(k0), v = inner(v0);
    Tensor o = at::empty({B, H, Dv}, v.options());
    srvp_linear_attention_step_desc d = {};
    d.q = ptr(q); d.k = ptr(k); d.v = ptr(v); d.o = ptr(o);
    for (int i = 0; i < 2; ++i) { d.qs[i] = q.stride(i); d.ks[i] = k.stride(i); d.vs[i] = v.stride(i); d.os[i] = o.stride(i); }
    d.log_decay = (const float*)ptr(ld); d.state = (float*)ptr(state); d.slots = (const int64_t*)ptr(sl);
    d.B = B; d.H = H; d.Dk = Dk; d.Dv = Dv; d.nslots = state.size(0); d.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)Dk)); d.elem_f32 = f32(q);
    check(lib.srvp_linear_attention_step(&d, stream_of(o)), "srvp_linear_attention_step");
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();      // (changed behind autograd's back)
    return o;
}

// ========================================================================================================================= rotary
struct Turn {
    bool interleaved, back;
    double magnitude;
};
variable_list turn(const Tensor& q0, const Tensor& k0, const Tensor& positions, const Tensor& freq, const Turn& t, bool back) {
    const c10::DeviceGuard guard(q0.device());
    const Tensor q = inner(q0), k = inner(k0);
    Tensor oq = at::empty(q.sizes(), q.options()), ok;
    if (k.defined()) ok = at::empty(k.sizes(), k.options());
    srvp_rotary_desc d = {};
    d.q = ptr(q); d.k = ptr(k); d.oq = ptr(oq); d.ok = ptr(ok);
    strides3(d.qs, q); strides3(d.ks, k); strides3(d.oqs, oq); strides3(d.oks, ok);
    d.positions = (const int64_t*)ptr(positions);
    d.pos_t = positions.stride(0);
    d.pos_b = positions.dim() == 2 ? positions.stride(1) : 0;
    d.freq = (const double*)ptr(freq);
    d.T = q.size(0); d.B = q.size(1); d.Hq = q.size(2); d.Hk = k.defined() ? k.size(2) : 0; d.D = q.size(3); d.pairs = freq.size(0);
    d.interleaved = t.interleaved; d.back = back; d.magnitude = (float)t.magnitude; d.elem_f32 = f32(q);
    check(lib.srvp_rotary(&d, stream_of(oq)), "srvp_rotary");
    if (k.defined()) return {oq, ok};
    return {oq};
}
struct RotaryNode : torch::autograd::Function<RotaryNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Maybe& k, const Tensor& positions, const Tensor& freq, bool interleaved, bool back, double magnitude) {
        ctx->save_for_backward({positions, freq});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["back"] = back;
        ctx->saved_data["magnitude"] = magnitude;
        ctx->set_materialize_grads(false);
        return turn(q, get(k), positions, freq, Turn{interleaved, back, magnitude}, back);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once();
        const auto s = ctx->get_saved_variables();
        const Turn t{ctx->saved_data["interleaved"].toBool(), ctx->saved_data["back"].toBool(), ctx->saved_data["magnitude"].toDouble()};
        variable_list r(7);
        const Tensor gq = g[0], gk = g.size() > 1 ? g[1] : Tensor();
        if (gq.defined()) {
            auto o = turn(gq, gk, s[0], s[1], t, !t.back);
            r[0] = o[0];
            if (gk.defined()) r[1] = o[1];
        } else if (gk.defined()) {
            r[1] = turn(gk, Tensor(), s[0], s[1], t, !t.back)[0];
        }
        return r;
    }
};
py::object rotary(const Tensor& q, const Maybe& k, const Tensor& positions0, const Tensor& freq, bool interleaved, bool back, double magnitude) {
    const char* what = "rotary";
    on_device(what, q);
    const Tensor kk = get(k);
    if (q.dim() != 4 || (k && (kk.dim() != 4 || kk.size(0) != q.size(0) || kk.size(1) != q.size(1) || kk.size(3) != q.size(3))))
        value_error(std::string(what) + ": q (T, B, Hq, D) and k (T, B, Hk, D), got " + shape(q) + (k ? ", " + shape(kk) : ""));
    floats(what, {&q, &kk});
    no_tangent(what, {&q, &kk, &freq});
    const int64_t T = q.size(0), B = q.size(1), D = q.size(3);
    if (T >= (1LL << 31) || B >= (1LL << 31) || T * B >= (1LL << 31) || q.size(2) >= (1 << 20) || (k && kk.size(2) >= (1 << 20)))
        value_error(std::string(what) + ": fewer than 2^31 rows and 2^20 heads, got " + shape(q) + (k ? ", " + shape(kk) : ""));
    if (D < 1 || D > 4096) value_error(std::string(what) + ": heads of 1 to 4096 features, got " + std::to_string(D));
    if (!(positions0.dim() == 1 && positions0.size(0) == T) && !(positions0.dim() == 2 && positions0.size(0) == T && positions0.size(1) == B))
        value_error(std::string(what) + ": positions (" + std::to_string(T) + ",) or (" + std::to_string(T) + ", " + std::to_string(B) + "), got " + shape(positions0));
    if (freq.scalar_type() != at::kDouble || freq.dim() != 1 || 2 * freq.size(0) > D || !freq.is_contiguous())
        value_error(std::string(what) + ": frequencies is a contiguous float64 tensor of at most " + std::to_string(D / 2) + " pairs, got " + shape(freq) + " " + dtype(freq));
    if (any_grad({&freq})) value_error(std::string(what) + ": the frequencies are constants: they must not require a gradient");
    if (!std::isfinite((float)magnitude)) value_error(std::string(what) + ": magnitude must be finite");
    const Tensor positions = whole(what, "positions", positions0);
    same_device(what, q, {&kk, &positions, &freq});
    const variable_list r = records(what, q, {&q, &kk}) ? RotaryNode::apply(q, k, positions, freq, interleaved, back, magnitude)
                                                        : turn(q, kk, positions, freq, Turn{interleaved, back, magnitude}, back);
    return k ? (py::object)py::make_tuple(r[0], r[1]) : py::cast(r[0]);
}

// =========================================================================================================================== norm
void norm_args(const char* what, const Tensor& x, const Tensor& weight, const Tensor& residual) {
    on_device(what, x);
    floats(what, {&x, &residual});
    no_tangent(what, {&x, &weight, &residual});
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > 16384) value_error(std::string(what) + ": rows of 1 to 16384 features, got " + shape(x));
    if (x.numel() / x.size(-1) >= (1LL << 31)) value_error(std::string(what) + ": fewer than 2^31 rows");
    if (residual.defined() && residual.sizes() != x.sizes()) value_error(std::string(what) + ": residual " + shape(residual) + " for x " + shape(x));
    if (weight.defined() && (weight.scalar_type() != at::kFloat || weight.dim() != 1 || weight.size(0) != x.size(-1)))
        value_error(std::string(what) + ": weight is a float32 tensor (" + std::to_string(x.size(-1)) + ",), got " + shape(weight) + " " + dtype(weight));
    same_device(what, x, {&weight, &residual});
}
int64_t row_stride(const Tensor& m) { return m.defined() ? m.stride(0) : 0; }
variable_list norm_fwd(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps) {
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = matrix(x), r2 = matrix(residual), w = weight.contiguous();
    Tensor y = at::empty(x.sizes(), x.options()), sum;
    if (residual.defined()) sum = at::empty(x.sizes(), x.options());
    srvp_rms_norm_desc d = {};
    d.x = ptr(x2); d.residual = ptr(r2); d.w = (const float*)ptr(w); d.y = ptr(y); d.sum = ptr(sum);
    d.N = x.size(-1);
    d.xs = row_stride(x2); d.rs = row_stride(r2); d.ys = d.ss = d.N; d.M = x2.size(0);
    d.eps = (float)eps; d.elem_f32 = f32(x);
    check(lib.srvp_rms_norm(&d, stream_of(y)), "srvp_rms_norm");
    if (sum.defined()) return {y, sum};
    return {y};
}
variable_list norm_bwd(const Tensor& d_y, const Tensor& d_sum, const Tensor& x, const Tensor& weight, const Tensor& residual, double eps) {
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = matrix(x), r2 = matrix(residual), y2 = matrix(d_y), s2 = matrix(d_sum), w = weight.contiguous();
    Tensor dx = at::empty(x.sizes(), x.options());
    const int64_t M = x2.size(0), N = x.size(-1);
    if (M == 0) return {dx, at::zeros({N}, weight.options())};
    Tensor dw = at::empty({N}, weight.options());
    srvp_rms_norm_bwd_desc d = {};
    d.ws_bytes = lib.srvp_rms_norm_bwd_ws_bytes(M, N, f32(x));
    const Tensor ws = bytes(d.ws_bytes, x);
    d.x = ptr(x2); d.residual = ptr(r2); d.d_y = ptr(y2); d.d_sum = ptr(s2); d.w = (const float*)ptr(w); d.dx = ptr(dx); d.dw = (float*)ptr(dw); d.ws = ptr(ws);
    d.xs = row_stride(x2); d.rs = row_stride(r2); d.dys = row_stride(y2); d.dss = row_stride(s2); d.dxs = N; d.M = M; d.N = N;
    d.eps = (float)eps; d.elem_f32 = f32(x);
    check(lib.srvp_rms_norm_bwd(&d, stream_of(dx)), "srvp_rms_norm_bwd");
    return {dx, dw};
}
struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& residual, double eps) {
        ctx->save_for_backward({x, weight, get(residual)});
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        return norm_fwd(x, weight, get(residual), eps);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once();
        const auto s = ctx->get_saved_variables();
        const Tensor d_sum = g.size() > 1 ? g[1] : Tensor();
        if (!g[0].defined()) return {d_sum, Tensor(), s[2].defined() ? d_sum : Tensor(), Tensor()};
        const auto r = norm_bwd(g[0], d_sum, s[0], s[1], s[2], ctx->saved_data["eps"].toDouble());
        return {r[0], r[1], s[2].defined() ? r[0] : Tensor(), Tensor()};
    }
};
py::object rms_norm(const Tensor& x, const Tensor& weight, const Maybe& residual, double eps) {
    const Tensor r = get(residual);
    norm_args("rms_norm", x, weight, r);
    const variable_list o = records("rms_norm", x, {&x, &weight, &r}) ? NormNode::apply(x, weight, residual, eps) : norm_fwd(x, weight, r, eps);
    return residual ? (py::object)py::make_tuple(o[0], o[1]) : py::cast(o[0]);
}
py::tuple rms_norm_backward(const Tensor& d_y, const Tensor& x, const Tensor& weight, const Maybe& residual, const Maybe& d_sum, double eps) {
    const char* what = "rms_norm_backward";
    const Tensor r = get(residual), ds = get(d_sum);
    norm_args(what, x, weight, r);
    norm_args(what, x, weight, d_y);
    norm_args(what, x, weight, ds);
    no_gradient(what, {&d_y, &x, &weight, &r, &ds});
    const auto o = norm_bwd(d_y, ds, x, weight, r, eps);
    return py::make_tuple(o[0], o[1]);
}

// ========================================================================================================================= 8 bits
// weight undefined: the rows themselves
py::tuple rows_int8(const char* what, const Tensor& x, const Tensor& weight, const Tensor& residual, double eps) {
    norm_args(what, x, weight, residual);
    no_gradient(what, {&x, &weight, &residual});
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = matrix(x), r2 = matrix(residual), w = weight.defined() ? weight.contiguous() : weight;
    const int64_t N = x.size(-1), P = (N + 15) / 16 * 16;      // rows start at 16-byte borders, for the product's loads
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = P;
    Tensor q = at::empty(s, x.options().dtype(at::kChar)), sum;
    s.pop_back();
    Tensor scale = at::empty(s, x.options().dtype(at::kFloat));
    if (residual.defined()) sum = at::empty(x.sizes(), x.options());
    srvp_rms_norm_desc d = {};
    d.x = ptr(x2); d.residual = ptr(r2); d.w = (const float*)ptr(w); d.sum = ptr(sum); d.q8 = ptr(q); d.scale = (float*)ptr(scale);
    d.N = N; d.xs = row_stride(x2); d.rs = row_stride(r2); d.ss = N; d.qs = P; d.M = x2.size(0); d.eps = (float)eps; d.elem_f32 = f32(x);
    check(lib.srvp_rms_norm(&d, stream_of(q)), "srvp_rms_norm");
    if (P != N) q = q.narrow(-1, 0, N);
    return sum.defined() ? py::make_tuple(q, scale, sum) : py::make_tuple(q, scale);
}
py::tuple rms_norm_int8(const Tensor& x, const Tensor& weight, const Maybe& residual, double eps) { return rows_int8("rms_norm_int8", x, weight, get(residual), eps); }
py::tuple quantize_int8(const Tensor& x) { return rows_int8("quantize_int8", x, Tensor(), Tensor(), 0.0); }

Tensor linear_int8(const Tensor& x, const Tensor& x_scale, const Tensor& w0, const Tensor& w_scale, const Maybe& bias, at::ScalarType out) {
    const char* what = "linear_int8";
    on_device(what, x);
    if (x.scalar_type() != at::kChar || w0.scalar_type() != at::kChar) type_error(std::string(what) + ": x and w are int8 tensors, got " + dtype(x) + " and " + dtype(w0));
    if (x.dim() < 1 || w0.dim() != 2 || x.size(-1) != w0.size(1)) value_error(std::string(what) + ": x (..., K) and w (N, K), got " + shape(x) + " and " + shape(w0));
    const int64_t N = w0.size(0), K = w0.size(1);
    if (K > 131071) value_error(std::string(what) + ": the sum of " + std::to_string(K) + " products could pass 32 bits (at most 131071)");
    const auto scales = [&](const Tensor& t, at::IntArrayRef s, const char* name) {
        if (t.scalar_type() != at::kFloat || t.sizes() != s) value_error(std::string(what) + ": " + name + " is a float32 tensor, one value a " + (t.is_same(x_scale) ? "row of x" : "row of w") + ", got " + shape(t) + " " + dtype(t));
    };
    std::vector<int64_t> s = x.sizes().vec();
    s.pop_back();
    scales(x_scale, s, "x_scale");
    scales(w_scale, {N}, "w_scale");
    const Tensor b0 = get(bias);
    if (bias) scales(b0, {N}, "bias");
    if (out != at::kFloat && out != at::kBFloat16) type_error(std::string(what) + ": float32 or bfloat16 output");
    same_device(what, x, {&x_scale, &w0, &w_scale, &b0});
    no_tangent(what, {&x_scale, &w_scale, &b0});
    no_gradient(what, {&x_scale, &w_scale, &b0});
    const c10::DeviceGuard guard(x.device());
    s.push_back(N);
    Tensor y = at::empty(s, x.options().dtype(out));
    if (K == 0) return bias ? y.copy_(b0.expand_as(y)) : y.zero_();
    const Tensor x2 = matrix(x), w = inner(w0), xs = x_scale.contiguous(), ws = w_scale.contiguous(), b = bias ? b0.contiguous() : b0;
    if (x2.size(0) >= (1LL << 31) || N >= (1LL << 31)) value_error(std::string(what) + ": fewer than 2^31 rows");
    srvp_linear_int8_desc d = {};
    d.x = ptr(x2); d.w = ptr(w); d.x_scale = (const float*)ptr(xs); d.w_scale = (const float*)ptr(ws); d.bias = (const float*)ptr(b); d.y = ptr(y);
    d.ldx = x2.stride(0); d.ldw = w.stride(0); d.ldy = N; d.M = x2.size(0); d.N = N; d.K = K; d.out_f32 = out == at::kFloat;
    check(lib.srvp_linear_int8(&d, stream_of(y)), "srvp_linear_int8");
    return y;
}

}  // namespace

PYBIND11_MODULE(_temporal, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const HipError& e) {
            PyErr_SetString(hip_error ? hip_error : PyExc_RuntimeError, e.what());
        } catch (const c10::OutOfMemoryError& e) {
            PyErr_SetString(memory_error ? memory_error : PyExc_RuntimeError, e.what_without_backtrace());
        }
    });
    m.def("bind", &bind);
    m.def("linear_attention", &linear_attention);
    m.def("linear_attention_backward", &linear_attention_backward);
    m.def("linear_attention_step", &linear_attention_step);
    m.def("rotary", &rotary);
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_backward", &rms_norm_backward);
    m.def("rms_norm_int8", &rms_norm_int8);
    m.def("quantize_int8", &quantize_int8);
    m.def("linear_int8", &linear_int8);
}
