// Host glue of flash_cqt.sequence and flash_cqt.optim for ordinary calls: arguments, outputs, autograd nodes and the
// launch in one C++ call (host code only; the kernels are libflashcqt_seq.so's, reached through the C ABI function
// pointers that Python passes in). A token's attention takes 3 us on the GPU and 6 us a call from here, 23 us from
// Python; a small training pass 62 to 68 us against 150. Every function returns None for a call that is not plain (another
// type or device, tensor subclasses, function or dispatch modes, functorch, tracing, tangents, arguments that do not
// fit): the Python path, which has the same results, then takes it, or says what is wrong with it.
#include <cmath>
#include <string>
#include <vector>

#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "../../include/flashcqt_seq.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

struct Calls {
    decltype(&fcqt_head_norm_rotary) norm;
    decltype(&fcqt_head_norm_rotary_partial) norm_partial;
    decltype(&fcqt_head_norm_rotary_bwd) norm_bwd;
    decltype(&fcqt_decay_attention_workspace) attention_workspace;
    decltype(&fcqt_decay_attention) attention;
    decltype(&fcqt_decay_attention_bwd) attention_bwd;
    decltype(&fcqt_decay_attention_step) step;
    decltype(&fcqt_adamw) adamw;
    decltype(&fcqt_adamw_drawn) adamw_drawn;
    decltype(&fcqt_adamw_read) read;
} lib;

// _seq_native.check's error for a status, as a C++ exception
void check(int status, const char* what) {
    if (!status) return;
    py::gil_scoped_acquire gil;
    try {
        py::module_::import("flash_cqt._seq_native").attr("check")(status, what);
    } catch (py::error_already_set& err) {
        err.restore();
    }
    python_error err;
    err.persist();
    throw std::move(err);
}

template <typename F>
auto guarded(F f) {
    try {
        return f();
    } catch (python_error& e) {
        e.restore();
        throw py::error_already_set();
    }
}

bool plain_call() {
    return !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::impl::torch_function_mode_enabled() &&
           !torch::jit::tracer::isTracing() &&
           !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
           !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Functionalize);
}

// A strided tensor of the given GPU with values of its own, no subclass, tangent, lazy conjugation or negation.
bool plain(const Tensor& t, at::ScalarType type, int device) {
    static const c10::DispatchKeySet odd({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                          c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                          c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
                                          c10::DispatchKey::ZeroTensor});
    return t.defined() && t.is_cuda() && !t.key_set().has_any(odd) && t.layout() == c10::kStrided &&
           t.scalar_type() == type && t.get_device() == device &&
           (!t.unsafeGetTensorImpl()->autograd_meta() || !t._fw_grad(0).defined());
}

// (asking for the current GPU fails where there is none: a CPU tensor's call must get to the Python path's error)
bool plain(const Tensor& t, at::ScalarType type) { return t.defined() && t.is_cuda() && plain(t, type, c10::hip::current_device()); }

// What a kernel wrote in place: autograd must see that a graph's saved tensor has changed.
void written(const Tensor& t) {
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool plain_or_none(const Tensor& t, at::ScalarType type) { return !t.defined() || (plain(t, type) && t.is_contiguous()); }

int kind_of(at::ScalarType type) {
    return type == at::kFloat ? FCQT_F32 : type == at::kBFloat16 ? FCQT_BF16 : type == at::kHalf ? FCQT_F16 : -1;
}

// the tensors' requires_grad, where gradients are recorded
template <typename... T>
bool wants_grad(const T&... t) {
    return at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
}

// a last dimension that lies contiguously, heads that the kernels take
bool heads_fit(const Tensor& t, int most) {
    const int64_t d = t.size(-1);
    return t.stride(-1) == 1 && d >= 8 && d <= most && d % 8 == 0 && t.size(-2) >= 1;
}

// [batch][tokens][heads][dim], or without tokens
fcqt_heads heads(const Tensor& t) {
    if (t.dim() == 3) return {t.data_ptr(), t.stride(0), 0, t.stride(1), int32_t(t.size(1))};
    return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2), int32_t(t.size(2))};
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// Gradients that may not be differentiated again, as once_differentiable's
variable_list once(variable_list g) {
    if (!at::GradMode::is_enabled()) return g;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", g.size());
    variable_list fresh;
    for (const Tensor& t : g) fresh.push_back(t.defined() ? t.detach().requires_grad_(true) : t);
    return (*error)(std::move(fresh));
}

Tensor contiguous_last(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

// What a node saves. Saved-tensor hooks may give it back with other strides, but nothing else may have changed.
struct Kept : torch::CustomClassHolder {
    struct One {
        at::DimVector sizes;
        at::ScalarType type;
        at::Device device;
    };
    std::vector<std::optional<One>> all;
};

void keep(AutogradContext* ctx, const variable_list& list) {
    const auto k = c10::make_intrusive<Kept>();
    for (const Tensor& t : list)
        k->all.push_back(t.defined() ? std::optional<Kept::One>({at::DimVector(t.sizes()), t.scalar_type(), t.device()}) : std::nullopt);
    ctx->saved_data["kept"] = c10::IValue::make_capsule(k);
    ctx->save_for_backward(list);
}

variable_list kept(AutogradContext* ctx) {
    const auto k = c10::static_intrusive_pointer_cast<Kept>(ctx->saved_data["kept"].toCapsule());
    variable_list list = ctx->get_saved_variables();
    for (size_t i = 0; i < list.size(); ++i) {
        const auto& one = k->all[i];
        TORCH_CHECK(!one || (list[i].defined() && list[i].sizes() == at::IntArrayRef(one->sizes) && list[i].scalar_type() == one->type &&
                             list[i].device() == one->device),
                    "a saved tensor came back with another shape, type or device");
    }
    return list;
}

Tensor contiguous(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// t as a node saves it, no input of its graph
Tensor saved_form(const Tensor& t) { return !t.defined() ? t : t.is_inference() ? t.clone() : t.detach(); }

// ------------------------------------------------- head norm and rotary positions

struct Rotary : torch::CustomClassHolder {
    Tensor positions, freq;         // until the node has saved them
    fcqt_rotary rot{};
    double eps;
    bool norm;
};
using Turn = c10::intrusive_ptr<Rotary>;

variable_list norm_rotary_out(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Rotary& r) {
    const Tensor oq = at::empty(q.sizes(), q.options()), ok = at::empty(k.sizes(), k.options());
    const fcqt_heads hq = heads(q), hk = heads(k);
    if (q.size(0) && q.size(1))
        check(lib.norm(&hq, &hk, &r.rot, floats(wq), floats(wk), oq.data_ptr(), ok.data_ptr(), q.size(0), q.size(1),
                       int32_t(q.size(3)), kind_of(q.scalar_type()), r.norm, float(r.eps), stream_of(q)),
              "head_norm_rotary");
    return {oq, ok};
}

struct NormRotary : torch::autograd::Function<NormRotary> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Maybe& wq_,
                                 const Maybe& wk_, const Turn& r) {
        const Tensor wq = wq_.value_or(Tensor()), wk = wk_.value_or(Tensor());
        ctx->saved_data["turn"] = c10::IValue::make_capsule(r);
        // (positions and frequencies are saved too: a change of them in place before the backward pass is seen)
        keep(ctx, {q, k, wq, wk, saved_form(r->positions), saved_form(r->freq)});
        r->positions = r->freq = Tensor();
        return norm_rotary_out(q, k, wq, wk, *r);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& g) {
        const auto saved = kept(ctx);
        variable_list out;
        {
            at::AutoGradMode off(false);
            const Tensor q = contiguous_last(saved[0]), k = contiguous_last(saved[1]), wq = contiguous(saved[2]);
            const Tensor wk = contiguous(saved[3]), positions = contiguous(saved[4]), freq = contiguous(saved[5]);
            const Turn r = c10::static_intrusive_pointer_cast<Rotary>(ctx->saved_data["turn"].toCapsule());
            fcqt_rotary rot = r->rot;
            rot.positions = floats(positions), rot.freq = floats(freq);
            const Tensor gq = contiguous_last(g[0]), gk = contiguous_last(g[1]);
            const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
            const int64_t B = q.size(0), T = q.size(1);
            const int32_t D = int32_t(q.size(3)), kind = kind_of(q.scalar_type());
            const auto fp32 = q.options().dtype(at::kFloat);
            const bool some = B && T;
            Tensor dw, partial;
            if (wq.defined() || wk.defined()) {
                dw = some ? at::empty({2, D}, fp32) : at::zeros({2, D}, fp32);
                if (some) partial = at::empty({lib.norm_partial(B, T, int32_t(q.size(2) + k.size(2)), D, kind)}, fp32);
            }
            if (some) {
                const fcqt_heads hq = heads(q), hk = heads(k), hgq = heads(gq), hgk = heads(gk);
                check(lib.norm_bwd(&hq, &hk, &hgq, &hgk, &rot, floats(wq), floats(wk), dq.data_ptr(), dk.data_ptr(),
                                   floats(dw), floats(partial), B, T, D, kind, r->norm, float(r->eps), stream_of(q)),
                      "head_norm_rotary backward");
            }
            out = {dq, dk, wq.defined() ? dw[0] : Tensor(), wk.defined() ? dw[1] : Tensor(), Tensor()};
        }
        return once(std::move(out));
    }
};

py::object norm_rotary(const Tensor& q, const Tensor& k, const Maybe& positions,
                       const Maybe& freq, const std::vector<int64_t>& sections,
                       const Maybe& wq_, const Maybe& wk_, double eps, bool interleaved,
                       bool norm) {
    const Tensor wq = wq_.value_or(Tensor()), wk = wk_.value_or(Tensor());
    if (!q.defined() || !k.defined()) return py::none();
    const auto type = q.scalar_type();
    if (!plain_call() || kind_of(type) < 0 || !plain(q, type) || !plain(k, type) || q.dim() != 4 || k.dim() != 4 ||
        !heads_fit(q, FCQT_SEQ_MAX_DIM) || !heads_fit(k, FCQT_SEQ_MAX_DIM) || !(eps >= 0))
        return py::none();
    const int64_t B = q.size(0), T = q.size(1), D = q.size(3), axes = sections.size();
    if (k.size(0) != B || k.size(1) != T || k.size(3) != D) return py::none();
    for (const Tensor& w : {wq, wk})
        if (w.defined() && (!norm || !plain_or_none(w, at::kFloat) || w.dim() != 1 || w.size(0) != D)) return py::none();
    const auto r = c10::make_intrusive<Rotary>();
    r->eps = eps;
    r->norm = norm;
    if (positions.has_value() != freq.has_value() || positions.has_value() != (axes > 0) || axes > FCQT_ROTARY_AXES)
        return py::none();
    if (axes) {
        const Tensor &p = *positions, &f = *freq;
        if (!plain_or_none(p, at::kFloat) || !plain_or_none(f, at::kFloat) || f.dim() != 1) return py::none();
        int64_t pairs = 0;
        for (int64_t i = 0; i < axes; ++i) {
            if (sections[i] < 0 || sections[i] > D) return py::none();
            r->rot.ends[i] = int32_t(pairs += sections[i]);
        }
        const bool each = p.dim() == 3;
        if (2 * pairs > D || (!interleaved && pairs % 4) || f.size(0) != pairs || p.dim() < 2 || p.dim() > 3 ||
            p.size(-1) != axes || p.size(-2) != T || (each && p.size(0) != B))
            return py::none();
        if (pairs) {
            r->positions = p, r->freq = f;
            r->rot.positions = p.data_ptr<float>(), r->rot.freq = f.data_ptr<float>();
            r->rot.positions_batch = each ? T * axes : 0;
            r->rot.axes = int32_t(axes), r->rot.interleaved = interleaved;
        }
    }
    return guarded([&]() -> py::object {
        variable_list y;
        {
            py::gil_scoped_release nogil;
            y = wants_grad(q, k, wq, wk) ? NormRotary::apply(q, k, wq_, wk_, r) : norm_rotary_out(q, k, wq, wk, *r);
        }
        return py::make_tuple(y[0], y[1]);
    });
}

// ------------------------------------------------------- attention with a decay

bool placed(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// whether the kernels over whole sequences can read it as it lies (16 bytes at a time, 32-bit offsets inside a chunk)
bool wide(const Tensor& t) {
    const int64_t e = t.element_size(), b = t.stride(0), n = t.stride(1), h = t.stride(2);
    return t.stride(3) == 1 && placed(t) && (b | n | h) * e % 16 == 0 &&
           n >= 0 && n <= (int64_t(1) << 31) / (64 * e) - FCQT_DECAY_MAX_DIM;
}

// contiguous, at a multiple of 16 bytes
Tensor made_placed(const Tensor& t) {
    const Tensor c = contiguous(t);
    return !c.defined() || placed(c) ? c : c.clone();
}

Tensor made_wide(const Tensor& t) { return wide(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

int64_t workspace_of(const Tensor& q, const Tensor& k, const Tensor& v, bool ragged, int backward) {
    return lib.attention_workspace(q.size(0), q.size(1), int32_t(q.size(2)), int32_t(k.size(2)), int32_t(q.size(3)),
                                   int32_t(v.size(3)), kind_of(q.scalar_type()), ragged, backward);
}

const int32_t* ints(const Tensor& t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }

// o, the last states, the workspace
variable_list attention_out(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& state,
                            const Tensor& lengths, double scale) {
    const int64_t B = q.size(0), T = q.size(1), size = workspace_of(q, k, v, lengths.defined(), 0);
    const auto fp32 = q.options().dtype(at::kFloat);
    const Tensor o = at::empty({B, T, q.size(2), v.size(3)}, q.options());
    const Tensor last = at::empty({B, k.size(2), q.size(3), v.size(3)}, fp32);
    const Tensor work = size ? at::empty({size / 4}, fp32) : Tensor();
    const fcqt_heads hq = heads(q), hk = heads(k), hv = heads(v);
    check(lib.attention(&hq, &hk, &hv, floats(g), ints(lengths), floats(state), floats(last), o.data_ptr(), floats(work),
                        size, B, T, int32_t(q.size(3)), int32_t(v.size(3)), kind_of(q.scalar_type()), float(scale),
                        stream_of(q)),
          "decay_attention");
    return {o, last, work};
}

// (needs_input_grad counts the tensors that are there: the state is the fifth where there is one)
struct DecayAttention : torch::autograd::Function<DecayAttention> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& g, const Maybe& state_, const Maybe& lengths_, double scale) {
        const Tensor state = state_.value_or(Tensor()), lengths = lengths_.value_or(Tensor());
        ctx->set_materialize_grads(false);
        ctx->saved_data["scale"] = scale;
        variable_list y = attention_out(q, k, v, g, state, lengths, scale);
        keep(ctx, {q, k, v, g, state, lengths, y[2]});                  // the workspace: states that segments start from
        y.pop_back();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list out(7);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const auto saved = kept(ctx);
        {
            at::AutoGradMode off(false);
            const Tensor q = made_wide(saved[0]), k = made_wide(saved[1]), v = made_wide(saved[2]), g = contiguous(saved[3]);
            const Tensor state = made_placed(saved[4]), lengths = contiguous(saved[5]), starts = made_placed(saved[6]);
            const int64_t B = q.size(0), T = q.size(1);
            const Tensor go = grads[0].defined() ? made_wide(grads[0])
                                                 : at::zeros({B, T, q.size(2), v.size(3)}, q.options());
            const Tensor glast = made_placed(grads[1]);
            const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
            const Tensor dv = at::empty(v.sizes(), v.options());
            const Tensor dg = ctx->needs_input_grad(3) ? at::empty(g.sizes(), g.options()) : Tensor();
            const Tensor ds = state.defined() && ctx->needs_input_grad(4) ? at::empty(state.sizes(), state.options()) : Tensor();
            const int64_t size = workspace_of(q, k, v, lengths.defined(), dg.defined() ? 2 : 1);
            const Tensor work = size ? at::empty({size / 4}, g.options()) : Tensor();
            const fcqt_heads hq = heads(q), hk = heads(k), hv = heads(v), ho = heads(go);
            check(lib.attention_bwd(&hq, &hk, &hv, floats(g), ints(lengths), floats(state), floats(starts), &ho,
                                    floats(glast), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), floats(dg), floats(ds),
                                    floats(work), size, B, T, int32_t(q.size(3)), int32_t(v.size(3)),
                                    kind_of(q.scalar_type()), float(ctx->saved_data["scale"].toDouble()), stream_of(q)),
                  "decay_attention backward");
            out = {dq, dk, dv, dg, ds, Tensor(), Tensor()};
        }
        return once(std::move(out));
    }
};

bool attention_fits(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, int64_t dims, int most) {
    if (!q.defined()) return false;
    const auto type = q.scalar_type();
    if (!plain_call() || kind_of(type) < 0) return false;
    for (const Tensor& t : {q, k, v})
        if (!plain(t, type) || t.dim() != dims || !heads_fit(t, most)) return false;
    for (int64_t i = 0; i + 2 < dims; ++i)
        if (k.size(i) != q.size(i) || v.size(i) != q.size(i)) return false;
    return k.size(-1) == q.size(-1) && v.size(-2) == k.size(-2) && q.size(-2) % k.size(-2) == 0 && plain(g, at::kFloat) &&
           g.is_contiguous() && g.dim() == 1 && g.size(0) == k.size(-2);
}

py::object attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Maybe& state_,
                     const Maybe& lengths_, std::optional<double> scale_) {
    const Tensor state = state_.value_or(Tensor()), lengths = lengths_.value_or(Tensor());
    if (!attention_fits(q, k, v, g, 4, FCQT_DECAY_MAX_DIM) || q.size(0) > 65535 || !wide(q) || !wide(k) || !wide(v))
        return py::none();
    if (!plain_or_none(state, at::kFloat) || !plain_or_none(lengths, at::kInt)) return py::none();
    if (state.defined() && !placed(state)) return py::none();        // (the Python path copies it)
    if (state.defined() && state.sizes() != at::IntArrayRef({q.size(0), k.size(2), q.size(3), v.size(3)})) return py::none();
    if (lengths.defined() && (lengths.dim() != 1 || lengths.size(0) != q.size(0))) return py::none();
    const double scale = scale_.value_or(std::pow(double(q.size(3)), -0.5));
    return guarded([&]() -> py::object {
        variable_list y;
        {
            py::gil_scoped_release nogil;
            y = wants_grad(q, k, v, g, state) ? DecayAttention::apply(q, k, v, g, state_, lengths_, scale)
                                              : attention_out(q, k, v, g, state, lengths, scale);
        }
        return py::make_tuple(y[0], y[1]);
    });
}

py::object step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& state,
                const Maybe& slots_, std::optional<double> scale) {
    const Tensor slots = slots_.value_or(Tensor());
    if (!attention_fits(q, k, v, g, 3, FCQT_SEQ_MAX_DIM) || wants_grad(q, k, v, g, state)) return py::none();
    const int64_t B = q.size(0), Dk = q.size(2), Dv = v.size(2);
    if (!plain(state, at::kFloat) || !state.is_contiguous() || state.dim() != 4 || state.size(1) != k.size(1) ||
        state.size(2) != Dk || state.size(3) != Dv || !plain_or_none(slots, at::kInt))
        return py::none();
    if (slots.defined() ? slots.dim() != 1 || slots.size(0) != B : state.size(0) < B) return py::none();
    return guarded([&]() -> py::object {
        const Tensor o = at::empty({B, q.size(1), Dv}, q.options());
        const fcqt_heads hq = heads(q), hk = heads(k), hv = heads(v);
        if (B)
            check(lib.step(&hq, &hk, &hv, floats(g), floats(state), ints(slots), o.data_ptr(), B, state.size(0),
                           int32_t(Dk), int32_t(Dv), kind_of(q.scalar_type()),
                           float(scale.value_or(std::pow(double(Dk), -0.5))), stream_of(q)),
                  "decay_attention_step");
        if (B) written(state);
        return py::cast(o);
    });
}

// ---------------------------------------------------------------------- AdamW

int64_t blocks_of(int64_t size) { return (size + FCQT_ADAMW_BLOCK - 1) / FCQT_ADAMW_BLOCK; }

bool held_by(const Tensor& t, at::ScalarType type, int64_t size, int device) {
    return plain(t, type, device) && t.numel() == size && t.is_contiguous();
}

// The values of 8-bit moments into fp32 tensors. True when done.
bool moments(const std::vector<Tensor>& m, const std::vector<Tensor>& v, const std::vector<Tensor>& ms,
             const std::vector<Tensor>& vs, const std::vector<Tensor>& om, const std::vector<Tensor>& ov) {
    const size_t n = m.size();
    if (!n || v.size() != n || ms.size() != n || vs.size() != n || om.size() != n || ov.size() != n || !plain_call()) return false;
    if (!m[0].defined() || !m[0].is_cuda()) return false;
    const int device = c10::hip::current_device();
    std::vector<fcqt_adamw_tensor> ts(n);
    for (size_t i = 0; i < n; ++i) {
        const int64_t size = m[i].defined() ? m[i].numel() : 0;
        if (!held_by(m[i], at::kByte, size, device) || !held_by(v[i], at::kByte, size, device) ||
            !held_by(om[i], at::kFloat, size, device) || !held_by(ov[i], at::kFloat, size, device) ||
            !held_by(ms[i], at::kFloat, blocks_of(size), device) || !held_by(vs[i], at::kFloat, blocks_of(size), device))
            return false;
        ts[i] = {om[i].data_ptr(), ov[i].data_ptr(), m[i].data_ptr(), v[i].data_ptr(), floats(ms[i]), floats(vs[i]), size};
    }
    guarded([&] { check(lib.read(ts.data(), int64_t(n), stream_of(m[0])), "read_moments"); });
    for (const auto* list : {&om, &ov})
        for (const Tensor& t : *list) written(t);
    return true;
}

// True when done. Tensors of one type on the current GPU; factors as _seq_native.AdamwFactors has them. seed: 8-bit codes
// are drawn.
bool adamw(const std::vector<Tensor>& p, const std::vector<Tensor>& g, const std::vector<Tensor>& m,
           const std::vector<Tensor>& v, const std::vector<Tensor>& ms, const std::vector<Tensor>& vs, bool eight,
           const std::vector<double>& factors, const Maybe& grad_scale, std::optional<uint64_t> seed, int64_t step) {
    const size_t n = p.size();
    if (!n || g.size() != n || m.size() != n || v.size() != n || factors.size() != 8 || !plain_call() ||
        !p[0].defined() || !p[0].is_cuda() || kind_of(p[0].scalar_type()) < 0 || (eight && (ms.size() != n || vs.size() != n)))
        return false;
    const auto type = p[0].scalar_type(), held = eight ? at::kByte : at::kFloat;
    if (grad_scale && (!plain(*grad_scale, at::kFloat) || grad_scale->numel() != 1)) return false;
    std::vector<fcqt_adamw_tensor> ts(n);
    const int device = c10::hip::current_device();
    for (size_t i = 0; i < n; ++i) {
        const int64_t size = p[i].defined() ? p[i].numel() : 0;
        if (!held_by(p[i], type, size, device) || !held_by(g[i], type, size, device) || !held_by(m[i], held, size, device) ||
            !held_by(v[i], held, size, device))
            return false;
        if (eight && (!held_by(ms[i], at::kFloat, blocks_of(size), device) || !held_by(vs[i], at::kFloat, blocks_of(size), device)))
            return false;
        ts[i] = {p[i].data_ptr(), g[i].data_ptr(), m[i].data_ptr(), v[i].data_ptr(),
                 eight ? floats(ms[i]) : nullptr, eight ? floats(vs[i]) : nullptr, size};
    }
    const fcqt_adamw_factors f{float(factors[0]), float(factors[1]), float(factors[2]), float(factors[3]),
                               float(factors[4]), float(factors[5]), float(factors[6]), float(factors[7])};
    const float* gs = grad_scale ? floats(*grad_scale) : nullptr;
    guarded([&] {
        check(eight && seed ? lib.adamw_drawn(ts.data(), int64_t(n), kind_of(type), &f, gs, *seed, step, stream_of(p[0]))
                            : lib.adamw(ts.data(), int64_t(n), kind_of(type), eight ? 8 : 32, &f, gs, stream_of(p[0])),
              "adamw_step");
    });
    for (const auto* list : {&p, &m, &v, &ms, &vs})
        for (const Tensor& t : *list) written(t);
    return true;
}

void attach(int64_t norm, int64_t norm_partial, int64_t norm_bwd, int64_t attention_workspace, int64_t attention,
            int64_t attention_bwd, int64_t step, int64_t adamw, int64_t adamw_drawn, int64_t read) {
    lib = {reinterpret_cast<decltype(lib.norm)>(norm), reinterpret_cast<decltype(lib.norm_partial)>(norm_partial),
           reinterpret_cast<decltype(lib.norm_bwd)>(norm_bwd),
           reinterpret_cast<decltype(lib.attention_workspace)>(attention_workspace),
           reinterpret_cast<decltype(lib.attention)>(attention), reinterpret_cast<decltype(lib.attention_bwd)>(attention_bwd),
           reinterpret_cast<decltype(lib.step)>(step), reinterpret_cast<decltype(lib.adamw)>(adamw),
           reinterpret_cast<decltype(lib.adamw_drawn)>(adamw_drawn),
           reinterpret_cast<decltype(lib.read)>(read)};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.attr("abi_version") = FCQT_SEQ_ABI_VERSION;
    m.attr("torch_version") = FCQT_TORCH_VERSION;
    m.def("attach", &attach);
    m.def("norm_rotary", &norm_rotary);
    m.def("attention", &attention);
    m.def("step", &step);
    m.def("adamw", &adamw);
    m.def("read", &moments);
}
