// The block operators as autograd operators in C++ (block_ops.py checks the arguments and calls these; the
// kernels are libnbx.so's, include/nbx.h "Block operators").  A training pass through one of them is a few
// launches of a few microseconds each: with the backward pass in Python the interpreter, entered on autograd's
// own thread, took longer than the kernels (layer scale of 6400 x 128: 125 us a pass, of which 15 on the GPU).
// Built by build.py with the host compiler.  Entry points are handed over by address, so this file's calls go
// to the library that the package has loaded.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <cstring>
#include <tuple>
#include <unordered_map>

#include "../../include/nbx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Entries {
    decltype(&nbx_last_error) last_error = nullptr;
    decltype(&nbx_dropout) dropout = nullptr;
    decltype(&nbx_residual_norm) residual = nullptr;
    decltype(&nbx_residual_norm_backward_workspace_bytes) residual_ws = nullptr;
    decltype(&nbx_residual_norm_backward) residual_bwd = nullptr;
    decltype(&nbx_sh_residual_norm) sh = nullptr;
    decltype(&nbx_sh_residual_norm_backward_workspace_bytes) sh_ws = nullptr;
    decltype(&nbx_sh_residual_norm_backward) sh_bwd = nullptr;
    decltype(&nbx_segment_attention_workspace_bytes) attention_ws = nullptr;
    decltype(&nbx_segment_attention) attention = nullptr;
    decltype(&nbx_segment_attention_backward) attention_bwd = nullptr;
};
Entries entries;
PyObject* error_type = nullptr;   // _lib.NbxError

// NbxError in Python, also from autograd's threads
[[noreturn]] void fail(const std::string& what) {
    pybind11::gil_scoped_acquire gil;
    PyErr_SetString(error_type, what.c_str());
    python_error e;
    e.persist();
    throw e;
}

void check(int rc, const char* what) {
    if (rc) fail(std::string(what) + ": " + entries.last_error() + " (code " + std::to_string(rc) + ")");
}

void first_derivatives_only() {
    if (at::GradMode::is_enabled())
        fail("block operators have no second derivatives (a backward pass with create_graph)");
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

template <typename T = void>
T* ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
Tensor value_or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// A new contiguous tensor, from the allocator at once: the dispatcher's way to it takes as long again, and on
// autograd's thread a pass allocates up to nine.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& on) {
    return Tensor(at::detail::empty_cuda(sizes, type, on.device(), std::nullopt));
}
Tensor fresh_like(const Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }
Tensor empty_if(bool wanted, const Tensor& like) { return wanted && like.defined() ? fresh_like(like) : Tensor(); }
Tensor used_state(const Tensor& state) { return state.defined() ? fresh_like(state) : Tensor(); }

constexpr at::ScalarType TYPES[] = {at::kFloat, at::kBFloat16, at::kHalf};   // NBX_F32, NBX_BF16, NBX_F16

// A saved tensor as it was saved: hooks (torch.autograd.graph.saved_tensors_hooks) may give back any other.
// Contiguous but for the residual rows, whose strides are asked for (rows_of).
Tensor unchanged(const Tensor& t, int64_t numel, at::ScalarType type, const Tensor& on) {
    if (t.defined() && (t.numel() != numel || t.scalar_type() != type || t.device() != on.device()))
        fail("a saved tensor came back as another: " + std::to_string(t.numel()) + " x " + toString(t.scalar_type()) +
             " on " + t.device().str() + ", saved were " + std::to_string(numel) + " x " + toString(type) + " on " +
             on.device().str());
    return t;
}
Tensor restored(const Tensor& t, int64_t numel, at::ScalarType type, const Tensor& on) {
    return dense(unchanged(t, numel, type, on));
}

Tensor workspace(size_t bytes, const Tensor& on) {
    return bytes ? fresh({(int64_t)bytes}, at::kByte, on) : Tensor();
}

// Whether the call is recorded.  A dual tensor (forward-mode derivatives) need not require a gradient, and its
// tangent would be lost without a word: refused.
bool wants_grad(std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->defined() && t->_fw_grad(0).defined()) fail("block operators have no forward-mode derivatives");
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// ---------------------------------------------------------------- dropout
struct DropoutHow {
    int64_t dtype, per, n, S, C, group, threshold, call;
};

Tensor run_dropout(const Tensor& x, const DropoutHow& h, const Tensor& state, const Tensor& used) {
    Tensor y = fresh_like(x);
    c10::DeviceGuard guard(x.device());
    check(entries.dropout((int32_t)h.dtype, (int32_t)h.per, h.n, h.S, h.C, h.group, (uint32_t)h.threshold,
                          ptr<int64_t>(state), (uint32_t)h.call, ptr<int64_t>(used), x.data_ptr(), y.data_ptr(),
                          stream_of(x)),
          "nbx_dropout");
    return y;
}

struct DropoutFn : torch::autograd::Function<DropoutFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& state, const DropoutHow& h) {
        Tensor used = fresh_like(state);
        Tensor y = run_dropout(x, h, state, used);
        ctx->save_for_backward({used});
        ctx->saved_data["how"] = std::vector<int64_t>{h.dtype, h.per, h.n, h.S, h.C, h.group, h.threshold, h.call};
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& dy) {
        first_derivatives_only();
        const auto v = ctx->saved_data["how"].toIntVector();
        const DropoutHow h{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
        const Tensor used = restored(ctx->get_saved_variables()[0], 2, at::kLong, dy[0]);
        return {run_dropout(dy[0].contiguous(), h, used, Tensor()), Tensor(), Tensor()};
    }
};

Tensor dropout(const Tensor& x_, const Tensor& state, int64_t dtype, int64_t per, int64_t n, int64_t S, int64_t C,
               int64_t group, int64_t threshold, int64_t call) {
    const DropoutHow h{dtype, per, n, S, C, group, threshold, call};
    const Tensor x = x_.contiguous();
    return wants_grad({&x}) ? DropoutFn::apply(x, state, h) : run_dropout(x, h, state, Tensor());
}

// ---------------------------------------------------------------- residual add, norms, gate
// a plain struct of the call's numbers, kept as bytes: pointers are filled in per direction
template <typename Args>
std::string bytes_of(const Args& a) {
    return std::string(reinterpret_cast<const char*>(&a), sizeof(a));
}
template <typename Args>
Args args_of(AutogradContext* ctx) {
    Args a;
    const std::string& s = ctx->saved_data["how"].toStringRef();
    TORCH_INTERNAL_ASSERT(s.size() == sizeof(a));
    memcpy(&a, s.data(), sizeof(a));
    return a;
}

using ResidualArgs = nbx_residual_norm_args;

// (tensor, elements between its rows): strided rows are read in place, anything else is copied
std::pair<Tensor, int64_t> rows_of(const Tensor& t, int64_t C) {
    if (t.dim() == 2 && t.size(0) > 1 && t.size(1) == C && t.stride(1) == 1 && t.stride(0) >= C) return {t, t.stride(0)};
    return {t.contiguous(), C};
}

void set_params(ResidualArgs& a, const Tensor& gate, const Tensor& post_w, const Tensor& post_b, const Tensor& pre_w,
                const Tensor& pre_b) {
    a.gate = ptr(gate);
    a.post_w = ptr(post_w);
    a.post_b = ptr(post_b);
    a.pre_w = ptr(pre_w);
    a.pre_b = ptr(pre_b);
}

std::pair<Tensor, Tensor> run_residual(ResidualArgs a, const Tensor& x, const Tensor& y, const Tensor& state,
                                       const Tensor& used, const Tensor& stats) {
    Tensor h = fresh_like(x), z;
    if (a.pre_w) z = fresh_like(y);
    a.x = x.data_ptr();
    a.y = y.data_ptr();
    a.rng = ptr<int64_t>(state);
    a.used = ptr<int64_t>(used);
    a.h = h.data_ptr();
    a.z = ptr(z);
    a.stats = ptr<float>(stats);
    c10::DeviceGuard guard(x.device());
    check(entries.residual(&a, stream_of(x)), "nbx_residual_norm");
    return {h, z};
}

struct ResidualFn : torch::autograd::Function<ResidualFn> {
    // h, or h and z: an undefined output is no output of autograd's
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const OptTensor& gate_,
                                 const OptTensor& post_w_, const OptTensor& post_b_, const OptTensor& pre_w_,
                                 const OptTensor& pre_b_, const OptTensor& state_, ResidualArgs a) {
        const Tensor gate = value_or_none(gate_), post_w = value_or_none(post_w_), post_b = value_or_none(post_b_),
                     pre_w = value_or_none(pre_w_), pre_b = value_or_none(pre_b_), state = value_or_none(state_);
        const bool norms = post_w.defined() || pre_w.defined();
        Tensor used = used_state(state), stats;
        if (norms) stats = fresh({4, a.rows}, at::kFloat, x);
        ctx->saved_data["how"] = bytes_of(a);
        set_params(a, gate, post_w, post_b, pre_w, pre_b);
        auto [h, z] = run_residual(a, x, y, state, used, stats);
        // y is read again for its norm and the gate's gradient; for the norm behind the sum h, or in 16 bits x and y
        const bool again = z.defined() && a.x_dtype != NBX_F32;
        const bool keep_y = again || post_w.defined() || (gate.defined() && gate.requires_grad());
        ctx->save_for_backward({keep_y ? y : Tensor(), again ? x : z.defined() ? h : Tensor(), gate, post_w, post_b, pre_w, pre_b, used,
                                stats});
        ctx->saved_data["x"] = x.sizes().vec();
        ctx->set_materialize_grads(false);
        if (z.defined()) return {h, z};
        return {h};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& g) {
        first_derivatives_only();
        variable_list out(9);
        const Tensor dh = dense(g[0]), dz = g.size() > 1 ? dense(g[1]) : Tensor();
        if (!dh.defined() && !dz.defined()) return out;
        auto a = args_of<ResidualArgs>(ctx);
        auto s = ctx->get_saved_variables();
        const Tensor& any = dh.defined() ? dh : dz;
        const at::ScalarType param = TYPES[a.param_dtype];
        for (int i = 2; i < 7; ++i) s[i] = restored(s[i], i == 2 ? a.gate_groups * a.C : a.C, param, any);
        const Tensor used = restored(s[7], 2, at::kLong, any), stats = restored(s[8], 4 * a.rows, at::kFloat, any);
        Tensor y = unchanged(s[0], a.rows * a.C, TYPES[a.y_dtype], any), h = unchanged(s[1], a.rows * a.C, TYPES[a.x_dtype], any), x;
        if (h.defined() && a.x_dtype != NBX_F32) {
            std::tie(x, a.ldx) = rows_of(h, a.C);
            h = Tensor();
        }
        h = dense(h);
        if (y.defined()) std::tie(y, a.ldy) = rows_of(y, a.C);
        set_params(a, s[2], s[3], s[4], s[5], s[6]);
        const auto shape = ctx->saved_data["x"].toIntVector();
        if (ctx->needs_input_grad(0)) out[0] = fresh(shape, TYPES[a.x_dtype], any);
        if (ctx->needs_input_grad(1)) out[1] = fresh(shape, TYPES[a.y_dtype], any);
        // without dz nothing reaches the norm behind the sum: its parameters' gradients are 0
        for (int i = 2, edge = 2; i < 7; ++i)   // an absent input has no edge
            if (s[i].defined()) out[i] = empty_if(ctx->needs_input_grad(edge++), s[i]);
        a.x = ptr(x);
        a.y = ptr(y);
        a.h = ptr(h);
        a.rng = ptr<int64_t>(used);
        a.stats = ptr<float>(stats);
        a.dh = ptr(dh);
        a.dz = ptr(dz);
        a.dx = ptr(out[0]);
        a.dy = ptr(out[1]);
        a.dgate = ptr(out[2]);
        a.dpost_w = ptr(out[3]);
        a.dpost_b = ptr(out[4]);
        a.dpre_w = ptr(out[5]);
        a.dpre_b = ptr(out[6]);
        c10::DeviceGuard guard(any.device());
        check(entries.residual_ws(&a, &a.workspace_bytes), "nbx_residual_norm_backward_workspace_bytes");
        const Tensor ws = workspace(a.workspace_bytes, any);
        a.workspace = ptr(ws);
        check(entries.residual_bwd(&a, stream_of(any)), "nbx_residual_norm_backward");
        return out;
    }
};

std::pair<Tensor, OptTensor> residual_norm(const Tensor& x_, const Tensor& y_, const OptTensor& gate_,
                                           const OptTensor& post_w_, const OptTensor& post_b_, const OptTensor& pre_w_,
                                           const OptTensor& pre_b_, const OptTensor& state_, int64_t x_dtype,
                                           int64_t y_dtype, int64_t param_dtype, int64_t norm, double eps, double scale,
                                           int64_t threshold, int64_t group, int64_t call) {
    const int64_t C = x_.size(-1);
    const auto [x, ldx] = rows_of(x_, C);
    const auto [y, ldy] = rows_of(y_, C);
    const Tensor gate = dense(value_or_none(gate_)), post_w = dense(value_or_none(post_w_)),
                 post_b = dense(value_or_none(post_b_)), pre_w = dense(value_or_none(pre_w_)),
                 pre_b = dense(value_or_none(pre_b_)), state = value_or_none(state_);
    ResidualArgs a = {};
    a.rows = x.numel() / C;
    a.C = C;
    a.ldx = ldx;
    a.ldy = ldy;
    a.gate_groups = gate.defined() ? gate.numel() / C : 0;
    a.group = group;
    a.x_dtype = (int32_t)x_dtype;
    a.y_dtype = (int32_t)y_dtype;
    a.param_dtype = (int32_t)param_dtype;
    a.norm = (int32_t)norm;
    a.eps = (float)eps;
    a.scale = (float)scale;
    a.threshold = (uint32_t)threshold;
    a.call = (uint32_t)call;
    if (wants_grad({&x, &y, &gate, &post_w, &post_b, &pre_w, &pre_b})) {
        const auto out = ResidualFn::apply(x, y, opt(gate), opt(post_w), opt(post_b), opt(pre_w), opt(pre_b), state_, a);
        return {out[0], out.size() > 1 ? OptTensor(out[1]) : OptTensor()};
    }
    set_params(a, gate, post_w, post_b, pre_w, pre_b);
    auto [h, z] = run_residual(a, x, y, state, Tensor(), Tensor());
    return {h, opt(z)};
}

// ---------------------------------------------------------------- residual add, spherical-harmonics norm
using ShArgs = nbx_sh_residual_norm_args;

std::pair<Tensor, Tensor> run_sh(ShArgs a, const Tensor& x, const Tensor& y, const Tensor& weight, const Tensor& bias,
                                 const Tensor& state, const Tensor& used, const Tensor& stats) {
    Tensor h = fresh_like(x), z = fresh_like(x);
    a.x = x.data_ptr();
    a.y = y.data_ptr();
    a.weight = weight.data_ptr();
    a.bias = bias.data_ptr();
    a.rng = ptr<int64_t>(state);
    a.used = ptr<int64_t>(used);
    a.h = h.data_ptr();
    a.z = z.data_ptr();
    a.stats = ptr<float>(stats);
    c10::DeviceGuard guard(x.device());
    check(entries.sh(&a, stream_of(x)), "nbx_sh_residual_norm");
    return {h, z};
}

struct ShFn : torch::autograd::Function<ShFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const Tensor& weight,
                                 const Tensor& bias, const OptTensor& state_, const ShArgs& a) {
        const Tensor state = value_or_none(state_);
        Tensor used = used_state(state), stats = fresh({2, a.V}, at::kFloat, x);
        ctx->saved_data["how"] = bytes_of(a);
        auto [h, z] = run_sh(a, x, y, weight, bias, state, used, stats);
        const bool again = a.dtype != NBX_F32;   // the backward pass forms h again from x and y
        ctx->save_for_backward({again ? x : h, weight, bias, used, stats, again ? y : Tensor()});
        ctx->set_materialize_grads(false);
        return {h, z};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& g) {
        first_derivatives_only();
        variable_list out(6);
        const Tensor dh = dense(g[0]), dz = dense(g[1]);
        if (!dh.defined() && !dz.defined()) return out;
        auto a = args_of<ShArgs>(ctx);
        auto s = ctx->get_saved_variables();
        const Tensor& any = dh.defined() ? dh : dz;
        const int64_t L = a.lmax + 1, sizes[] = {a.V * L * L * a.C, L * a.C, a.C, 2, 2 * a.V, a.V * L * L * a.C};
        const at::ScalarType types[] = {TYPES[a.dtype], TYPES[a.param_dtype], TYPES[a.param_dtype], at::kLong, at::kFloat,
                                        TYPES[a.dtype]};
        for (int i = 0; i < 6; ++i) s[i] = restored(s[i], sizes[i], types[i], any);
        for (int i = 0; i < 4; ++i) out[i] = empty_if(ctx->needs_input_grad(i), s[i < 2 ? 0 : i - 1]);
        if (a.dtype != NBX_F32) a.x = ptr(s[0]);
        else a.h = ptr(s[0]);
        a.y = ptr(s[5]);
        a.weight = ptr(s[1]);
        a.bias = ptr(s[2]);
        a.rng = ptr<int64_t>(s[3]);
        a.stats = ptr<float>(s[4]);
        a.dh = ptr(dh);
        a.dz = ptr(dz);
        a.dx = ptr(out[0]);
        a.dy = ptr(out[1]);
        a.dweight = ptr(out[2]);
        a.dbias = ptr(out[3]);
        c10::DeviceGuard guard(s[0].device());
        check(entries.sh_ws(&a, &a.workspace_bytes), "nbx_sh_residual_norm_backward_workspace_bytes");
        const Tensor ws = workspace(a.workspace_bytes, s[0]);
        a.workspace = ptr(ws);
        check(entries.sh_bwd(&a, stream_of(s[0])), "nbx_sh_residual_norm_backward");
        return out;
    }
};

std::pair<Tensor, Tensor> sh_residual_norm(const Tensor& x_, const Tensor& y_, const Tensor& weight_,
                                           const Tensor& bias_, const OptTensor& state_, int64_t lmax, int64_t dtype,
                                           int64_t param_dtype, double eps, int64_t path_threshold, int64_t path_group,
                                           int64_t channel_threshold, int64_t call) {
    const Tensor x = x_.contiguous(), y = y_.contiguous(), weight = weight_.contiguous(), bias = bias_.contiguous(),
                 state = value_or_none(state_);
    ShArgs a = {};
    a.V = x.size(0);
    a.path_group = path_group;
    a.lmax = (int32_t)lmax;
    a.C = (int32_t)x.size(2);
    a.dtype = (int32_t)dtype;
    a.param_dtype = (int32_t)param_dtype;
    a.eps = (float)eps;
    a.path_threshold = (uint32_t)path_threshold;
    a.channel_threshold = (uint32_t)channel_threshold;
    a.call = (uint32_t)call;
    if (wants_grad({&x, &y, &weight, &bias})) {
        const auto out = ShFn::apply(x, y, weight, bias, state_, a);
        return {out[0], out[1]};
    }
    return run_sh(a, x, y, weight, bias, state, Tensor(), Tensor());
}

// ---------------------------------------------------------------- segment attention
using AttentionArgs = nbx_segment_attention_args;

void set_lists(AttentionArgs& a, const Tensor& values, const Tensor& logits, const Tensor& lists, const Tensor& eid) {
    a.values = values.data_ptr();
    a.logits = logits.data_ptr();
    a.ptr = static_cast<const int32_t*>(lists.data_ptr());
    a.eid = static_cast<const int32_t*>(eid.data_ptr());
}

Tensor run_attention(AttentionArgs a, const Tensor& values, const Tensor& logits, const Tensor& lists, const Tensor& eid,
                     const Tensor& state, const Tensor& used, const Tensor& stats) {
    Tensor out = fresh({a.V, a.K, a.H, a.D}, values.scalar_type(), values);
    set_lists(a, values, logits, lists, eid);
    a.rng = ptr<int64_t>(state);
    a.used = ptr<int64_t>(used);
    a.out = out.data_ptr();
    a.stats = ptr<float>(stats);
    c10::DeviceGuard guard(values.device());
    check(entries.attention_ws(&a, 0, &a.workspace_bytes), "nbx_segment_attention_workspace_bytes");
    const Tensor ws = workspace(a.workspace_bytes, values);
    a.workspace = ptr(ws);
    check(entries.attention(&a, stream_of(values)), "nbx_segment_attention");
    return out;
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& values, const Tensor& logits, const Tensor& lists,
                          const Tensor& eid, const OptTensor& state_, const AttentionArgs& a) {
        const Tensor state = value_or_none(state_);
        Tensor used = used_state(state), stats = fresh({2, a.V, a.H}, at::kFloat, values);
        ctx->saved_data["how"] = bytes_of(a);
        Tensor out = run_attention(a, values, logits, lists, eid, state, used, stats);
        ctx->save_for_backward({values, logits, lists, eid, used, stats});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& g) {
        first_derivatives_only();
        variable_list out(6);
        auto a = args_of<AttentionArgs>(ctx);
        auto s = ctx->get_saved_variables();
        const Tensor dout = g[0].contiguous();
        const int64_t sizes[] = {a.E * a.K * a.H * a.D, a.E * a.H, a.V + 1, a.E, 2, 2 * a.V * a.H};
        const at::ScalarType types[] = {TYPES[a.v_dtype], TYPES[a.l_dtype], at::kInt, at::kInt, at::kLong, at::kFloat};
        for (int i = 0; i < 6; ++i) s[i] = restored(s[i], sizes[i], types[i], dout);
        for (int i = 0; i < 2; ++i) out[i] = empty_if(ctx->needs_input_grad(i), s[i]);
        set_lists(a, s[0], s[1], s[2], s[3]);
        a.rng = ptr<int64_t>(s[4]);
        a.stats = ptr<float>(s[5]);
        a.dout = ptr(dout);
        a.dvalues = ptr(out[0]);
        a.dlogits = ptr(out[1]);
        c10::DeviceGuard guard(dout.device());
        check(entries.attention_ws(&a, 1, &a.workspace_bytes), "nbx_segment_attention_workspace_bytes");
        const Tensor ws = workspace(a.workspace_bytes, dout);
        a.workspace = ptr(ws);
        check(entries.attention_bwd(&a, stream_of(dout)), "nbx_segment_attention_backward");
        return out;
    }
};

Tensor segment_attention(const Tensor& values_, const Tensor& logits_, const Tensor& lists_, const Tensor& eid_,
                         const OptTensor& state_, int64_t v_dtype, int64_t l_dtype, int64_t threshold, int64_t call) {
    const Tensor values = values_.contiguous(), logits = logits_.contiguous(), lists = lists_.contiguous(),
                 eid = eid_.contiguous(), state = value_or_none(state_);
    AttentionArgs a = {};
    a.V = lists.numel() - 1;
    a.E = values.size(0);
    a.K = values.size(1);
    a.H = (int32_t)values.size(2);
    a.D = (int32_t)values.size(3);
    a.v_dtype = (int32_t)v_dtype;
    a.l_dtype = (int32_t)l_dtype;
    a.threshold = (uint32_t)threshold;
    a.call = (uint32_t)call;
    if (wants_grad({&values, &logits})) return AttentionFn::apply(values, logits, lists, eid, state_, a);
    return run_attention(a, values, logits, lists, eid, state, Tensor(), Tensor());
}

void bind(const std::unordered_map<std::string, uintptr_t>& at, pybind11::object error) {
    auto set = [&](auto& f, const char* name) { f = reinterpret_cast<std::decay_t<decltype(f)>>(at.at(name)); };
    set(entries.last_error, "nbx_last_error");
    set(entries.dropout, "nbx_dropout");
    set(entries.residual, "nbx_residual_norm");
    set(entries.residual_ws, "nbx_residual_norm_backward_workspace_bytes");
    set(entries.residual_bwd, "nbx_residual_norm_backward");
    set(entries.sh, "nbx_sh_residual_norm");
    set(entries.sh_ws, "nbx_sh_residual_norm_backward_workspace_bytes");
    set(entries.sh_bwd, "nbx_sh_residual_norm_backward");
    set(entries.attention_ws, "nbx_segment_attention_workspace_bytes");
    set(entries.attention, "nbx_segment_attention");
    set(entries.attention_bwd, "nbx_segment_attention_backward");
    error_type = error.release().ptr();   // kept for the process's life
}

}  // namespace

PYBIND11_MODULE(nbx_torch, m) {
    pybind11::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (python_error& e) {
            e.restore();
        }
    });
    m.def("bind", &bind);
    m.attr("abi_version") = NBX_ABI_VERSION;
    m.def("dropout", &dropout);
    m.def("residual_norm", &residual_norm);
    m.def("sh_residual_norm", &sh_residual_norm);
    m.def("segment_attention", &segment_attention);
}
