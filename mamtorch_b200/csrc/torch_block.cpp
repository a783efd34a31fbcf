// PyTorch operators over the layer norm, dropout and GELU entry points of the C ABI, in the `mamtorch_b200` namespace.
//
// The `*_forward` / `*_backward` operators validate, allocate and call the library (CUDA only: a CPU tensor gets the
// dispatcher's NotImplementedError).  The differentiable ones (layer_norm, dropout_add_layer_norm, dropout, gelu) call
// them below an autograd node where a gradient is wanted, and directly where none is: for a few rows the host's time
// is the call's time.  Each differentiates once and in reverse; what would be anything else is refused, never a zero.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <vector>

#include "../../include/mam_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

void check_status(int st, const char* what) {
    if (st == MAM_OK) return;
    TORCH_CHECK(false, what, ": ", mam_status_str(st), st == MAM_ERR_CUDA ? ": " : "",
                st == MAM_ERR_CUDA ? mam_last_cuda_error() : "");
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mut(Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

int dtype_code(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return MAM_F32;
        case at::kHalf: return MAM_F16;
        case at::kBFloat16: return MAM_BF16;
        default: TORCH_CHECK(false, name, " must be float32, float16 or bfloat16, not ", t.scalar_type());
    }
}
void check_like(const Tensor& t, const Tensor& x, const char* name) {
    TORCH_CHECK(t.device() == x.device(), name, " must be on the device of x");
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have the dtype of x");
    TORCH_CHECK(t.sizes() == x.sizes(), name, " must have the shape of x");
}
// weight and bias: one value a column, fp32 or the dtype of x, both of the same; their dtype code
int check_params(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    int code = -1;
    const int own = dtype_code(x, "x");
    for (const Tensor* t : {&weight, &bias}) {
        if (!t->defined()) continue;
        TORCH_CHECK(t->device() == x.device(), "weight and bias must be on the device of x");
        TORCH_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), "weight and bias must have one value per column of x");
        const int c = dtype_code(*t, "weight and bias");
        TORCH_CHECK(c == own || c == MAM_F32, "weight and bias must be float32 or have the dtype of x");
        TORCH_CHECK(code < 0 || code == c, "weight and bias must have the same dtype");
        code = c;
    }
    return code < 0 ? own : code;
}
void check_drop(const Tensor& x, double rate, const OptTensor& seed_at) {
    TORCH_CHECK(rate >= 0.0 && rate < 1.0, "drop_rate must be in [0, 1)");
    if (has(seed_at))
        TORCH_CHECK(seed_at->device() == x.device() && seed_at->scalar_type() == at::kLong && seed_at->numel() == 1,
                    "a drop_seed tensor must hold one int64 on the device of x");
}
const int64_t* seed_ptr(const OptTensor& seed_at) { return has(seed_at) ? seed_at->const_data_ptr<int64_t>() : nullptr; }

// t[..., width] as rows with a uniform distance: in place where its strides are such, else a contiguous copy
Tensor as_rows(const Tensor& t, int64_t& pitch) {
    const int64_t width = t.size(-1);
    pitch = width;
    if (t.is_contiguous()) return t;
    if (t.stride(-1) == 1 || width == 1) {
        int64_t step = -1, expect = -1;   // of the innermost leading dimension that is longer than one; of the next
        bool uniform = true;
        for (int64_t i = t.dim() - 2; i >= 0; --i) {
            if (t.size(i) == 1) continue;
            if (step < 0) step = t.stride(i);
            else if (t.stride(i) != expect) uniform = false;
            expect = t.stride(i) * t.size(i);
        }
        if (uniform && (step < 0 || step >= width)) {
            if (step >= 0) pitch = step;
            return t;
        }
    }
    return t.contiguous();
}

// a contiguous tensor without the dispatcher's detour: for a few rows these calls are a tenth of the operator's time
Tensor fresh(at::IntArrayRef sizes, at::ScalarType t, const Tensor& like) {
    return at::detail::empty_cuda(sizes, t, like.device(), std::nullopt);
}
Tensor fresh(const Tensor& like) { return fresh(like.sizes(), like.scalar_type(), like); }

// ---------------------------------------------------------------- CUDA operators

std::vector<Tensor> layer_norm_forward(const Tensor& x, const OptTensor& residual, const OptTensor& weight,
                                       const OptTensor& bias, double eps, double rate, int64_t seed,
                                       const OptTensor& seed_at, bool want_stats) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int dtype = dtype_code(x, "x");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "x must have a last dimension to normalise");
    TORCH_CHECK(eps >= 0.0, "eps must not be negative");
    const Tensor w = has(weight) ? weight->contiguous() : Tensor(), b = has(bias) ? bias->contiguous() : Tensor();
    const int pdtype = check_params(x, w, b);
    check_drop(x, rate, seed_at);
    if (has(residual)) check_like(*residual, x, "residual");
    else TORCH_CHECK(rate == 0.0, "dropout before the norm needs a residual");
    c10::cuda::CUDAGuard guard(x.device());
    int64_t xp = 0, rp = 0;
    const Tensor xr = as_rows(x, xp), rr = has(residual) ? as_rows(*residual, rp) : Tensor();
    const int64_t width = x.size(-1), rows = x.numel() / width;
    std::vector<Tensor> out;
    out.reserve(3);
    out.push_back(fresh(x));
    if (rr.defined()) out.push_back(fresh(x));
    if (want_stats) out.push_back(fresh({rows, 2}, at::kFloat, x));
    if (rows == 0) return out;
    check_status(mam_layer_norm_fwd(ptr(xr), xp, ptr(rr), rp, ptr(w), ptr(b), pdtype, (float)eps, (float)rate,
                                    (uint64_t)seed, seed_ptr(seed_at), mut(out[0]), rr.defined() ? mut(out[1]) : nullptr,
                                    want_stats ? out.back().mutable_data_ptr<float>() : nullptr, rows, width, dtype,
                                    at::cuda::getCurrentCUDAStream().stream()),
                 "mam_layer_norm_fwd");
    return out;
}

// ds, dx (where something is dropped; else ds is the gradient of x too), dweight, dbias: those that are wanted
std::vector<Tensor> layer_norm_backward(const OptTensor& gy, const OptTensor& gsum, const Tensor& s, const Tensor& stats,
                                        const OptTensor& weight, double rate, int64_t seed, const OptTensor& seed_at,
                                        bool params_f32, bool want_weight, bool want_bias) {
    TORCH_CHECK(s.is_cuda(), "s must be a CUDA tensor");
    const int dtype = dtype_code(s, "s");
    TORCH_CHECK(s.dim() >= 1 && s.size(-1) > 0, "s must have a last dimension to normalise");
    const int64_t width = s.size(-1), rows = s.numel() / width;
    TORCH_CHECK(stats.device() == s.device() && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                    stats.numel() == 2 * rows,
                "stats must be the forward's");
    const Tensor w = has(weight) ? weight->contiguous() : Tensor();
    const int pdtype = w.defined() ? check_params(s, w, Tensor()) : params_f32 ? MAM_F32 : dtype;
    TORCH_CHECK((pdtype == MAM_F32) == (params_f32 || dtype == MAM_F32), "params_f32 and the dtype of weight differ");
    check_drop(s, rate, seed_at);
    if (has(gy)) check_like(*gy, s, "the gradient of y");
    if (has(gsum)) check_like(*gsum, s, "the gradient of the sum");
    c10::cuda::CUDAGuard guard(s.device());
    const Tensor g = has(gy) ? gy->contiguous() : Tensor(), gs = has(gsum) ? gsum->contiguous() : Tensor();
    int64_t sp = 0;
    const Tensor sr = as_rows(s, sp);
    Tensor ds = fresh(s), dx, dw, db;
    if (rate > 0) dx = fresh(s);
    const at::ScalarType kind = pdtype == MAM_F32 ? at::kFloat : s.scalar_type();
    if (want_weight) dw = fresh({width}, kind, s);
    if (want_bias) db = fresh({width}, kind, s);
    if (rows) {
        const size_t bytes = want_weight || want_bias ? mam_layer_norm_bwd_workspace_bytes(rows, width) : 0;
        Tensor ws;
        if (bytes) ws = fresh({(int64_t)bytes}, at::kByte, s);
        check_status(mam_layer_norm_bwd(ptr(g), ptr(gs), ptr(sr), sp, stats.const_data_ptr<float>(), ptr(w), pdtype,
                                        (float)rate, (uint64_t)seed, seed_ptr(seed_at), mut(ds), mut(dx), mut(dw),
                                        mut(db), rows, width, dtype, mut(ws), bytes,
                                        at::cuda::getCurrentCUDAStream().stream()),
                     "mam_layer_norm_bwd");
    }
    std::vector<Tensor> out;
    out.reserve(4);
    for (Tensor* g : {&ds, &dx, &dw, &db})
        if (g->defined()) out.push_back(std::move(*g));
    if (rows == 0)
        for (auto& g : out) g.zero_();
    return out;
}

Tensor dropout_forward(const Tensor& x, const OptTensor& residual, double rate, int64_t seed, const OptTensor& seed_at) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int dtype = dtype_code(x, "x");
    check_drop(x, rate, seed_at);
    if (has(residual)) check_like(*residual, x, "residual");
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor xc = x.contiguous(), rc = has(residual) ? residual->contiguous() : Tensor();
    Tensor y = fresh(x);
    if (y.numel())
        check_status(mam_dropout_add(ptr(xc), ptr(rc), mut(y), y.numel(), dtype, (float)rate, (uint64_t)seed,
                                     seed_ptr(seed_at), at::cuda::getCurrentCUDAStream().stream()),
                     "mam_dropout_add");
    return y;
}

Tensor gelu_forward(const Tensor& x, double rate, int64_t seed, const OptTensor& seed_at) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int dtype = dtype_code(x, "x");
    check_drop(x, rate, seed_at);
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor xc = x.contiguous();
    Tensor y = fresh(x);
    if (y.numel())
        check_status(mam_gelu_fwd(ptr(xc), mut(y), y.numel(), dtype, (float)rate, (uint64_t)seed, seed_ptr(seed_at),
                                  at::cuda::getCurrentCUDAStream().stream()),
                     "mam_gelu_fwd");
    return y;
}

Tensor gelu_backward(const Tensor& gy, const Tensor& x, double rate, int64_t seed, const OptTensor& seed_at) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int dtype = dtype_code(x, "x");
    check_drop(x, rate, seed_at);
    check_like(gy, x, "the gradient of y");
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor gc = gy.contiguous(), xc = x.contiguous();
    Tensor dx = fresh(x);
    if (dx.numel())
        check_status(mam_gelu_bwd(ptr(gc), ptr(xc), mut(dx), dx.numel(), dtype, (float)rate, (uint64_t)seed,
                                  seed_ptr(seed_at), at::cuda::getCurrentCUDAStream().stream()),
                     "mam_gelu_bwd");
    return dx;
}

// ---------------------------------------------------------------- differentiable operators

// The operators above through the dispatcher, so that tracing with fake tensors reaches their shape functions.
// A seed is a number that may be symbolic: a compiled graph takes it as an argument instead of being compiled for each.
template <class A>
using Symbolic = std::conditional_t<std::is_same_v<A, int64_t>, c10::SymInt, A>;
template <class Fn>
struct SymbolicFn;
template <class R, class... A>
struct SymbolicFn<R(A...)> {
    using type = R(Symbolic<A>...);
};
#define MAM_OP(name, fn)                                                                                          \
    static const auto name = c10::Dispatcher::singleton()                                                         \
                                 .findSchemaOrThrow("mamtorch_b200::" #fn, "")                                    \
                                 .typed<SymbolicFn<decltype(fn)>::type>()

template <class... Ts>
bool wants_grad(const Ts&... ts) {
    return at::GradMode::is_enabled() && ((ts.defined() && ts.requires_grad()) || ...);
}
Tensor plain(const OptTensor& t) { return has(t) ? *t : Tensor(); }

// A tangent would be lost below the autograd keys, and torch takes a missing one for zero.
template <class... Ts>
void refuse_tangents(const Ts&... ts) {
    TORCH_CHECK_NOT_IMPLEMENTED(!((ts.defined() && ts._fw_grad(0).defined()) || ...),
                                "mamtorch_b200: layer_norm, dropout and gelu have no forward-mode derivative");
}

// Whether a transform of torch.func is around the call: then every operator goes through the dispatcher, which takes it to
// the transform's levels one by one.
bool transformed() { return c10::impl::tls_is_dispatch_key_included(at::DispatchKey::FuncTorchDynamicLayerFrontMode); }

// The inner operators carry no derivative: where one would be wanted their outputs get a node that says so when it is run.
// A gradient that is differentiated again (create_graph, nested transforms) ends there.
const Tensor& tensor_of(const Tensor& t) { return t; }
Tensor tensor_of(const OptTensor& t) { return plain(t); }
template <class T>
Tensor tensor_of(const T&) { return Tensor(); }
void dead_end(Tensor& t, const std::shared_ptr<torch::autograd::Error>& node) { torch::autograd::set_history(t, node); }
void dead_end(std::vector<Tensor>& ts, const std::shared_ptr<torch::autograd::Error>& node) {
    for (auto& t : ts) dead_end(t, node);
}
template <class Fn, const char* NAME>
struct Inner;
template <class R, class... A, const char* NAME>
struct Inner<R(A...), NAME> {
    static R call(Symbolic<A>... args) {
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(NAME, "").typed<R(Symbolic<A>...)>();
        refuse_tangents(tensor_of(args)...);
        std::shared_ptr<torch::autograd::Error> node;
        if (wants_grad(tensor_of(args)...))
            node.reset(new torch::autograd::Error("mamtorch_b200: layer_norm, dropout and gelu are differentiable once",
                                                  torch::autograd::collect_next_edges(tensor_of(args)...)),
                       torch::autograd::deleteNode);
        R out = [&] {
            at::AutoDispatchBelowADInplaceOrView below;
            return op.call(args...);
        }();
        if (node) dead_end(out, node);
        return out;
    }
};

// The nodes are written out, as torch's own are: the generic C++ Function keeps its arguments in a dictionary by name, which
// took as long as an allocation.
struct BlockNode : torch::autograd::Node {
    double rate = 0;
    c10::SymInt seed = 0;
    SavedVariable seed_at;
    void release_variables() override { seed_at.reset_data(); }
};
template <class N, class... Ts>
std::shared_ptr<N> make_node(double rate, c10::SymInt seed, const OptTensor& seed_at, const Ts&... inputs) {
    std::shared_ptr<N> n(new N(), torch::autograd::deleteNode);
    n->rate = rate;
    n->seed = seed;
    if (has(seed_at)) n->seed_at = SavedVariable(*seed_at, false);
    n->set_next_edges(torch::autograd::collect_next_edges(inputs...));
    return n;
}

struct NormBackward : BlockNode {       // inputs: x, residual, weight, bias
    SavedVariable s, stats, weight;
    bool add = false, f32 = false;
    std::string name() const override { return "MamLayerNormBackward"; }
    void release_variables() override {
        BlockNode::release_variables();
        s.reset_data();
        stats.reset_data();
        weight.reset_data();
    }
    variable_list apply(variable_list&& g) override {
        const Tensor gs = add ? g[1] : Tensor();
        variable_list r(4);
        if (!g[0].defined() && !gs.defined()) return r;
        const auto self = shared_from_this();
        const Tensor w = weight.unpack(), at = seed_at.unpack();
        const bool want_w = task_should_compute_output(2), want_b = task_should_compute_output(3);
        MAM_OP(op, layer_norm_backward);
        auto d = op.call(opt(g[0]), opt(gs), s.unpack(add ? self : nullptr), stats.unpack(), opt(w), rate, seed, opt(at), f32,
                         want_w, want_b);
        size_t next = 1;
        if (task_should_compute_output(1)) r[1] = d[0];
        if (rate > 0) {
            if (task_should_compute_output(0)) r[0] = std::move(d[next]);
            ++next;
        } else if (task_should_compute_output(0)) {
            r[0] = d[0];
        }
        if (want_w) r[2] = std::move(d[next++]);
        if (want_b) r[3] = std::move(d[next]);
        return r;
    }
};

struct DropoutBackward : BlockNode {    // inputs: x, residual
    std::string name() const override { return "MamDropoutBackward"; }
    variable_list apply(variable_list&& g) override {
        variable_list r(2);
        if (!g[0].defined()) return r;
        if (task_should_compute_output(0)) {
            MAM_OP(op, dropout_forward);
            r[0] = rate > 0 ? op.call(g[0], std::nullopt, rate, seed, opt(seed_at.unpack())) : g[0];
        }
        if (task_should_compute_output(1)) r[1] = g[0];
        return r;
    }
};

struct GeluBackward : BlockNode {       // input: x
    SavedVariable x;
    std::string name() const override { return "MamGeluBackward"; }
    void release_variables() override {
        BlockNode::release_variables();
        x.reset_data();
    }
    variable_list apply(variable_list&& g) override {
        variable_list r(1);
        if (!g[0].defined()) return r;
        MAM_OP(op, gelu_backward);
        r[0] = op.call(g[0], x.unpack(), rate, seed, opt(seed_at.unpack()));
        return r;
    }
};

// The differentiable operators.  Without a transform they call the inner operator themselves; with one, their own operator
// below the autograd keys, so that the levels further out differentiate it too.  (The norm's node needs the statistics
// and calls the inner operator: what a level further out would differentiate then is refused there.)
std::vector<Tensor> norm_node(const Tensor& x, const Tensor& res, const Tensor& w, const Tensor& b, double eps, double rate,
                              c10::SymInt seed, const OptTensor& seed_at) {
    MAM_OP(op, layer_norm_forward);
    auto node = make_node<NormBackward>(rate, seed, seed_at, x, res, w, b);
    std::vector<Tensor> out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = op.call(x, opt(res), opt(w), opt(b), eps, rate, seed, seed_at, true);
    }
    node->stats = SavedVariable(out.back(), false);
    out.pop_back();
    node->add = res.defined();
    const Tensor& param = w.defined() ? w : b;
    node->f32 = param.defined() && param.scalar_type() == at::kFloat;
    node->weight = SavedVariable(w, false);
    for (auto& y : out) torch::autograd::set_history(y, node);
    node->s = res.defined() ? SavedVariable(out[1], true) : SavedVariable(x, false);
    return out;
}
std::vector<Tensor> norm_plain(const Tensor& x, const OptTensor& residual, const OptTensor& weight, const OptTensor& bias,
                               double eps, double rate, c10::SymInt seed, const OptTensor& seed_at) {
    MAM_OP(op, layer_norm_forward);
    return op.call(x, residual, weight, bias, eps, rate, seed, seed_at, false);
}
Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    const Tensor w = plain(weight), b = plain(bias);
    refuse_tangents(x, w, b);
    if (wants_grad(x, w, b)) return std::move(norm_node(x, Tensor(), w, b, eps, 0.0, 0, std::nullopt)[0]);
    at::AutoDispatchBelowADInplaceOrView below;
    if (transformed()) {
        MAM_OP(self, layer_norm);
        return self.call(x, weight, bias, eps);
    }
    return std::move(norm_plain(x, std::nullopt, weight, bias, eps, 0.0, 0, std::nullopt)[0]);
}
std::tuple<Tensor, Tensor> dropout_add_layer_norm(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                                  const OptTensor& bias, double eps, double rate, c10::SymInt seed,
                                                  const OptTensor& seed_at) {
    const Tensor w = plain(weight), b = plain(bias);
    refuse_tangents(x, residual, w, b);
    std::vector<Tensor> out;
    if (wants_grad(x, residual, w, b)) {
        out = norm_node(x, residual, w, b, eps, rate, seed, seed_at);
    } else {
        at::AutoDispatchBelowADInplaceOrView below;
        if (transformed()) {
            MAM_OP(self, dropout_add_layer_norm);
            return self.call(x, residual, weight, bias, eps, rate, seed, seed_at);
        }
        out = norm_plain(x, residual, weight, bias, eps, rate, seed, seed_at);
    }
    return {std::move(out[0]), std::move(out[1])};
}
Tensor dropout(const Tensor& x, const OptTensor& residual, double rate, c10::SymInt seed, const OptTensor& seed_at) {
    MAM_OP(op, dropout_forward);
    MAM_OP(self, dropout);
    const Tensor res = plain(residual);
    refuse_tangents(x, res);
    const auto node = wants_grad(x, res) ? make_node<DropoutBackward>(rate, seed, seed_at, x, res) : nullptr;
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = (transformed() ? self : op).call(x, residual, rate, seed, seed_at);
    }
    if (node) torch::autograd::set_history(y, node);
    return y;
}
Tensor gelu(const Tensor& x, double rate, c10::SymInt seed, const OptTensor& seed_at) {
    MAM_OP(op, gelu_forward);
    MAM_OP(self, gelu);
    refuse_tangents(x);
    const auto node = wants_grad(x) ? make_node<GeluBackward>(rate, seed, seed_at, x) : nullptr;
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = (transformed() ? self : op).call(x, rate, seed, seed_at);
    }
    if (node) {
        node->x = SavedVariable(x, false);
        torch::autograd::set_history(y, node);
    }
    return y;
}

// The same operators below the autograd keys.
Tensor layer_norm_below(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    return std::move(norm_plain(x, std::nullopt, weight, bias, eps, 0.0, 0, std::nullopt)[0]);
}
std::tuple<Tensor, Tensor> dropout_add_layer_norm_below(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                                        const OptTensor& bias, double eps, double rate, c10::SymInt seed,
                                                        const OptTensor& seed_at) {
    auto out = norm_plain(x, residual, weight, bias, eps, rate, seed, seed_at);
    return {std::move(out[0]), std::move(out[1])};
}
Tensor dropout_below(const Tensor& x, const OptTensor& residual, double rate, c10::SymInt seed, const OptTensor& seed_at) {
    MAM_OP(op, dropout_forward);
    return op.call(x, residual, rate, seed, seed_at);
}
Tensor gelu_below(const Tensor& x, double rate, c10::SymInt seed, const OptTensor& seed_at) {
    MAM_OP(op, gelu_forward);
    return op.call(x, rate, seed, seed_at);
}

// Eager calls from Python: straight to the functions above, under a transform by way of the dispatcher.
template <class Fn, const char* NAME>
struct Eager;
template <class A>
using Plain = std::conditional_t<std::is_same_v<A, c10::SymInt>, int64_t, A>;
template <class R, class... A, const char* NAME>
struct Eager<R(A...), NAME> {
    template <R (*FN)(A...)>
    static R call(Plain<A>... args) {
        if (!transformed()) return FN(args...);
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(NAME, "").typed<R(A...)>();
        return op.call(args...);
    }
};

constexpr char kNormForward[] = "mamtorch_b200::layer_norm_forward", kNormBackward[] = "mamtorch_b200::layer_norm_backward",
               kDropoutForward[] = "mamtorch_b200::dropout_forward", kGeluForward[] = "mamtorch_b200::gelu_forward",
               kGeluBackward[] = "mamtorch_b200::gelu_backward", kLayerNorm[] = "mamtorch_b200::layer_norm",
               kAddNorm[] = "mamtorch_b200::dropout_add_layer_norm", kDropout[] = "mamtorch_b200::dropout",
               kGelu[] = "mamtorch_b200::gelu";

}  // namespace

TORCH_LIBRARY_FRAGMENT(mamtorch_b200, m) {
    m.def("layer_norm_forward(Tensor x, Tensor? residual, Tensor? weight, Tensor? bias, float eps, float drop_rate, SymInt drop_seed, Tensor? drop_seed_at, bool want_stats) -> Tensor[]");
    m.def("layer_norm_backward(Tensor? gy, Tensor? gsum, Tensor s, Tensor stats, Tensor? weight, float drop_rate, SymInt drop_seed, Tensor? drop_seed_at, bool params_f32, bool want_weight, bool want_bias) -> Tensor[]");
    m.def("dropout_forward(Tensor x, Tensor? residual, float drop_rate, SymInt drop_seed, Tensor? drop_seed_at) -> Tensor");
    m.def("gelu_forward(Tensor x, float drop_rate, SymInt drop_seed, Tensor? drop_seed_at) -> Tensor");
    m.def("gelu_backward(Tensor gy, Tensor x, float drop_rate, SymInt drop_seed, Tensor? drop_seed_at) -> Tensor");
    m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
    m.def("dropout_add_layer_norm(Tensor x, Tensor residual, Tensor? weight, Tensor? bias, float eps, float drop_rate, SymInt drop_seed, Tensor? drop_seed_at) -> (Tensor, Tensor)");
    m.def("dropout(Tensor x, Tensor? residual, float drop_rate, SymInt drop_seed, Tensor? drop_seed_at) -> Tensor");
    m.def("gelu(Tensor x, float drop_rate, SymInt drop_seed, Tensor? drop_seed_at) -> Tensor");
}
TORCH_LIBRARY_IMPL(mamtorch_b200, CUDA, m) {
    m.impl("layer_norm_forward", &layer_norm_forward);
    m.impl("layer_norm_backward", &layer_norm_backward);
    m.impl("dropout_forward", &dropout_forward);
    m.impl("gelu_forward", &gelu_forward);
    m.impl("gelu_backward", &gelu_backward);
}

TORCH_LIBRARY_IMPL(mamtorch_b200, Autograd, m) {
    m.impl("layer_norm_forward", &Inner<decltype(layer_norm_forward), kNormForward>::call);
    m.impl("layer_norm_backward", &Inner<decltype(layer_norm_backward), kNormBackward>::call);
    m.impl("dropout_forward", &Inner<decltype(dropout_forward), kDropoutForward>::call);
    m.impl("gelu_forward", &Inner<decltype(gelu_forward), kGeluForward>::call);
    m.impl("gelu_backward", &Inner<decltype(gelu_backward), kGeluBackward>::call);
    m.impl("layer_norm", &layer_norm);
    m.impl("dropout_add_layer_norm", &dropout_add_layer_norm);
    m.impl("dropout", &dropout);
    m.impl("gelu", &gelu);
}
TORCH_LIBRARY_IMPL(mamtorch_b200, CompositeExplicitAutograd, m) {
    m.impl("layer_norm", &layer_norm_below);
    m.impl("dropout_add_layer_norm", &dropout_add_layer_norm_below);
    m.impl("dropout", &dropout_below);
    m.impl("gelu", &gelu_below);
}

// The differentiable operators as plain functions of the module mamtorch_b200._C, for eager calls: the way through
// torch.ops (a schema's arguments, boxed) takes a microsecond of the seven that a small call lasts.
PYBIND11_MODULE(_C, m) {
    const pybind11::call_guard<pybind11::gil_scoped_release> free;
    m.def("layer_norm", &Eager<decltype(layer_norm), kLayerNorm>::call<&layer_norm>, free);
    m.def("dropout_add_layer_norm", &Eager<decltype(dropout_add_layer_norm), kAddNorm>::call<&dropout_add_layer_norm>, free);
    m.def("dropout", &Eager<decltype(dropout), kDropout>::call<&dropout>, free);
    m.def("gelu", &Eager<decltype(gelu), kGelu>::call<&gelu>, free);
}
