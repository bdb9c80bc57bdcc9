// The head operators on torch tensors: argument checks, outputs and workspaces from torch's allocator, and the autograd
// functions. Every computation is a call into librocal_b200 through the addresses that bind() gets, so that one
// binding serves whichever build of the library the process has loaded. In C++ because a step of a small head is
// shorter than the interpreter's work on its arguments, and because the backward pass then runs on autograd's threads
// without the interpreter.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <array>
#include <cstring>
#include <functional>
#include <optional>
#include <stdexcept>
#include <string>
#include <unordered_set>
#include <vector>

#include "rb200_kernels.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

// ---- the library ------------------------------------------------------------------------------------------
struct Api {
    decltype(&rb200k_linear_workspace_bytes) linear_bytes;
    decltype(&rb200k_linear) linear;
    decltype(&rb200k_linear_probe) linear_probe;
    decltype(&rb200k_linear_backward_workspace_bytes) linear_backward_bytes;
    decltype(&rb200k_linear_backward) linear_backward;
    decltype(&rb200k_linear_ce_workspace_bytes) ce_bytes;
    decltype(&rb200k_linear_ce) ce;
    decltype(&rb200k_linear_ce_backward_workspace_bytes) ce_backward_bytes;
    decltype(&rb200k_linear_ce_backward) ce_backward;
    decltype(&rb200k_grad_clip_workspace_bytes) clip_bytes;
    decltype(&rb200k_grad_clip) clip;
    decltype(&rb200k_last_error) last_error;
} api;

// A library call that failed; Python sees it as rocal_b200.Rb200Error.
struct LibraryError : std::runtime_error {
    using std::runtime_error::runtime_error;
};
PyObject* library_error = nullptr;

void bind(const std::vector<uintptr_t>& a, py::object error) {
    TORCH_CHECK(a.size() * sizeof(uintptr_t) == sizeof(Api), "the binding and the library do not go together");
    memcpy(&api, a.data(), sizeof(Api));
    library_error = error.release().ptr();
}

void check(int rc, const char* what) {
    if (rc) throw LibraryError(c10::str(what, " failed (", rc, "): ", api.last_error()));
}

// ---- arguments ----------------------------------------------------------------------------------------------
int head_dtype(const Tensor& x) {
    TORCH_CHECK_VALUE(x.is_cuda(), "x is on ", x.device(), ": the head operators run on a GPU");
    TORCH_CHECK_VALUE(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, "x is ", x.scalar_type(),
                      ": the head operators take float16 and bfloat16");
    return x.scalar_type() == at::kHalf ? RB200_FP16 : RB200_BF16;
}

void same_kind(const Tensor& t, const char* name, const Tensor& like) {
    TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type() && t.device() == like.device(), name, " is ", t.scalar_type(), " on ", t.device(),
                      ", the input is ", like.scalar_type(), " on ", like.device());
}

// Rows contiguous and not overlapping.
bool has_rows(const Tensor& t) {
    return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}
int64_t pitch(const Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// What the kernels read are the bytes: a view whose negation is still to come (the imaginary part of a conjugate) is made first.
Tensor settled(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// A matrix of the input's type and device, its rows contiguous (copied if need be).
Tensor matrix(const Tensor& t, const char* name, const Tensor& like, int64_t rows, int64_t cols) {
    TORCH_CHECK_VALUE(t.dim() == 2, name, " has ", t.dim(), " dimensions, a matrix is needed");
    same_kind(t, name, like);
    TORCH_CHECK_VALUE(cols < 0 || t.size(1) == cols, name, " has ", t.size(1), " columns, ", cols, " are needed");
    TORCH_CHECK_VALUE(rows < 0 || t.size(0) == rows, name, " has ", t.size(0), " rows, ", rows, " are needed");
    const Tensor s = settled(t);
    return has_rows(s) ? s : s.contiguous();
}
Tensor vector(const Tensor& t, const char* name, const Tensor& like, int64_t n) {
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, name, " has shape ", t.sizes(), ", (", n, ",) is needed");
    same_kind(t, name, like);
    return settled(t).contiguous();
}
bool given(const MaybeTensor& t) { return t.has_value() && t->defined(); }
Tensor or_undefined(const MaybeTensor& t) { return given(t) ? *t : Tensor(); }
MaybeTensor or_absent(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

Tensor workspace(uint64_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int32_t* status_word(const MaybeTensor& status, const Tensor& like) {
    if (!given(status)) return nullptr;
    TORCH_CHECK_VALUE(status->scalar_type() == at::kInt && status->device() == like.device() && status->numel() >= 1, "status has to be an int32 tensor on ",
                      like.device());
    return status->data_ptr<int32_t>();
}
// Waits inside the products are bounded: one that gives up leaves its results unfinished and raises a status word. Calls for which
// the caller gives no word of their own through the kernel layer (single launches: the library-wide word) raise this one, which lies
// in pinned host memory: the host reads it without waiting, and the next call says what has happened. Kept for the whole process; captured
// graphs hold its address.
int32_t* unfinished_word() {
    static int32_t* const word = [] {
        c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
        const auto* kept = new Tensor(at::empty({1}, at::TensorOptions().dtype(at::kInt).pinned_memory(true)));
        int32_t* w = kept->data_ptr<int32_t>();
        __atomic_store_n(w, 0, __ATOMIC_RELAXED);
        return w;
    }();
    return word;
}
void check_unfinished() {
    if (__atomic_load_n(unfinished_word(), __ATOMIC_RELAXED) && __atomic_exchange_n(unfinished_word(), 0, __ATOMIC_RELAXED))
        throw LibraryError("a bounded wait of an earlier head operator ran out: its results, and what was made from them, are unfinished");
}
struct Status {
    MaybeTensor given;      // the caller's word, or none: the library-wide one
    bool watched = false;   // unfinished_word()
};
constexpr bool kWatched = true;
int32_t* status_word(const Status& s, const Tensor& like) { return s.watched ? unfinished_word() : status_word(s.given, like); }

// The library has written to a tensor of the caller's: autograd's version check has to know.
void written(const Tensor& t) {
    if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}
void* stream_of(const Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.device().index()).stream(); }

int activation(const std::string& name) {
    if (name == "none") return RB200_ACT_NONE;
    if (name == "relu") return RB200_ACT_RELU;
    if (name == "gelu") return RB200_ACT_GELU;
    if (name == "silu") return RB200_ACT_SILU;
    TORCH_CHECK_VALUE(false, "activation '", name, "': one of none, relu, gelu, silu is needed");
}
int reduction(const std::string& name) {
    if (name == "none") return RB200_REDUCE_NONE;
    if (name == "mean") return RB200_REDUCE_MEAN;
    if (name == "sum") return RB200_REDUCE_SUM;
    TORCH_CHECK_VALUE(false, "reduction '", name, "': one of none, mean, sum is needed");
}

// ---- linear -----------------------------------------------------------------------------------------------
// x, weight and residual are matrices, bias a vector.
Tensor linear_run(const Tensor& x_, const Tensor& weight_, const Tensor& bias_, const Tensor& residual_, int act, Tensor out, Tensor* preact,
                  const Status& status, std::optional<std::pair<uint64_t, int>> probe) {
    rb200_linear_params p = {};
    p.dtype = head_dtype(x_);
    c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = matrix(x_, "x", x_, -1, -1), weight = matrix(weight_, "weight", x, -1, x.size(1));
    const int64_t n = x.size(0), m = weight.size(0);
    p.activation = act;
    p.rows = n;
    p.in_features = x.size(1);
    p.out_features = m;
    p.x = x.data_ptr();
    p.ldx = pitch(x);
    p.weight = weight.data_ptr();
    p.ldw = pitch(weight);
    Tensor bias, residual;
    if (bias_.defined()) {
        bias = vector(bias_, "bias", x, m);
        p.bias = bias.data_ptr();
    }
    if (residual_.defined()) {
        residual = matrix(residual_, "residual", x, -1, m);
        const int64_t r = residual.size(0);
        TORCH_CHECK_VALUE(r > 0 ? n % r == 0 : n == 0, "residual has ", r, " rows, which do not divide the ", n, " rows of x");
        p.residual = residual.data_ptr();
        p.ldr = pitch(residual);
        p.residual_rows = r;
    }
    if (out.defined()) {
        TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == n && out.size(1) == m && has_rows(out) && !out.is_neg(), "out has shape ", out.sizes(), ", strides ",
                          out.strides(), "; (", n, ", ", m, ") with contiguous rows is needed");
        same_kind(out, "out", x);
        written(out);
    } else {
        out = at::empty({n, m}, x.options());
    }
    p.out = out.data_ptr();
    p.ldo = pitch(out);
    if (preact) {
        *preact = at::empty({n, m}, x.options());
        p.preact = preact->data_ptr();
        p.ldp = m;
    }
    if (n == 0) return out;
    p.status = status_word(status, x);
    const uint64_t need = api.linear_bytes(&p);
    const Tensor ws = workspace(need, x);
    p.workspace = data(ws);
    p.workspace_bytes = need;
    if (probe)
        check(api.linear_probe(&p, stream_of(x), probe->first, probe->second), "rb200k_linear_probe");
    else
        check(api.linear(&p, stream_of(x)), "rb200k_linear");
    return out;
}

std::vector<Tensor> linear_backward_run(const Tensor& dout_, const Tensor& x_, const Tensor& weight_, const Tensor& preact_, int act,
                                        int64_t residual_rows, std::array<bool, 4> need, const Status& status) {
    rb200_linear_backward_params p = {};
    p.dtype = head_dtype(x_);
    c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = matrix(x_, "x", x_, -1, -1), weight = matrix(weight_, "weight", x, -1, x.size(1));
    const int64_t n = x.size(0), k = x.size(1), m = weight.size(0);
    const Tensor dout = matrix(dout_, "dout", x, n, m);
    p.activation = act;
    p.rows = n;
    p.in_features = k;
    p.out_features = m;
    p.dout = dout.data_ptr();
    p.lddo = pitch(dout);
    p.x = x.data_ptr();
    p.ldx = pitch(x);
    p.weight = weight.data_ptr();
    p.ldw = pitch(weight);
    Tensor preact;
    if (act != RB200_ACT_NONE && (need[0] || need[1] || need[2])) {
        TORCH_CHECK_VALUE(preact_.defined(), "the backward pass of an activation needs preact");
        preact = matrix(preact_, "preact", x, n, m);
        p.preact = preact.data_ptr();
        p.ldp = pitch(preact);
    }
    std::vector<Tensor> g(4);
    if (need[0]) p.dx = (g[0] = at::empty({n, k}, x.options())).data_ptr();
    if (need[1]) p.dweight = (g[1] = at::empty({m, k}, x.options())).data_ptr();
    if (need[2]) p.dbias = (g[2] = at::empty({m}, x.options())).data_ptr();
    if (need[3]) {
        TORCH_CHECK_VALUE(residual_rows > 0 && n % residual_rows == 0, "residual_rows ", residual_rows, " does not divide the ", n, " rows");
        p.residual_rows = residual_rows;
        p.dresidual = (g[3] = at::empty({residual_rows, m}, x.options())).data_ptr();
    }
    p.lddx = p.lddw = k;
    p.lddr = m;
    p.status = status_word(status, x);
    const uint64_t bytes = api.linear_backward_bytes(&p);
    const Tensor ws = workspace(bytes, x);
    p.workspace = data(ws);
    p.workspace_bytes = bytes;
    check(api.linear_backward(&p, stream_of(x)), "rb200k_linear_backward");
    return g;
}

// The kernels see values only: a dual tensor's tangent (forward-mode differentiation) would be lost, and count as zero.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative: an input carries a tangent");
}

constexpr const char* kOnce = " is differentiable once: create_graph is not supported";

struct Linear : torch::autograd::Function<Linear> {
    // Absent tensors are empty optionals here: autograd numbers the inputs that are there.
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight, const MaybeTensor& bias_,
                          const MaybeTensor& residual_, int64_t act) {
        Tensor preact, bias = or_undefined(bias_), residual = or_undefined(residual_);
        const Tensor y = linear_run(x, weight, bias, residual, (int)act, Tensor(), act != RB200_ACT_NONE ? &preact : nullptr, {{}, kWatched}, {});
        ctx->save_for_backward({x, weight, preact});
        ctx->saved_data["act"] = act;
        ctx->saved_data["rows"] = residual.defined() ? residual.size(0) : (int64_t)0;
        ctx->saved_data["bias"] = bias.defined();
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear", kOnce);
        const auto saved = ctx->get_saved_variables();
        const Tensor& dout = grads[0];
        const int64_t rows = ctx->saved_data["rows"].toInt();
        if (!dout.defined()) return torch::autograd::variable_list(5);
        refuse_tangents("linear's backward pass", {&dout});
        const bool has_bias = ctx->saved_data["bias"].toBool();
        std::array<bool, 4> need = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), has_bias && ctx->needs_input_grad(2),
                                    rows > 0 && ctx->needs_input_grad(has_bias ? 3 : 2)};
        const bool whole = need[3] && rows == saved[0].size(0);   // nothing is summed: the gradient goes through as it is
        if (whole) need[3] = false;
        std::vector<Tensor> g(4);
        if (need[0] || need[1] || need[2] || need[3])
            g = linear_backward_run(dout, saved[0], saved[1], saved[2], (int)ctx->saved_data["act"].toInt(), rows, need, {{}, kWatched});
        return {g[0], g[1], g[2], whole ? dout : g[3], Tensor()};
    }
};

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A leaf's gradient node lives as long as any graph that holds it, and belongs to the stream that was current when it was
// made. In a capture, autograd would make the legacy default stream wait for the capturing one if an eager graph of
// the same leaf were still alive there: CUDA does not allow that, and the error ends the process. Refused here, before anything is
// captured. A leaf may also lie behind operations of the capture itself (a cast, a view): the graph is followed through nodes of other
// streams than the default one.
void refuse_stale_leaves(std::initializer_list<const Tensor*> tensors) {
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    using torch::autograd::Node;
    std::vector<std::shared_ptr<Node>> todo;
    std::unordered_set<const Node*> seen;
    auto take = [&](std::shared_ptr<Node> node) {
        if (node && seen.insert(node.get()).second) todo.push_back(std::move(node));
    };
    for (const Tensor* t : tensors)
        if (wants_grad(*t)) take(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    while (!todo.empty()) {
        const std::shared_ptr<Node> node = std::move(todo.back());
        todo.pop_back();
        const auto stream = node->stream();
        const bool eager = stream && *stream == c10::cuda::getDefaultCUDAStream(stream->device_index()).unwrap();
        TORCH_CHECK(!eager || !dynamic_cast<torch::autograd::AccumulateGrad*>(node.get()),
                    "capture with gradients: a graph of the same leaf, made on the default stream, is still alive; drop it "
                    "(its outputs and losses) before the capture, or make it on another stream");
        if (!eager)
            for (const auto& edge : node->next_edges()) take(edge.function);
    }
}

Tensor linear(const Tensor& x, const Tensor& weight, const MaybeTensor& bias_, const MaybeTensor& residual_, const std::string& act_name) {
    const int act = activation(act_name);
    TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1), "x ", x.sizes(), " does not go with weight ", weight.sizes());
    const Tensor bias = or_undefined(bias_);
    Tensor residual = or_undefined(residual_);
    refuse_tangents("linear", {&x, &weight, &bias, &residual});
    const int64_t m = weight.size(0);
    if (x.is_cuda()) check_unfinished();
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = m;
    if (residual.defined()) {
        const int64_t d = residual.dim();
        const bool tail = d >= 1 && d <= (int64_t)shape.size() && std::equal(residual.sizes().begin(), residual.sizes().end(), shape.end() - d);
        TORCH_CHECK_VALUE(tail || (d == 2 && x.dim() == 2 && residual.size(1) == m), "residual ", residual.sizes(),
                          " is not a tail of the result's shape ", at::IntArrayRef(shape));
        if (d != 2) residual = residual.reshape({-1, m});
    }
    const bool flat = x.dim() == 2;
    const Tensor x2 = flat ? x : x.reshape({-1, x.size(-1)});
    Tensor y;
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual))) {
        refuse_stale_leaves({&x, &weight, &bias, &residual});
        y = Linear::apply(x2, weight, or_absent(bias), or_absent(residual), (int64_t)act);
    } else {
        y = linear_run(x2, weight, bias, residual, act, Tensor(), nullptr, {{}, kWatched}, {});
    }
    return flat ? y : y.reshape(shape);
}

// ---- linear cross entropy -----------------------------------------------------------------------------------
struct CeArgs {
    rb200_linear_ce_params p = {};
    Tensor x, weight, labels, bias;   // what the parameters point into
};
CeArgs ce_args(const Tensor& x, const Tensor& weight, const Tensor& labels, const Tensor& bias, int64_t ignore_index, double smoothing, int reduce) {
    CeArgs a;
    a.p.dtype = head_dtype(x);
    a.x = matrix(x, "x", x, -1, -1);
    a.weight = matrix(weight, "weight", x, -1, a.x.size(1));
    a.p.reduction = reduce;
    a.p.rows = a.x.size(0);
    a.p.features = a.x.size(1);
    a.p.classes = a.weight.size(0);
    TORCH_CHECK_VALUE(labels.dim() == 1 && labels.size(0) == a.p.rows && labels.device() == x.device() &&
                          (labels.scalar_type() == at::kInt || labels.scalar_type() == at::kLong),
                      "labels are ", labels.scalar_type(), " ", labels.sizes(), " on ", labels.device(), ", needed: int32 or int64 of shape (",
                      a.p.rows, ",) on ", x.device());
    TORCH_CHECK_VALUE(smoothing >= 0.0 && smoothing <= 1.0, "label_smoothing ", smoothing, " outside [0, 1]");
    a.labels = labels.contiguous();
    a.p.x = a.x.data_ptr();
    a.p.ldx = pitch(a.x);
    a.p.weight = a.weight.data_ptr();
    a.p.ldw = pitch(a.weight);
    if (bias.defined()) {
        a.bias = vector(bias, "bias", x, a.p.classes);
        a.p.bias = a.bias.data_ptr();
    }
    a.p.labels = a.labels.data_ptr();
    a.p.label_bytes = labels.scalar_type() == at::kInt ? 4 : 8;
    a.p.label_smoothing = (float)smoothing;
    a.p.ignore_index = ignore_index;
    return a;
}

// (loss, stats, info)
std::array<Tensor, 3> ce_run(const Tensor& x, const Tensor& weight, const Tensor& labels, const Tensor& bias, int64_t ignore_index, double smoothing,
                             int reduce, const Status& status) {
    head_dtype(x);
    c10::cuda::CUDAGuard guard(x.device());
    CeArgs a = ce_args(x, weight, labels, bias, ignore_index, smoothing, reduce);
    const auto fp32 = x.options().dtype(at::kFloat);
    const Tensor loss = reduce == RB200_REDUCE_NONE ? at::empty({a.p.rows}, fp32) : at::empty({}, fp32);
    const Tensor stats = at::empty({3, a.p.rows}, fp32), info = at::empty({4}, x.options().dtype(at::kInt));
    a.p.loss = loss.data_ptr<float>();
    a.p.stats = stats.data_ptr<float>();
    a.p.info = info.data_ptr<int32_t>();
    a.p.status = status_word(status, x);
    const uint64_t bytes = api.ce_bytes(&a.p);
    const Tensor ws = workspace(bytes, x);
    a.p.workspace = data(ws);
    a.p.workspace_bytes = bytes;
    check(api.ce(&a.p, stream_of(x)), "rb200k_linear_ce");
    return {loss, stats, info};
}

std::vector<Tensor> ce_backward_run(const Tensor& dloss_, const Tensor& x, const Tensor& weight, const Tensor& labels, const Tensor& stats,
                                    const Tensor& info, const Tensor& bias, int64_t ignore_index, double smoothing, int reduce,
                                    std::array<bool, 3> need, const Status& status) {
    head_dtype(x);
    c10::cuda::CUDAGuard guard(x.device());
    CeArgs a = ce_args(x, weight, labels, bias, ignore_index, smoothing, reduce);
    const int64_t n = a.p.rows, k = a.p.features, v = a.p.classes;
    TORCH_CHECK_VALUE(dloss_.scalar_type() == at::kFloat && dloss_.device() == x.device() &&
                          (reduce == RB200_REDUCE_NONE ? dloss_.dim() == 1 && dloss_.size(0) == n : dloss_.dim() == 0),
                      "dloss is ", dloss_.scalar_type(), " ", dloss_.sizes(), " on ", dloss_.device(), ", it has to be like the loss");
    TORCH_CHECK_VALUE(stats.dim() == 2 && stats.size(0) == 3 && stats.size(1) == n && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                          stats.device() == x.device() && info.dim() == 1 && info.size(0) == 4 && info.scalar_type() == at::kInt &&
                          info.is_contiguous() && info.device() == x.device(),
                      "stats and info are not those of this forward pass");
    const Tensor dloss = settled(dloss_).contiguous();
    std::vector<Tensor> g(3);
    if (need[0]) a.p.dx = (g[0] = at::empty({n, k}, x.options())).data_ptr();
    if (need[1]) a.p.dweight = (g[1] = at::empty({v, k}, x.options())).data_ptr();
    if (need[2]) a.p.dbias = (g[2] = at::empty({v}, x.options())).data_ptr();
    a.p.lddx = a.p.lddw = k;
    a.p.dloss = dloss.data_ptr<float>();
    a.p.stats = stats.data_ptr<float>();
    a.p.info = info.data_ptr<int32_t>();
    a.p.status = status_word(status, x);
    const uint64_t bytes = api.ce_backward_bytes(&a.p);
    const Tensor ws = workspace(bytes, x);
    a.p.workspace = data(ws);
    a.p.workspace_bytes = bytes;
    check(api.ce_backward(&a.p, stream_of(x)), "rb200k_linear_ce_backward");
    return g;
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& labels,
                          const MaybeTensor& bias_, int64_t ignore_index, double smoothing, int64_t reduce) {
        const Tensor bias = or_undefined(bias_);
        const auto r = ce_run(x, weight, labels, bias, ignore_index, smoothing, (int)reduce, {{}, kWatched});
        ctx->save_for_backward({x, weight, labels, bias, r[1], r[2]});
        ctx->saved_data["ignore"] = ignore_index;
        ctx->saved_data["smoothing"] = smoothing;
        ctx->saved_data["reduce"] = reduce;
        return r[0];
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_cross_entropy", kOnce);
        if (!grads[0].defined()) return torch::autograd::variable_list(7);
        refuse_tangents("linear_cross_entropy's backward pass", {&grads[0]});
        const auto s = ctx->get_saved_variables();
        const auto g = ce_backward_run(grads[0], s[0], s[1], s[2], s[4], s[5], s[3], ctx->saved_data["ignore"].toInt(),
                                       ctx->saved_data["smoothing"].toDouble(), (int)ctx->saved_data["reduce"].toInt(),
                                       {ctx->needs_input_grad(0), ctx->needs_input_grad(1), s[3].defined() && ctx->needs_input_grad(3)}, {{}, kWatched});
        return {g[0], g[1], Tensor(), g[2], Tensor(), Tensor(), Tensor()};
    }
};

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& labels, const MaybeTensor& bias_, int64_t ignore_index,
                            double smoothing, const std::string& reduce_name) {
    const int reduce = reduction(reduce_name);
    TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1) && labels.dim() == x.dim() - 1 &&
                          std::equal(labels.sizes().begin(), labels.sizes().end(), x.sizes().begin()),
                      "x ", x.sizes(), ", weight ", weight.sizes(), " and labels ", labels.sizes(), " do not go together");
    const Tensor bias = or_undefined(bias_);
    refuse_tangents("linear_cross_entropy", {&x, &weight, &bias});
    if (x.is_cuda()) check_unfinished();
    const bool flat = x.dim() == 2;
    const Tensor x2 = flat ? x : x.reshape({-1, x.size(-1)}), l1 = flat ? labels : labels.reshape({-1});
    Tensor loss;
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias))) {
        refuse_stale_leaves({&x, &weight, &bias});
        loss = LinearCrossEntropy::apply(x2, weight, l1, or_absent(bias), ignore_index, smoothing, (int64_t)reduce);
    } else {
        loss = ce_run(x2, weight, l1, bias, ignore_index, smoothing, reduce, {{}, kWatched})[0];
    }
    return flat || reduce != RB200_REDUCE_NONE ? loss : loss.reshape(labels.sizes());
}

// ---- gradient norm and clipping -------------------------------------------------------------------------------
int grad_dtype(const Tensor& t, const Tensor& first) {
    TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.device() == first.device(), "a gradient is ", t.layout(), " on ", t.device(),
                      "; strided tensors on ", first.device(), " are needed");
    switch (t.scalar_type()) {
        case at::kFloat: return RB200_FP32;
        case at::kHalf: return RB200_FP16;
        case at::kBFloat16: return RB200_BF16;
        default: TORCH_CHECK_VALUE(false, "a gradient is ", t.scalar_type(), "; float32, float16 or bfloat16 is needed");
    }
}

// The tensors of a list as they lie in their Python objects, which `items` keeps alive. Copying them into a vector as the
// binding does it by itself took 58 of the 79 us of host time that a call of 334 gradients and outputs had.
struct TensorList {
    py::object items;
    TensorList(const py::object& list, const char* name) : items(py::reinterpret_steal<py::object>(PySequence_Tuple(list.ptr()))) {
        if (!items) throw py::error_already_set();
        for (size_t i = 0; i < size(); i++)
            if (!THPVariable_Check(PyTuple_GET_ITEM(items.ptr(), i)))
                throw py::type_error(std::string(name) + " has to be tensors, one of them is " + Py_TYPE(PyTuple_GET_ITEM(items.ptr(), i))->tp_name);
    }
    size_t size() const { return (size_t)PyTuple_GET_SIZE(items.ptr()); }
    const Tensor& operator[](size_t i) const { return THPVariable_Unpack(PyTuple_GET_ITEM(items.ptr(), i)); }
};

// The memory of tensors that the library sees a dense copy of: it compares ranges of addresses, and theirs are the copies'. Whether such
// a tensor meets another one is decided here, by the elements themselves.
struct Extent {
    const Tensor* t;
    uintptr_t begin, end;   // first byte, and the one behind the last element
    explicit Extent(const Tensor& tensor) : t(&tensor), begin((uintptr_t)tensor.data_ptr()), end(begin) {
        if (!tensor.numel()) return;
        int64_t reach = 1;
        for (int64_t d = 0; d < tensor.dim(); d++) reach += (tensor.size(d) - 1) * tensor.stride(d);
        end += (uintptr_t)reach * tensor.element_size();
    }
};
// Whether sum c_k v_k = rest has a solution with 0 <= v_k <= most_k; the c_k fall, reach[k] = sum of c_j most_j from k on. Strides of
// slices of one array leave one or two candidates a step. Gives up, and says yes, when `steps` are spent.
bool reaches(const std::vector<std::pair<int64_t, int64_t>>& terms, const std::vector<int64_t>& reach, size_t k, int64_t rest, int64_t& steps) {
    if (rest < 0 || rest > reach[k]) return false;
    if (k == terms.size() || --steps <= 0) return true;   // k == size: reach is 0, and so is the rest
    const auto [c, most] = terms[k];
    const int64_t low = rest > reach[k + 1] ? (rest - reach[k + 1] + c - 1) / c : 0, high = std::min(most, rest / c);
    for (int64_t v = low; v <= high; v++)
        if (reaches(terms, reach, k + 1, rest - v * c, steps)) return true;
    return false;
}
// Whether an element of `a` and one of `b` share a byte: begin_a + sum x_i s_i + i = begin_b + sum y_j t_j + j, bytes of elements included; y
// is counted from its end, so that every coefficient is positive.
bool share_memory(const Extent& a, const Extent& b) {
    if (a.begin >= b.end || b.begin >= a.end || a.begin == a.end || b.begin == b.end) return false;
    std::vector<std::pair<int64_t, int64_t>> terms;
    for (const Extent* e : {&a, &b}) {
        const int64_t size = (int64_t)e->t->element_size();
        terms.emplace_back(1, size - 1);
        for (int64_t d = 0; d < e->t->dim(); d++)
            if (e->t->size(d) > 1 && e->t->stride(d)) terms.emplace_back(e->t->stride(d) * size, e->t->size(d) - 1);
    }
    std::sort(terms.begin(), terms.end(), std::greater<>());
    size_t n = 0;
    for (size_t i = 1; i < terms.size(); i++)   // equal strides are one term
        if (terms[i].first == terms[n].first)
            terms[n].second += terms[i].second;
        else
            terms[++n] = terms[i];
    terms.resize(n + 1);
    std::vector<int64_t> reach(terms.size() + 1, 0);
    for (size_t k = terms.size(); k-- > 0;) reach[k] = reach[k + 1] + terms[k].first * terms[k].second;
    int64_t steps = 100000;
    return reaches(terms, reach, 0, (int64_t)(b.end - 1) - (int64_t)a.begin, steps);
}
// Every stride steps over all that the smaller ones reach.
bool overlaps_itself(const Tensor& t) {
    if (!t.numel()) return false;
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t d = 0; d < t.dim(); d++)
        if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
    std::sort(dims.begin(), dims.end());
    int64_t reach = 0;
    for (const auto& [stride, size] : dims) {
        if (stride <= reach) return true;
        reach += stride * (size - 1);
    }
    return false;
}
// No output meets itself, another output or another tensor's gradients. copied[i]: the library sees a copy of tensor i; those that
// it sees as they are it compares by itself.
void refuse_overlaps(const TensorList& grads, const TensorList& out, bool apart, const std::vector<bool>& copied) {
    std::vector<Extent> outs, ins;
    for (size_t i = 0; i < out.size(); i++) {
        outs.emplace_back(out[i]);
        if (apart) ins.emplace_back(grads[i]);
    }
    for (size_t i = 0; i < outs.size(); i++) {
        if (!copied[i]) continue;
        bool meets = overlaps_itself(out[i]);
        for (size_t j = 0; j < outs.size() && !meets; j++) {
            if (j == i || (copied[j] && j < i)) continue;   // that pair has been looked at
            meets = share_memory(outs[i], outs[j]) || (apart && (share_memory(outs[i], ins[j]) || share_memory(outs[j], ins[i])));
        }
        if (meets) throw LibraryError("grad_clip: an output overlaps itself, another output or another tensor's gradients");
    }
}

Tensor grad_clip(const py::object& grads_, double max_norm, const py::object& out_, double inv_scale) {
    const bool apart = !out_.is_none();
    const TensorList grads(grads_, "grads"), out = apart ? TensorList(out_, "out") : grads;
    TORCH_CHECK_VALUE(grads.size() > 0, "no gradients");
    TORCH_CHECK_VALUE(out.size() == grads.size(), out.size(), " outputs for ", grads.size(), " gradients");
    for (size_t i = 0; i < grads.size(); i++) refuse_tangents("grad_clip", {&grads[i], &out[i]});
    TORCH_CHECK_VALUE(grads[0].is_cuda(), "the gradients are on ", grads[0].device(), ": the head operators run on a GPU");
    check_unfinished();
    TORCH_CHECK_VALUE(max_norm >= 0 && inv_scale > 0, "max_norm ", max_norm, ", inv_scale ", inv_scale);
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(grads[0].device());
    const size_t n = grads.size();
    std::vector<rb200_grad_tensor> table(n);
    std::vector<Tensor> held;                              // dense copies of tensors with gaps
    std::vector<bool> copied(n);
    std::vector<std::pair<Tensor, Tensor>> back;           // (the tensor with gaps, its dense result)
    for (size_t i = 0; i < n; i++) {
        const Tensor& g = grads[i];
        const Tensor& o = out[i];
        rb200_grad_tensor& t = table[i];
        t.grad_dtype = grad_dtype(g, grads[0]);
        t.out_dtype = apart ? grad_dtype(o, grads[0]) : t.grad_dtype;
        t.count = g.numel();
        TORCH_CHECK_VALUE(o.numel() == t.count, "an output has ", o.numel(), " elements for a gradient of ", t.count);
        TORCH_CHECK_VALUE(t.out_dtype == t.grad_dtype || t.out_dtype == RB200_FP32, "an output is ", o.scalar_type(), " for a gradient ", g.scalar_type());
        const bool settled_both = !g.is_neg() && !o.is_neg(), plain = g.is_contiguous() && (!apart || o.is_contiguous());
        if (settled_both && (plain || (g.is_non_overlapping_and_dense() && (!apart || (o.sizes() == g.sizes() && o.strides() == g.strides()))))) {
            t.grad = g.data_ptr();
            t.out = o.data_ptr();
            continue;
        }
        TORCH_CHECK_VALUE(o.sizes() == g.sizes(), "an output has shape ", o.sizes(), " for a gradient ", g.sizes());
        copied[i] = true;
        Tensor dense = settled(g).contiguous(), result = !apart ? dense : o.is_contiguous() && !o.is_neg() ? o : at::empty(o.sizes(), o.options());
        if (!result.is_same(o)) back.emplace_back(o, result);
        t.grad = dense.data_ptr();
        t.out = result.data_ptr();
        held.push_back(std::move(dense));
    }
    if (!held.empty()) refuse_overlaps(grads, out, apart, copied);
    const Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
    const uint64_t bytes = api.clip_bytes((int)n);
    const Tensor ws = workspace(bytes, grads[0]);
    check(api.clip(table.data(), (int)n, (float)max_norm, (float)inv_scale, norm.data_ptr<float>(), data(ws), bytes, stream_of(grads[0])),
          "rb200k_grad_clip");
    for (size_t i = 0; i < n; i++) written(out[i]);
    for (auto& b : back) b.first.copy_(b.second);
    return norm;
}

// ---- single launches (rocal_b200.kernels) -----------------------------------------------------------------------
std::pair<Tensor, MaybeTensor> linear_raw(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& residual,
                                          const std::string& act, const MaybeTensor& out, bool want_preact, const MaybeTensor& status,
                                          std::optional<std::pair<uint64_t, int>> probe, bool watched) {
    Tensor preact;
    Tensor y = linear_run(x, weight, or_undefined(bias), or_undefined(residual), activation(act), or_undefined(out), want_preact ? &preact : nullptr,
                          Status{status, watched}, probe);
    return {y, want_preact ? MaybeTensor(preact) : std::nullopt};
}
template <typename G>
std::vector<MaybeTensor> listed(const G& g) {
    std::vector<MaybeTensor> r;
    for (const Tensor& t : g) r.push_back(t.defined() ? MaybeTensor(t) : std::nullopt);
    return r;
}

}  // namespace

PYBIND11_MODULE(_head, m) {
    py::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const LibraryError& e) {
            PyErr_SetString(library_error ? library_error : PyExc_RuntimeError, e.what());
        }
    });
    m.def("bind", &bind);
    m.def("linear", &linear);
    m.def("linear_cross_entropy", &linear_cross_entropy);
    m.def("grad_clip", &grad_clip);
    m.def("share_memory", [](const Tensor& a, const Tensor& b) { return share_memory(Extent(a), Extent(b)); });
    m.def("overlaps_itself", &overlaps_itself);
    m.def("check_unfinished", &check_unfinished);
    m.def("linear_raw", &linear_raw, py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(),
          py::arg("watched") = false);
    m.def("linear_backward_raw", [](const Tensor& dout, const Tensor& x, const Tensor& weight, const MaybeTensor& preact, const std::string& act,
                                    int64_t residual_rows, std::array<bool, 4> need, const MaybeTensor& status) {
        return listed(linear_backward_run(dout, x, weight, or_undefined(preact), activation(act), residual_rows, need, Status{status}));
    });
    m.def("linear_ce_raw", [](const Tensor& x, const Tensor& weight, const Tensor& labels, const MaybeTensor& bias, int64_t ignore_index,
                              double smoothing, const std::string& reduce, const MaybeTensor& status) {
        return listed(ce_run(x, weight, labels, or_undefined(bias), ignore_index, smoothing, reduction(reduce), Status{status}));
    });
    m.def("linear_ce_backward_raw", [](const Tensor& dloss, const Tensor& x, const Tensor& weight, const Tensor& labels, const Tensor& stats,
                                       const Tensor& info, const MaybeTensor& bias, int64_t ignore_index, double smoothing,
                                       const std::string& reduce, std::array<bool, 3> need, const MaybeTensor& status) {
        return listed(ce_backward_run(dloss, x, weight, labels, stats, info, or_undefined(bias), ignore_index, smoothing, reduction(reduce), need,
                                      {status}));
    });
}
