// Python binding of the operators around the layer (a norm takes the GPU 2 us: argument checks, output tensors and the call have to cost less than they do in Python).
// Checks tensors, allocates outputs and workspaces from torch's allocator on the current stream, and calls the C ABI; any error becomes a RuntimeError.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/megamoe_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

const Tensor* optional_tensor(PyObject* o, const char* name) {
    if (o == Py_None) return nullptr;
    TORCH_CHECK(THPVariable_Check(o), name, " must be a tensor");
    return &THPVariable_Unpack(o);
}
const Tensor& tensor(PyObject* o, const char* name) {
    const Tensor* t = optional_tensor(o, name);
    TORCH_CHECK(t != nullptr, name, " must be a tensor");
    return *t;
}
double number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); TORCH_CHECK(false, name, " must be a number"); }
    return v;
}
int64_t whole(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); TORCH_CHECK(false, name, " must be a whole number"); }
    return v;
}

int dtype_of(ScalarType t) { return t == at::kBFloat16 ? MM_DTYPE_BF16 : (t == at::kHalf ? MM_DTYPE_FP16 : (t == at::kFloat ? MM_DTYPE_FP32 : -1)); }
void* address(const Tensor* t) { return t != nullptr ? t->data_ptr() : nullptr; }

Tensor empty(at::IntArrayRef shape, ScalarType type, const Tensor& like) { return at::detail::empty_cuda(shape, type, like.device(), std::nullopt); }
// a tensor of the caller's that has been written: autograd is to know (inference tensors keep no count)
void written(const Tensor* t) {
    if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
// Nothing here is recorded by autograd: an input that asks for a gradient would not get it, an output that asks for one would be written behind autograd's back.
void no_tangent(const char* call, const Tensor* t, const char* name) {
    TORCH_CHECK(t == nullptr || !c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t->_fw_grad(0).defined(), call, " is not recorded by autograd, and ", name,
                " carries a forward-mode derivative");
}
void not_recorded(const char* call, const Tensor* t, const char* name, const char* backward) {
    if (t == nullptr) return;
    TORCH_CHECK(!c10::GradMode::is_enabled() || !t->requires_grad(), call, " is not recorded by autograd, and ", name, " requires a gradient: call it under torch.no_grad(), with "
                "detached tensors, or in a torch.autograd.Function whose backward pass calls ", backward);
    no_tangent(call, t, name);
}
void not_written(const char* call, const Tensor* t, const char* name) {
    TORCH_CHECK(t == nullptr || !c10::GradMode::is_enabled() || !t->requires_grad(), call, " is not recorded by autograd, and would write ", name,
                ", which requires a gradient: call it under torch.no_grad(), or give a detached tensor");
    no_tangent(call, t, name);
}
PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap_or_none(const Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}
PyObject* tuple_of(std::initializer_list<PyObject*> items) {
    PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
    Py_ssize_t i = 0;
    for (PyObject* o : items) PyTuple_SET_ITEM(out, i++, o);
    return out;
}

void check(int status, const char* what) {
    if (status == MM_OK) return;
    if (status == MM_ERR_CUDA) TORCH_CHECK(false, what, ": ", mm_status_string(status), " (", mm_last_cuda_error(), ")");
    TORCH_CHECK(false, what, ": ", mm_status_string(status));
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// ----------------------------------------------------------------------------- norms
// Row stride of a [tokens, hidden] tensor whose rows are packed.
int64_t rows(const Tensor& t, const char* name, int64_t tokens, int64_t hidden, ScalarType type, const Tensor& like) {
    TORCH_CHECK(t.dim() == 2 && t.size(0) == tokens && t.size(1) == hidden && t.scalar_type() == type, name, " must be ", type, " [", tokens, ", ", hidden, "]");
    TORCH_CHECK(t.device() == like.device(), name, " must be on the GPU of the other tensors");
    TORCH_CHECK(hidden <= 1 || t.stride(1) == 1, "the channels of ", name, " must lie next to each other");
    return t.stride(0);
}

struct Block {
    mm_block_norm_args_t a;
    const Tensor *residual, *y, *gate, *pre, *post;
    ScalarType type;
};

// What both directions check: the inputs, and `type`, that of the activations.
Block block_inputs(PyObject* const* arg, ScalarType type, const Tensor& residual, const Tensor* y) {
    Block b;
    memset(&b.a, 0, sizeof(b.a));
    b.residual = &residual; b.y = y; b.type = type;
    b.pre = optional_tensor(arg[0], "pre_weight");
    b.post = optional_tensor(arg[1], "post_weight");
    b.gate = optional_tensor(arg[2], "gate");
    const ScalarType stream = residual.scalar_type();
    TORCH_CHECK(residual.dim() == 2 && residual.is_cuda() && dtype_of(stream) >= 0 && dtype_of(type) >= 0,
                "residual must be a CUDA [tokens, hidden] tensor; types are bf16, fp16 and fp32");
    TORCH_CHECK(stream == type || stream == at::kFloat, "the residual stream must be of the type of the activations or fp32");
    const int64_t tokens = residual.size(0), hidden = residual.size(1);
    TORCH_CHECK(tokens <= (1ll << 30), "at most 2^30 tokens");
    TORCH_CHECK(hidden >= 1 && hidden <= 8192, "hidden must be 1 to 8192");
    TORCH_CHECK(y != nullptr || (b.gate == nullptr && b.post == nullptr && b.pre != nullptr),
                "without y there is only the norm of the stream: pre_weight, and neither post_weight nor gate");
    TORCH_CHECK(b.pre == nullptr || b.post == nullptr || b.pre->scalar_type() == b.post->scalar_type(), "both weights must be of one type");
    b.a.residual = address(&residual);
    b.a.residual_stride = rows(residual, "residual", tokens, hidden, stream, residual);
    if (y != nullptr) { b.a.y = address(y); b.a.y_stride = rows(*y, "y", tokens, hidden, type, residual); }
    for (const Tensor* w : {b.pre, b.post}) {
        if (w == nullptr) continue;
        TORCH_CHECK(w->dim() == 1 && w->size(0) == hidden && (w->scalar_type() == type || w->scalar_type() == at::kFloat) && w->device() == residual.device() && w->is_contiguous(),
                    "weights must be contiguous [hidden] tensors of the type of the activations or fp32, on their GPU");
        b.a.weight_dtype = dtype_of(w->scalar_type());
    }
    if (b.pre == nullptr && b.post == nullptr) b.a.weight_dtype = dtype_of(type);
    b.a.pre_weight = address(b.pre);
    b.a.post_weight = address(b.post);
    b.a.gate_dtype = dtype_of(type);
    if (b.gate != nullptr) {
        const Tensor& g = *b.gate;
        TORCH_CHECK((g.scalar_type() == type || g.scalar_type() == at::kFloat) && g.device() == residual.device(), "gate must be of the type of the activations or fp32, on their GPU");
        if (g.dim() == 1 && g.size(0) == hidden && g.is_contiguous()) {
            b.a.gate_mode = MM_GATE_CHANNEL;
        } else if (g.dim() == 2 && g.size(0) == tokens && g.size(1) == hidden && (hidden == 1 || g.stride(1) == 1)) {
            b.a.gate_mode = MM_GATE_ELEMENT;
            b.a.gate_stride = g.stride(0);
        } else {
            TORCH_CHECK(g.dim() == 2 && g.size(0) == tokens && g.size(1) == 1, "gate must be [hidden], [tokens, 1] or [tokens, hidden], its channels next to each other");
            b.a.gate_mode = MM_GATE_TOKEN;
            b.a.gate_stride = g.stride(0);
        }
        b.a.gate_dtype = dtype_of(g.scalar_type());
        b.a.gate = address(&g);
    }
    b.a.tokens = tokens;
    b.a.hidden = static_cast<int32_t>(hidden);
    b.a.dtype = dtype_of(type);
    b.a.stream_dtype = dtype_of(stream);
    b.a.scale = static_cast<float>(number(arg[3], "scale"));
    b.a.eps = static_cast<float>(number(arg[4], "eps"));
    b.a.weight_offset = static_cast<float>(number(arg[5], "weight_offset"));
    return b;
}

// residual, y, pre_weight, post_weight, gate, scale, eps, weight_offset, residual_out, normed
PyObject* block_norm(PyObject*, PyObject* const* arg, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 10, "block_norm: arguments");
    const Tensor& residual = tensor(arg[0], "residual");
    const Tensor* y = optional_tensor(arg[1], "y");
    const Tensor *out = optional_tensor(arg[8], "residual_out"), *normed = optional_tensor(arg[9], "normed");
    not_recorded("block_norm", &residual, "residual", "block_norm_backward");
    not_recorded("block_norm", y, "y", "block_norm_backward");
    not_recorded("block_norm", optional_tensor(arg[2], "pre_weight"), "pre_weight", "block_norm_backward");
    not_recorded("block_norm", optional_tensor(arg[3], "post_weight"), "post_weight", "block_norm_backward");
    not_recorded("block_norm", optional_tensor(arg[4], "gate"), "gate", "block_norm_backward");
    not_written("block_norm", out, "residual_out");
    not_written("block_norm", normed, "normed");
    const ScalarType type = y != nullptr ? y->scalar_type() : (normed != nullptr ? normed->scalar_type() : residual.scalar_type());
    Block b = block_inputs(arg + 2, type, residual, y);
    const int64_t tokens = b.a.tokens, hidden = b.a.hidden;
    TORCH_CHECK(y != nullptr || out == nullptr, "without y the stream stays as it is: no residual_out");
    TORCH_CHECK(b.pre != nullptr || normed == nullptr, "normed needs pre_weight");
    Tensor own_out, own_normed;
    if (y != nullptr) {
        if (out == nullptr) { own_out = empty({tokens, hidden}, residual.scalar_type(), residual); out = &own_out; }
        b.a.residual_out_stride = rows(*out, "residual_out", tokens, hidden, residual.scalar_type(), residual);
        b.a.residual_out = address(out);
    }
    if (b.pre != nullptr) {
        if (normed == nullptr) { own_normed = empty({tokens, hidden}, type, residual); normed = &own_normed; }
        b.a.normed_stride = rows(*normed, "normed", tokens, hidden, type, residual);
        b.a.normed = address(normed);
    }
    {
        const c10::cuda::CUDAGuard guard(residual.device());
        check(mm_block_norm(&b.a, stream_of(residual)), "block_norm");
    }
    if (!own_out.defined()) written(y != nullptr ? out : nullptr);
    if (!own_normed.defined()) written(normed);
    PyObject* first = own_out.defined() ? wrap(own_out) : Py_NewRef(y != nullptr ? arg[8] : arg[0]);
    return tuple_of({first, own_normed.defined() ? wrap(own_normed) : Py_NewRef(arg[9])});
    END_HANDLE_TH_ERRORS
}

// d_residual_out, d_normed, residual, y, pre_weight, post_weight, gate, scale, eps, weight_offset
PyObject* block_norm_backward(PyObject*, PyObject* const* arg, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 10, "block_norm_backward: arguments");
    const Tensor *d_out = optional_tensor(arg[0], "d_residual_out"), *d_normed = optional_tensor(arg[1], "d_normed");
    const Tensor& residual = tensor(arg[2], "residual");
    const Tensor* y = optional_tensor(arg[3], "y");
    no_tangent("block_norm_backward", d_out, "d_residual_out");
    no_tangent("block_norm_backward", d_normed, "d_normed");
    no_tangent("block_norm_backward", &residual, "residual");
    no_tangent("block_norm_backward", y, "y");
    for (int i = 4; i < 7; ++i) no_tangent("block_norm_backward", optional_tensor(arg[i], "weights and gate"), "a weight or the gate");
    TORCH_CHECK((d_normed != nullptr) == (arg[4] != Py_None), "d_normed goes with pre_weight");
    TORCH_CHECK(d_normed != nullptr || d_out != nullptr, "the gradient of at least one output must be given");
    const ScalarType type = y != nullptr ? y->scalar_type() : (d_normed != nullptr ? d_normed->scalar_type() : residual.scalar_type());
    Block b = block_inputs(arg + 4, type, residual, y);
    const int64_t tokens = b.a.tokens, hidden = b.a.hidden;
    mm_block_norm_grads_t g;
    memset(&g, 0, sizeof(g));
    if (d_out != nullptr) { g.d_residual_out = address(d_out); g.d_residual_out_stride = rows(*d_out, "d_residual_out", tokens, hidden, residual.scalar_type(), residual); }
    if (d_normed != nullptr) { g.d_normed = address(d_normed); g.d_normed_stride = rows(*d_normed, "d_normed", tokens, hidden, type, residual); }
    Tensor d_residual = empty({tokens, hidden}, residual.scalar_type(), residual), d_y, d_gate, d_pre, d_post, workspace;
    if (y != nullptr) d_y = empty({tokens, hidden}, type, residual);
    if (b.gate != nullptr) d_gate = empty(b.gate->sizes(), b.gate->scalar_type(), residual);
    if (b.pre != nullptr) d_pre = empty({hidden}, b.pre->scalar_type(), residual);
    if (b.post != nullptr) d_post = empty({hidden}, b.post->scalar_type(), residual);
    if (tokens > 0 && (d_pre.defined() || d_post.defined() || b.a.gate_mode == MM_GATE_CHANNEL)) {
        g.workspace_bytes = mm_block_norm_workspace_bytes(tokens, static_cast<int32_t>(hidden));
        workspace = empty({g.workspace_bytes}, at::kByte, residual);
        g.workspace = workspace.data_ptr();
    }
    g.d_residual = d_residual.data_ptr();
    g.d_y = d_y.defined() ? d_y.data_ptr() : nullptr;
    g.d_gate = d_gate.defined() ? d_gate.data_ptr() : nullptr;
    g.d_pre_weight = d_pre.defined() ? d_pre.data_ptr() : nullptr;
    g.d_post_weight = d_post.defined() ? d_post.data_ptr() : nullptr;
    g.d_residual_stride = g.d_y_stride = hidden;
    g.d_gate_stride = b.a.gate_mode == MM_GATE_TOKEN ? 1 : hidden;
    {
        const c10::cuda::CUDAGuard guard(residual.device());
        check(mm_block_norm_backward(&b.a, &g, stream_of(residual)), "block_norm_backward");
    }
    return tuple_of({wrap(d_residual), wrap_or_none(d_y), wrap_or_none(d_gate), wrap_or_none(d_pre), wrap_or_none(d_post)});
    END_HANDLE_TH_ERRORS
}

// ----------------------------------------------------------------------------- router
// What every call says about its logits.
mm_router_args_t router_inputs(const Tensor& logits, int64_t topk, PyObject* mode) {
    TORCH_CHECK(logits.dim() == 2 && logits.is_cuda() && dtype_of(logits.scalar_type()) >= 0, "logits must be a CUDA bf16, fp16 or fp32 [tokens, experts] tensor");
    const int64_t tokens = logits.size(0), experts = logits.size(1), score_mode = whole(mode, "score_mode");
    TORCH_CHECK((experts <= 1 || logits.stride(1) == 1) && (tokens <= 1 || logits.stride(0) >= experts), "the logits of a token must lie next to each other, and apart from other tokens'");
    TORCH_CHECK(topk >= 1 && topk <= 32 && topk <= experts && experts <= 1024, "topk must be 1 to 32 of at most 1024 experts");
    TORCH_CHECK(score_mode == 0 || score_mode == 1, "score_mode must be 0 (softmax) or 1 (sigmoid)");
    TORCH_CHECK(tokens <= (1 << 27), "at most 2^27 tokens");
    mm_router_args_t a;
    memset(&a, 0, sizeof(a));
    a.logits = address(&logits);
    a.logits_stride = logits.stride(0);
    a.tokens = static_cast<int32_t>(tokens);
    a.num_experts = static_cast<int32_t>(experts);
    a.topk = static_cast<int32_t>(topk);
    a.dtype = dtype_of(logits.scalar_type());
    a.score_mode = static_cast<int32_t>(score_mode);
    a.route_scale = 1.f;
    return a;
}
void* plain(const Tensor& t, const char* name, at::IntArrayRef shape, ScalarType type, const Tensor& like) {
    TORCH_CHECK(t.sizes() == shape && t.scalar_type() == type && t.device() == like.device() && t.is_contiguous(), name, " must be a contiguous ", type, " ", shape,
                " tensor on the GPU of the logits");
    return t.data_ptr();
}
int64_t topk_of(const Tensor& idx) {
    TORCH_CHECK(idx.dim() == 2, "topk_idx must be [tokens, topk]");
    return idx.size(1);
}
int32_t* sequences(const Tensor* cu, const Tensor& logits, int64_t* n) {
    *n = 1;
    if (cu == nullptr) return nullptr;
    TORCH_CHECK(cu->dim() == 1 && cu->size(0) >= 2 && cu->size(0) <= (1 << 21) + 1, "cu_seqlens must be int32 [sequences + 1] of at most 2^21 sequences");
    *n = cu->size(0) - 1;
    return static_cast<int32_t*>(plain(*cu, "cu_seqlens", cu->sizes(), at::kInt, logits));
}

// logits, topk, score_mode, expert_bias, valid, route_scale, topk_idx, topk_weights
PyObject* route_tokens(PyObject*, PyObject* const* arg, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 8, "route_tokens: arguments");
    const Tensor& logits = tensor(arg[0], "logits");
    const Tensor *bias = optional_tensor(arg[3], "expert_bias"), *valid = optional_tensor(arg[4], "valid");      // (neither has a gradient)
    const Tensor *idx = optional_tensor(arg[6], "topk_idx"), *weights = optional_tensor(arg[7], "topk_weights");
    not_recorded("route_tokens", &logits, "logits", "router_backward");
    not_written("route_tokens", weights, "topk_weights");
    mm_router_args_t a = router_inputs(logits, whole(arg[1], "topk"), arg[2]);
    a.route_scale = static_cast<float>(number(arg[5], "route_scale"));
    const int64_t shape[2] = {a.tokens, a.topk};
    const float* bias_ptr = nullptr;
    const uint8_t* valid_ptr = nullptr;
    if (bias != nullptr) {
        TORCH_CHECK(a.score_mode == 1, "expert_bias goes with score_mode 1");
        bias_ptr = static_cast<const float*>(plain(*bias, "expert_bias", {a.num_experts}, at::kFloat, logits));
    }
    if (valid != nullptr) valid_ptr = static_cast<const uint8_t*>(plain(*valid, "valid", {a.tokens}, valid->scalar_type() == at::kByte ? at::kByte : at::kBool, logits));
    Tensor own_idx, own_weights;
    if (idx == nullptr) { own_idx = empty(shape, at::kLong, logits); idx = &own_idx; }
    if (weights == nullptr) { own_weights = empty(shape, at::kFloat, logits); weights = &own_weights; }
    a.topk_idx = static_cast<int64_t*>(plain(*idx, "topk_idx", shape, at::kLong, logits));
    a.topk_weights = static_cast<float*>(plain(*weights, "topk_weights", shape, at::kFloat, logits));
    {
        const c10::cuda::CUDAGuard guard(logits.device());
        check(mm_route_tokens(&a, bias_ptr, valid_ptr, stream_of(logits)), "route_tokens");
    }
    if (!own_idx.defined()) written(idx);
    if (!own_weights.defined()) written(weights);
    return tuple_of({own_idx.defined() ? wrap(own_idx) : Py_NewRef(arg[6]), own_weights.defined() ? wrap(own_weights) : Py_NewRef(arg[7])});
    END_HANDLE_TH_ERRORS
}

// logits, topk_idx, score_mode, cu_seqlens, balance_coef, z_coef
PyObject* balance_loss(PyObject*, PyObject* const* arg, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 6, "balance_loss: arguments");
    const Tensor &logits = tensor(arg[0], "logits"), &idx = tensor(arg[1], "topk_idx");
    not_recorded("balance_loss", &logits, "logits", "router_backward");
    mm_router_args_t a = router_inputs(logits, topk_of(idx), arg[2]);
    a.topk_idx = static_cast<int64_t*>(plain(idx, "topk_idx", {a.tokens, a.topk}, at::kLong, logits));
    mm_balance_args_t b;
    memset(&b, 0, sizeof(b));
    int64_t s = 1;
    b.cu_seqlens = sequences(optional_tensor(arg[3], "cu_seqlens"), logits, &s);
    b.num_sequences = static_cast<int32_t>(s);
    b.balance_coef = static_cast<float>(number(arg[4], "balance_coef"));
    b.z_coef = static_cast<float>(number(arg[5], "z_coef"));
    const int64_t bytes = mm_balance_workspace_bytes(a.num_experts, b.num_sequences);
    const Tensor losses = empty({3}, at::kFloat, logits), counts = empty({s, a.num_experts}, at::kInt, logits), mean = empty({s, a.num_experts}, at::kFloat, logits),
                 tokens = empty({s}, at::kInt, logits), workspace = empty({bytes}, at::kByte, logits);
    b.losses = static_cast<float*>(losses.data_ptr());
    b.counts = static_cast<int32_t*>(counts.data_ptr());
    b.mean_probs = static_cast<float*>(mean.data_ptr());
    b.seq_tokens = static_cast<int32_t*>(tokens.data_ptr());
    {
        const c10::cuda::CUDAGuard guard(logits.device());
        check(mm_balance_loss(&a, &b, workspace.data_ptr(), bytes, stream_of(logits)), "balance_loss");
    }
    return tuple_of({wrap(losses), wrap(counts), wrap(mean), wrap(tokens)});
    END_HANDLE_TH_ERRORS
}

// logits, topk_idx, score_mode, d_topk_weights, route_scale, counts (None: no balance loss), seq_tokens, cu_seqlens, balance_coef, z_coef, d_loss, d_logits
PyObject* router_backward(PyObject*, PyObject* const* arg, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 12, "router_backward: arguments");
    const Tensor &logits = tensor(arg[0], "logits"), &idx = tensor(arg[1], "topk_idx");
    no_tangent("router_backward", &logits, "logits");
    no_tangent("router_backward", optional_tensor(arg[3], "d_topk_weights"), "d_topk_weights");
    if (THPVariable_Check(arg[10])) no_tangent("router_backward", &THPVariable_Unpack(arg[10]), "d_loss");
    not_written("router_backward", optional_tensor(arg[11], "d_logits"), "d_logits");
    mm_router_args_t a = router_inputs(logits, topk_of(idx), arg[2]);
    const int64_t shape[2] = {a.tokens, a.topk};
    a.topk_idx = static_cast<int64_t*>(plain(idx, "topk_idx", shape, at::kLong, logits));
    a.route_scale = static_cast<float>(number(arg[4], "route_scale"));
    const Tensor *dw = optional_tensor(arg[3], "d_topk_weights"), *counts = optional_tensor(arg[5], "balance.counts");
    TORCH_CHECK(dw != nullptr || counts != nullptr, "d_topk_weights or balance must be given");
    const float* dw_ptr = dw != nullptr ? static_cast<const float*>(plain(*dw, "d_topk_weights", shape, at::kFloat, logits)) : nullptr;
    mm_balance_args_t b;
    memset(&b, 0, sizeof(b));
    if (counts != nullptr) {
        int64_t s = 1;
        b.cu_seqlens = sequences(optional_tensor(arg[7], "cu_seqlens"), logits, &s);
        b.num_sequences = static_cast<int32_t>(s);
        b.counts = static_cast<int32_t*>(plain(*counts, "balance.counts", {s, a.num_experts}, at::kInt, logits));
        b.seq_tokens = static_cast<int32_t*>(plain(tensor(arg[6], "balance.tokens"), "balance.tokens", {s}, at::kInt, logits));
        b.balance_coef = static_cast<float>(number(arg[8], "balance_coef"));
        b.z_coef = static_cast<float>(number(arg[9], "z_coef"));
    }
    float d_loss = 0.f;
    const float* d_loss_ptr = nullptr;
    if (THPVariable_Check(arg[10])) {
        const Tensor& t = THPVariable_Unpack(arg[10]);
        TORCH_CHECK(t.numel() == 1 && t.scalar_type() == at::kFloat && t.device() == logits.device(), "d_loss must be a number or an fp32 tensor with one element on the GPU of the logits");
        d_loss_ptr = static_cast<const float*>(t.data_ptr());
    } else {
        d_loss = static_cast<float>(number(arg[10], "d_loss"));
    }
    const Tensor* d = optional_tensor(arg[11], "d_logits");
    Tensor own;
    if (d == nullptr) { own = empty({a.tokens, a.num_experts}, logits.scalar_type(), logits); d = &own; }
    TORCH_CHECK(d->dim() == 2 && d->sizes() == logits.sizes() && d->scalar_type() == logits.scalar_type() && d->device() == logits.device() && (a.num_experts <= 1 || d->stride(1) == 1),
                "d_logits must be like the logits");
    {
        const c10::cuda::CUDAGuard guard(logits.device());
        check(mm_router_backward(&a, dw_ptr, counts != nullptr ? &b : nullptr, d_loss, d_loss_ptr, d->data_ptr(), d->stride(0), stream_of(logits)), "router_backward");
    }
    if (own.defined()) return wrap(own);
    written(d);
    return Py_NewRef(arg[11]);
    END_HANDLE_TH_ERRORS
}

#define MM_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MM_METHOD(block_norm), MM_METHOD(block_norm_backward), MM_METHOD(route_tokens), MM_METHOD(balance_loss), MM_METHOD(router_backward), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "mm_block_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// `built_for`: the torch and the Python that it was compiled against, which the package looks for in the file before it loads it
PyMODINIT_FUNC PyInit_mm_block_binding(void) {
    PyObject* m = PyModule_Create(&module);
    if (m != nullptr && PyModule_AddStringConstant(m, "built_for", MM_BUILT_FOR) != 0) { Py_DECREF(m); return nullptr; }
    return m;
}
