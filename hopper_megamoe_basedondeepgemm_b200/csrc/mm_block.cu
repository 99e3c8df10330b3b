// C ABI of the operators around the layer: a block's norms, routing from logits, the balance loss. Argument checks and launches; no torch types, no exceptions.
#include <cuda_runtime.h>
#include <cfloat>
#include <cmath>
#include <cstring>

#include "../../include/megamoe_b200.h"
#include "mm_block_norm.h"
#include "mm_router.h"
#include "mm_error.h"

namespace {

int sm_count(int* out) {
    int dev = 0;
    MM_CUDA(cudaGetDevice(&dev));
    MM_CUDA(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
    return MM_OK;
}

int dtype_bytes(int dtype) { return dtype == MM_DTYPE_FP32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype == MM_DTYPE_BF16 || dtype == MM_DTYPE_FP16 || dtype == MM_DTYPE_FP32; }

// ----------------------------------------------------------------------------- norms
// Rows of a tensor in memory: what two of them share decides whether one may be written while the other is read.
struct Rows {
    const void* p;
    int64_t ld, width;                       // bytes between rows, bytes of a row
    int64_t n;
};

bool share_memory(const Rows& a, const Rows& b) {
    if (a.p == nullptr || b.p == nullptr || a.n == 0 || b.n == 0) return false;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    const uintptr_t ea = pa + (a.n - 1) * a.ld + a.width, eb = pb + (b.n - 1) * b.ld + b.width;
    if (ea <= pb || eb <= pa) return false;
    const int64_t ld = a.n == 1 ? b.ld : a.ld;                              // (a single one may lie between the others' rows)
    if ((b.n != 1 && b.ld != ld) || ld == 0) return true;
    const int64_t d = pa > pb ? static_cast<int64_t>((pa - pb) % ld) : static_cast<int64_t>((pb - pa) % ld);
    const int64_t first = pa > pb ? b.width : a.width, second = pa > pb ? a.width : b.width;       // columns of one buffer lie beside each other
    return !(d >= first && ld - d >= second);
}

// An output may be the very rows of an input that is read by the thread which writes them, and nothing else of any tensor of the call.
bool writes_safely(const Rows& out, const Rows* others, int n, bool in_place) {
    for (int i = 0; i < n; ++i)
        if (share_memory(out, others[i]) && !(in_place && out.p == others[i].p && out.ld == others[i].ld && out.width == others[i].width)) return false;
    return true;
}

int norm_check(const mm_block_norm_args_t* a) {
    if (a == nullptr || a->tokens < 0 || a->tokens > (1ll << 30) || a->hidden < 1) return MM_ERR_INVALID_ARGUMENT;
    if (!known_dtype(a->dtype) || !known_dtype(a->stream_dtype) || !known_dtype(a->weight_dtype) || !known_dtype(a->gate_dtype)) return MM_ERR_INVALID_ARGUMENT;
    if (a->hidden > mm::kBnMaxHidden) return MM_ERR_UNSUPPORTED;
    if (a->stream_dtype != a->dtype && a->stream_dtype != MM_DTYPE_FP32) return MM_ERR_UNSUPPORTED;
    if (a->weight_dtype != a->dtype && a->weight_dtype != MM_DTYPE_FP32) return MM_ERR_UNSUPPORTED;
    if (a->gate_dtype != a->dtype && a->gate_dtype != MM_DTYPE_FP32) return MM_ERR_UNSUPPORTED;
    if (a->gate_mode < MM_GATE_NONE || a->gate_mode > MM_GATE_ELEMENT) return MM_ERR_INVALID_ARGUMENT;
    if (a->tokens > 0) {                     // (tensors of no rows have no address)
        if ((a->gate_mode != MM_GATE_NONE) != (a->gate != nullptr) || (a->gate != nullptr && a->y == nullptr)) return MM_ERR_INVALID_ARGUMENT;
        if (a->y == nullptr && (a->post_weight != nullptr || a->pre_weight == nullptr)) return MM_ERR_INVALID_ARGUMENT;
    }
    // (a subnormal eps would stand beside squares that 32 bits no longer hold)
    if (!(a->eps >= FLT_MIN) || !std::isfinite(a->eps) || !std::isfinite(a->scale) || !std::isfinite(a->weight_offset)) return MM_ERR_INVALID_ARGUMENT;
    return MM_OK;
}

// Rows of a tensor as the call gives them; a single row needs no distance to the next.
Rows rows_of(const void* p, int64_t ld, int64_t n, int32_t hidden, int dtype) {
    return Rows{p, ld * dtype_bytes(dtype), static_cast<int64_t>(hidden) * dtype_bytes(dtype), n};
}

// Whether every row starts on 16 bytes, one of 32-bit elements on 32, and is made of whole groups of eight elements.
bool norm_rows_aligned(int hidden, const Rows* rows, int n) {
    if (hidden % 8 != 0) return false;
    for (int i = 0; i < n; ++i) {
        const int unit = rows[i].width == static_cast<int64_t>(hidden) * 4 ? 32 : 16;
        if (rows[i].p != nullptr && (reinterpret_cast<uintptr_t>(rows[i].p) % unit != 0 || rows[i].ld % unit != 0)) return false;
    }
    return true;
}

mm::BnParams norm_params(const mm_block_norm_args_t* a) {
    mm::BnParams q;
    memset(&q, 0, sizeof(q));
    q.residual = a->residual; q.y = a->y; q.gate = a->gate; q.pre_w = a->pre_weight; q.post_w = a->post_weight;
    q.residual_out = a->residual_out; q.normed = a->normed;
    q.tokens = a->tokens;
    q.residual_ld = a->residual_stride; q.y_ld = a->y_stride; q.gate_ld = a->gate_stride;
    q.residual_out_ld = a->residual_out_stride; q.normed_ld = a->normed_stride;
    q.hidden = a->hidden; q.gate_mode = a->gate_mode;
    q.weight32 = a->weight_dtype == MM_DTYPE_FP32; q.gate32 = a->gate_dtype == MM_DTYPE_FP32;
    q.scale = a->scale; q.eps = a->eps; q.offset = a->weight_offset;
    return q;
}

int launch_norm(int dtype, const mm::BnParams& q, const mm::BnLaunch& how, cudaStream_t stream) {
    return dtype == MM_DTYPE_BF16 ? mm::launch_block_norm_bf16(q, how, stream)
                                  : (dtype == MM_DTYPE_FP16 ? mm::launch_block_norm_fp16(q, how, stream) : mm::launch_block_norm_fp32(q, how, stream));
}

// ----------------------------------------------------------------------------- router
int router_check(const mm_router_args_t* a) {
    if (a == nullptr || a->tokens < 0 || a->num_experts < 1 || a->topk < 1) return MM_ERR_INVALID_ARGUMENT;
    if (!known_dtype(a->dtype) || (a->score_mode != 0 && a->score_mode != 1)) return MM_ERR_INVALID_ARGUMENT;
    if (a->num_experts > mm::kRtMaxExperts || a->topk > mm::kRtMaxTopk || a->tokens > (1 << 27)) return MM_ERR_UNSUPPORTED;
    if (a->topk > a->num_experts) return MM_ERR_INVALID_ARGUMENT;
    if (a->tokens > 0 && (a->logits == nullptr || a->topk_idx == nullptr)) return MM_ERR_INVALID_ARGUMENT;
    if (a->tokens > 1 && a->logits_stride < a->num_experts) return MM_ERR_INVALID_ARGUMENT;
    return MM_OK;
}

Rows logit_rows(const mm_router_args_t* a, const void* p, int64_t ld) {
    const int64_t bytes = dtype_bytes(a->dtype);
    return Rows{p, a->tokens > 1 ? ld * bytes : 0, a->num_experts * bytes, a->tokens};      // (how far the row behind a single one would be says nothing)
}
// A tensor without gaps, as rows: its own only one.
Rows packed(const void* p, int64_t bytes) { return Rows{p, 0, bytes, 1}; }

// Whether the router's outputs lie apart from each other and from what is read.
bool lie_apart(const Rows* outputs, int n_out, const Rows* inputs, int n_in) {
    for (int i = 0; i < n_out; ++i)
        if (!writes_safely(outputs[i], inputs, n_in, false) || !writes_safely(outputs[i], outputs + i + 1, n_out - i - 1, false)) return false;
    return true;
}

mm::RtParams router_params(const mm_router_args_t* a) {
    mm::RtParams q;
    memset(&q, 0, sizeof(q));
    q.logits = a->logits; q.logits_ld = a->logits_stride;
    q.idx = reinterpret_cast<long long*>(a->topk_idx); q.weights = a->topk_weights;
    q.T = a->tokens; q.E = a->num_experts; q.K = a->topk; q.S = 1; q.mode = a->score_mode;
    q.route_scale = a->route_scale;
    return q;
}

void balance_params(const mm_balance_args_t* b, mm::RtParams& q) {
    q.cu = b->cu_seqlens; q.S = b->num_sequences;
    q.balance_coef = b->balance_coef; q.z_coef = b->z_coef;
    q.counts = b->counts; q.tokens = b->seq_tokens; q.mean = b->mean_probs; q.losses = b->losses;
}

constexpr int kMaxSequences = 1 << 21;       // times 1024 experts: sums are numbered in 32 bits

int balance_check(const mm_balance_args_t* b) {
    if (b == nullptr || b->num_sequences < 1 || (b->cu_seqlens == nullptr && b->num_sequences != 1)) return MM_ERR_INVALID_ARGUMENT;
    if (b->num_sequences > kMaxSequences) return MM_ERR_UNSUPPORTED;
    if (b->counts == nullptr || b->seq_tokens == nullptr) return MM_ERR_INVALID_ARGUMENT;
    if (!std::isfinite(b->balance_coef) || !std::isfinite(b->z_coef)) return MM_ERR_INVALID_ARGUMENT;
    return MM_OK;
}

int launch_router(int dtype, mm::RtOp op, const mm::RtParams& q, void* stream) {
    int sms = 0;
    const int st = sm_count(&sms);
    if (st != MM_OK) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == MM_DTYPE_BF16 ? mm::launch_router_bf16(op, q, sms, s)
                                  : (dtype == MM_DTYPE_FP16 ? mm::launch_router_fp16(op, q, sms, s) : mm::launch_router_fp32(op, q, sms, s));
}

// Workspace of the balance loss: the sums (zeroed by the call), then a number per CTA.
int64_t balance_zeroed_bytes(int64_t experts, int64_t sequences) { return (sequences * experts * 12 + sequences * 4 + 4 + 7) / 8 * 8; }

}  // namespace

extern "C" {

int mm_block_norm(const mm_block_norm_args_t* a, void* stream_ptr) {
    int st = norm_check(a);
    if (st != MM_OK) return st;
    if (a->tokens == 0) return MM_OK;
    if (a->residual == nullptr || (a->y != nullptr) != (a->residual_out != nullptr) || (a->pre_weight != nullptr) != (a->normed != nullptr)) return MM_ERR_INVALID_ARGUMENT;
    const bool element = a->gate_mode == MM_GATE_ELEMENT;
    const int64_t t = a->tokens;
    Rows rows[7] = {rows_of(a->residual_out, a->residual_out_stride, t, a->hidden, a->stream_dtype), rows_of(a->normed, a->normed_stride, t, a->hidden, a->dtype),
                    rows_of(a->residual, a->residual_stride, t, a->hidden, a->stream_dtype), rows_of(a->y, a->y_stride, t, a->hidden, a->dtype),
                    element ? rows_of(a->gate, a->gate_stride, t, a->hidden, a->gate_dtype)
                            : rows_of(a->gate, a->gate_mode == MM_GATE_TOKEN ? a->gate_stride : 0, a->gate_mode == MM_GATE_TOKEN ? t : 1,
                                      a->gate_mode == MM_GATE_TOKEN ? 1 : a->hidden, a->gate_dtype),
                    rows_of(a->pre_weight, 0, 1, a->hidden, a->weight_dtype), rows_of(a->post_weight, 0, 1, a->hidden, a->weight_dtype)};
    if (t == 1) for (Rows& r : rows) r.ld = 0;                              // (how far the next row would be says nothing)
    for (int i = 0; i < 2; ++i)
        if (t > 1 && rows[i].p != nullptr && rows[i].ld < rows[i].width) return MM_ERR_INVALID_ARGUMENT;
    if (!writes_safely(rows[0], rows + 1, 1, false) || !writes_safely(rows[0], rows + 2, 2, true) || !writes_safely(rows[0], rows + 4, 3, false) ||
        !writes_safely(rows[1], rows + 2, 2, true) || !writes_safely(rows[1], rows + 4, 3, false)) return MM_ERR_INVALID_ARGUMENT;
    if (a->gate_mode == MM_GATE_TOKEN) rows[4].p = nullptr;                 // (read one by one)
    mm::BnLaunch how = {false, a->stream_dtype == MM_DTYPE_FP32, norm_rows_aligned(a->hidden, rows, 7), 0, 0};
    st = sm_count(&how.sms);
    return st != MM_OK ? st : launch_norm(a->dtype, norm_params(a), how, static_cast<cudaStream_t>(stream_ptr));
}

int64_t mm_block_norm_workspace_bytes(int64_t tokens, int32_t hidden) {
    if (tokens < 0 || hidden < 1 || hidden > mm::kBnMaxHidden) return -1;
    return mm::bn_backward_teams(tokens, hidden) * hidden * 2 * 4;
}

int mm_block_norm_backward(const mm_block_norm_args_t* a, const mm_block_norm_grads_t* g, void* stream_ptr) {
    int st = norm_check(a);
    if (st != MM_OK) return st;
    if (g == nullptr) return MM_ERR_INVALID_ARGUMENT;
    const bool channel = a->gate_mode == MM_GATE_CHANNEL, element = a->gate_mode == MM_GATE_ELEMENT, token = a->gate_mode == MM_GATE_TOKEN;
    if ((a->pre_weight != nullptr) != (g->d_pre_weight != nullptr) || (a->post_weight != nullptr) != (g->d_post_weight != nullptr)) return MM_ERR_INVALID_ARGUMENT;
    const int sums = (a->pre_weight != nullptr) + (a->post_weight != nullptr || channel);
    const int64_t t = a->tokens;
    if (channel && g->d_gate == nullptr) return MM_ERR_INVALID_ARGUMENT;
    if (t > 0) {
        if ((a->pre_weight != nullptr) != (g->d_normed != nullptr) || (a->y != nullptr) != (g->d_y != nullptr) || g->d_residual == nullptr) return MM_ERR_INVALID_ARGUMENT;
        if ((a->pre_weight != nullptr && a->residual == nullptr) || (a->gate != nullptr && g->d_gate == nullptr)) return MM_ERR_INVALID_ARGUMENT;
        if (sums > 0 && (g->workspace == nullptr || g->workspace_bytes < mm_block_norm_workspace_bytes(t, a->hidden) || (reinterpret_cast<uintptr_t>(g->workspace) & 31u) != 0u)) return MM_ERR_INVALID_ARGUMENT;
    }
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    const int64_t teams = mm::bn_backward_teams(t, a->hidden);
    const Rows none = {nullptr, 0, 0, 0};
    // gradients of rows, gradients of channels, working memory; what is read
    Rows rows[14] = {rows_of(g->d_residual, g->d_residual_stride, t, a->hidden, a->stream_dtype), rows_of(g->d_y, g->d_y_stride, t, a->hidden, a->dtype),
                     element ? rows_of(g->d_gate, g->d_gate_stride, t, a->hidden, a->gate_dtype) : (token ? rows_of(g->d_gate, g->d_gate_stride, t, 1, a->gate_dtype) : none),
                     channel ? rows_of(g->d_gate, 0, 1, a->hidden, a->gate_dtype) : none, rows_of(g->d_pre_weight, 0, 1, a->hidden, a->weight_dtype),
                     rows_of(g->d_post_weight, 0, 1, a->hidden, a->weight_dtype), t > 0 && sums > 0 ? Rows{g->workspace, 0, mm_block_norm_workspace_bytes(t, a->hidden), 1} : none,
                     rows_of(g->d_residual_out, g->d_residual_out_stride, t, a->hidden, a->stream_dtype), rows_of(g->d_normed, g->d_normed_stride, t, a->hidden, a->dtype),
                     rows_of(a->residual, a->residual_stride, t, a->hidden, a->stream_dtype), rows_of(a->y, a->y_stride, t, a->hidden, a->dtype),
                     element ? rows_of(a->gate, a->gate_stride, t, a->hidden, a->gate_dtype) : (token ? rows_of(a->gate, a->gate_stride, t, 1, a->gate_dtype) : rows_of(a->gate, 0, 1, a->hidden, a->gate_dtype)),
                     rows_of(a->pre_weight, 0, 1, a->hidden, a->weight_dtype), rows_of(a->post_weight, 0, 1, a->hidden, a->weight_dtype)};
    constexpr int kOutputs = 7;
    if (t == 1) for (Rows& r : rows) r.ld = 0;
    for (int i = 0; i < kOutputs; ++i) {
        if (i < 3 && t > 1 && rows[i].p != nullptr && rows[i].ld < rows[i].width) return MM_ERR_INVALID_ARGUMENT;
        for (int k = i + 1; k < 14; ++k)         // written apart from everything else
            if (share_memory(rows[i], rows[k])) return MM_ERR_INVALID_ARGUMENT;
    }
    if (t > 0) {
        const Rows eights[10] = {rows[0], rows[1], rows[7], rows[8], rows[9], rows[10], rows[12], rows[13], token ? none : rows[2], token ? none : rows[11]};   // (a token's gate is read one by one)
        mm::BnParams q = norm_params(a);
        q.d_residual_out = g->d_residual_out; q.d_residual_out_ld = g->d_residual_out_stride;
        q.d_normed = g->d_normed; q.d_normed_ld = g->d_normed_stride;
        q.d_residual = g->d_residual; q.d_residual_ld = g->d_residual_stride;
        q.d_y = g->d_y; q.d_y_ld = g->d_y_stride;
        q.d_gate = g->d_gate; q.d_gate_ld = g->d_gate_stride;
        q.partial = static_cast<float*>(g->workspace);
        st = launch_norm(a->dtype, q, {true, a->stream_dtype == MM_DTYPE_FP32, norm_rows_aligned(a->hidden, eights, 10), 0, static_cast<int>(teams)}, stream);
        if (st != MM_OK) return st;
    }
    if (sums > 0) {
        mm::BnSumsParams q;
        memset(&q, 0, sizeof(q));
        q.partial = static_cast<const float*>(g->workspace);
        q.rows = static_cast<int>(teams); q.hidden = a->hidden;
        q.gate = channel ? a->gate : nullptr; q.post_w = a->post_weight;
        q.d_pre_w = g->d_pre_weight; q.d_post_w = g->d_post_weight; q.d_gate = channel ? g->d_gate : nullptr;
        q.weight32 = a->weight_dtype == MM_DTYPE_FP32; q.gate32 = a->gate_dtype == MM_DTYPE_FP32;
        q.scale = a->scale; q.offset = a->weight_offset;
        q.sums = sums;
        return a->dtype == MM_DTYPE_BF16 ? mm::launch_block_norm_sums_bf16(q, stream)
                                         : (a->dtype == MM_DTYPE_FP16 ? mm::launch_block_norm_sums_fp16(q, stream) : mm::launch_block_norm_sums_fp32(q, stream));
    }
    return MM_OK;
}

int mm_route_tokens(const mm_router_args_t* a, const float* expert_bias, const uint8_t* valid, void* stream_ptr) {
    int st = router_check(a);
    if (st != MM_OK) return st;
    if ((expert_bias != nullptr && a->score_mode != 1) || !std::isfinite(a->route_scale)) return MM_ERR_INVALID_ARGUMENT;
    if (a->tokens == 0) return MM_OK;
    if (a->topk_weights == nullptr) return MM_ERR_INVALID_ARGUMENT;
    const int64_t t = a->tokens;
    const Rows outputs[2] = {packed(a->topk_idx, t * a->topk * 8), packed(a->topk_weights, t * a->topk * 4)};
    const Rows inputs[3] = {logit_rows(a, a->logits, a->logits_stride), packed(expert_bias, a->num_experts * 4), packed(valid, t)};
    if (!lie_apart(outputs, 2, inputs, 3)) return MM_ERR_INVALID_ARGUMENT;
    mm::RtParams q = router_params(a);
    q.bias = expert_bias; q.valid = valid;
    return launch_router(a->dtype, mm::kRtRoute, q, stream_ptr);
}

int64_t mm_balance_workspace_bytes(int32_t num_experts, int32_t num_sequences) {
    if (num_experts < 1 || num_experts > mm::kRtMaxExperts || num_sequences < 1 || num_sequences > kMaxSequences) return -1;
    return balance_zeroed_bytes(num_experts, num_sequences) + static_cast<int64_t>(mm::kRtBalanceCtas) * 16;
}

int mm_balance_loss(const mm_router_args_t* a, const mm_balance_args_t* b, void* workspace, int64_t workspace_bytes, void* stream_ptr) {
    int st = router_check(a);
    if (st == MM_OK) st = balance_check(b);
    if (st != MM_OK) return st;
    if (b->mean_probs == nullptr || b->losses == nullptr || workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 7u) != 0u ||
        workspace_bytes < mm_balance_workspace_bytes(a->num_experts, b->num_sequences)) return MM_ERR_INVALID_ARGUMENT;
    const int64_t s = b->num_sequences, t = a->tokens;
    const Rows outputs[5] = {packed(b->counts, s * a->num_experts * 4), packed(b->mean_probs, s * a->num_experts * 4), packed(b->seq_tokens, s * 4), packed(b->losses, 12),
                             packed(workspace, workspace_bytes)};
    const Rows inputs[3] = {logit_rows(a, a->logits, a->logits_stride), packed(a->topk_idx, t * a->topk * 8), packed(b->cu_seqlens, s * 4 + 4)};
    if (!lie_apart(outputs, 5, inputs, 3)) return MM_ERR_INVALID_ARGUMENT;
    mm::RtParams q = router_params(a);
    balance_params(b, q);
    const int64_t cells = static_cast<int64_t>(q.S) * q.E, zeroed = balance_zeroed_bytes(q.E, q.S);
    q.sums = static_cast<unsigned long long*>(workspace);
    q.sum_counts = reinterpret_cast<int*>(q.sums + cells);
    q.sum_tokens = q.sum_counts + cells;
    q.ticket = reinterpret_cast<unsigned*>(q.sum_tokens + q.S);
    q.z_part = reinterpret_cast<double*>(static_cast<char*>(workspace) + zeroed);
    q.end_part = q.z_part + mm::kRtBalanceCtas;
    q.zero_words = zeroed / 8;
    return launch_router(a->dtype, mm::kRtBalance, q, stream_ptr);
}

int mm_router_backward(const mm_router_args_t* a, const float* d_topk_weights, const mm_balance_args_t* b, float d_loss, const float* d_loss_ptr,
                       void* d_logits, int64_t d_logits_stride, void* stream_ptr) {
    int st = router_check(a);
    if (st == MM_OK && b != nullptr) st = balance_check(b);
    if (st != MM_OK) return st;
    if ((d_topk_weights == nullptr && b == nullptr) || !std::isfinite(a->route_scale)) return MM_ERR_INVALID_ARGUMENT;
    if (a->tokens == 0) return MM_OK;
    if (d_logits == nullptr || (a->tokens > 1 && d_logits_stride < a->num_experts)) return MM_ERR_INVALID_ARGUMENT;
    const int64_t slots = static_cast<int64_t>(a->tokens) * a->topk, s = b != nullptr ? b->num_sequences : 0;
    const Rows logits = logit_rows(a, a->logits, a->logits_stride), grads = logit_rows(a, d_logits, d_logits_stride);
    const Rows others[6] = {packed(a->topk_idx, slots * 8), packed(d_topk_weights, slots * 4), packed(d_loss_ptr, 4), packed(b != nullptr ? b->counts : nullptr, s * a->num_experts * 4),
                            packed(b != nullptr ? b->seq_tokens : nullptr, s * 4), packed(b != nullptr ? b->cu_seqlens : nullptr, s * 4 + 4)};
    if (!writes_safely(grads, &logits, 1, true) || !writes_safely(grads, others, 6, false)) return MM_ERR_INVALID_ARGUMENT;
    mm::RtParams q = router_params(a);
    if (b != nullptr) balance_params(b, q);
    q.balance = b != nullptr;
    q.d_weights = d_topk_weights; q.d_loss = d_loss; q.d_loss_ptr = d_loss_ptr;
    q.d_logits = d_logits; q.d_logits_ld = d_logits_stride;
    return launch_router(a->dtype, mm::kRtBackward, q, stream_ptr);
}

}  // extern "C"
