// Routing from logits, the balance loss and their gradient: launch parameters, and the entry points of the source files that hold the kernels of one type of
// logits each.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace mm {

constexpr int kRtMaxExperts = 1024, kRtMaxTopk = 32, kRtWarps = 8;
constexpr int kRtBalanceCtas = 1184;         // of the balance kernel at most (eight per SM of 148): the workspace does not depend on the device
constexpr int kRtEndCells = 8192;            // counts that the balance kernel's last CTA turns into the results itself; more of them get a launch of their own

// A balance loss of so few tokens, sequences and sums is one cluster's work.
constexpr int kRtSmallTokens = 384, kRtSmallCells = 2048, kRtSmallSequences = 512, kRtSmallExperts = 384, kRtSmallCtas = 8, kRtSmallWarps = 16;

struct RtParams {
    const void* logits;
    long long logits_ld;
    const float* bias;
    const uint8_t* valid;
    long long* idx;                          // [T][K]
    float* weights;                          // [T][K]
    const int* cu;                           // [S + 1], or nullptr: one sequence of all tokens
    int T, E, K, S, mode;
    int share, shares_more;                  // tokens of a CTA or warp, and how many of the first ones have one more
    float route_scale, balance_coef, z_coef, d_loss;
    float step;                              // of the sums of probabilities
    const float* d_loss_ptr;                 // device scalar, or nullptr: d_loss
    const float* d_weights;                  // [T][K] or nullptr
    int* counts;                             // [S][E]
    int* tokens;                             // [S]
    float* mean;                             // [S][E]
    float* losses;                           // loss, balance, z
    long long zero_words;                    // of 8 bytes, from `sums` on
    // workspace: zero at first
    unsigned long long* sums;                // [S][E]
    int* sum_counts;                         // [S][E]
    int* sum_tokens;                         // [S]
    unsigned* ticket;
    double *z_part, *end_part;               // one per CTA (not zeroed)
    int z_parts, balance;
    void* d_logits;
    long long d_logits_ld;
};

enum RtOp { kRtRoute, kRtBalance, kRtBackward };
int launch_router_bf16(RtOp op, const RtParams& q, int sms, cudaStream_t stream);
int launch_router_fp16(RtOp op, const RtParams& q, int sms, cudaStream_t stream);
int launch_router_fp32(RtOp op, const RtParams& q, int sms, cudaStream_t stream);

}  // namespace mm
