// The norms of a transformer block: launch parameters, and the entry points of the source files that hold the kernels of one activation type each.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace mm {

constexpr int kBnMaxHidden = 8192;
constexpr int kBnMaxThreads = 512;
constexpr int kBnPairThreads = 384;
constexpr int kBnOneHidden = 8 * kBnMaxThreads;              // channels that one CTA holds of a row; wider rows belong to two
enum BnGate { kBnGateNone = 0, kBnGateChannel = 1, kBnGateToken = 2, kBnGateElement = 3 };

struct BnParams {
    const void *residual, *y, *gate, *pre_w, *post_w;        // y, gate and either weight may be missing
    void *residual_out, *normed;
    const void *d_residual_out, *d_normed;                   // backward
    void *d_residual, *d_y, *d_gate;
    float* partial;                                          // backward: [sums][CTAs][hidden], sums: of dh n2 (if there is a w_pre), of dr n1 gate (if anything asks for it)
    long long tokens;
    long long residual_ld, y_ld, gate_ld, residual_out_ld, normed_ld, d_residual_out_ld, d_normed_ld, d_residual_ld, d_y_ld, d_gate_ld;
    int hidden, gate_mode, weight32, gate32;
    float scale, eps, offset;
};

struct BnSumsParams {
    const float* partial;                                    // [sums][rows][hidden]
    const void *gate, *post_w;                               // channel gate and w_post, where there are any
    void *d_pre_w, *d_post_w, *d_gate;
    int rows, hidden, weight32, gate32, sums;
    float scale, offset;
};

// `aligned`: rows start on 16 bytes (32-bit ones on 32) and are made of whole groups of eight channels. `teams`: of a backward pass, with its partial sums.
struct BnLaunch {
    bool backward, stream32, aligned;
    int sms, teams;
};
int launch_block_norm_bf16(const BnParams& q, const BnLaunch& how, cudaStream_t stream);
int launch_block_norm_wide_bf16(const BnParams& q, const BnLaunch& how, cudaStream_t stream);
int launch_block_norm_fp16(const BnParams& q, const BnLaunch& how, cudaStream_t stream);
int launch_block_norm_wide_fp16(const BnParams& q, const BnLaunch& how, cudaStream_t stream);
int launch_block_norm_fp32(const BnParams& q, const BnLaunch& how, cudaStream_t stream);
int launch_block_norm_wide_fp32(const BnParams& q, const BnLaunch& how, cudaStream_t stream);
int launch_block_norm_sums_bf16(const BnSumsParams& q, cudaStream_t stream);
int launch_block_norm_sums_fp16(const BnSumsParams& q, cudaStream_t stream);
int launch_block_norm_sums_fp32(const BnSumsParams& q, cudaStream_t stream);

// Threads of a CTA, and teams (CTAs, or pairs of them) of a backward pass: each leaves a row of partial sums, so the workspace goes by them, and as many as a B200 with its
// 148 SMs holds at a time (128 registers a thread) leave it.
inline int bn_threads(int hidden) {
    const int per = hidden <= kBnOneHidden ? 8 : 16;
    return ((hidden + per - 1) / per + 31) / 32 * 32;
}
inline long long bn_backward_teams(long long tokens, int hidden) {
    const int fit = 512 / bn_threads(hidden);
    const long long most = hidden > kBnOneHidden ? 74 : 148ll * (fit < 1 ? 1 : (fit > 8 ? 8 : fit));
    return tokens < most ? tokens : most;
}

}  // namespace mm
