// The norms of a transformer block fused with its gate and the residual stream, forward and backward.
//
// Per row of H channels, in 32 bits:
//   u = y,  or  y * rsqrt(mean(y^2) + eps) * (offset + w_post)          (norm after the block)
//   r' = r + scale * g * u                                              (gate: none, per channel, per token or per element)
//   h = r' * rsqrt(mean(r'^2) + eps) * (offset + w_pre)                 (norm before the next block; of r' as it is before it is rounded)
// Each output is rounded once, where it is stored.
//
// Backward, with i1, i2 the two reciprocal roots, n1 = y i1, n2 = r' i2, v = scale * g * u:
//   dr = d_r' + i2 (dh w2 - n2 mean(dh w2 n2))        dw_pre = sum over the rows of dh n2
//   dv = scale * dr,  dg = dv u (summed over what the gate is broadcast to),  du = dv g
//   dy = i1 (du w1 - n1 mean(du w1 n1)),  or du       dw_post = sum over the rows of du n1
//
// A row belongs to one CTA, which holds it in registers: eight neighbouring elements per thread and chunk.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace mm {

constexpr int kBnMaxHidden = 8192;
constexpr int kBnMaxThreads = 512;
enum BnGate { kBnGateNone = 0, kBnGateChannel = 1, kBnGateToken = 2, kBnGateElement = 3 };

struct BnParams {
    const void *residual, *y, *gate, *pre_w, *post_w;        // y, gate and either weight may be missing
    void *residual_out, *normed;
    const void *d_residual_out, *d_normed;                   // backward
    void *d_residual, *d_y, *d_gate;
    float* partial;                                          // backward: [sums][CTAs][hidden]
    long long tokens;
    long long residual_ld, y_ld, gate_ld, residual_out_ld, normed_ld, d_residual_out_ld, d_normed_ld, d_residual_ld, d_y_ld, d_gate_ld;
    int hidden, gate_mode, weight32, gate32;
    float scale, eps, offset;
};

template <typename T> __device__ __forceinline__ float bn_float(T v);
template <> __device__ __forceinline__ float bn_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float bn_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float bn_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T bn_round(float v);
template <> __device__ __forceinline__ float bn_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 bn_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half bn_round<__half>(float v) { return __float2half_rn(v); }

// Eight elements of a row as this thread sees them in chunk c. Rows that start on 16 bytes and hold a multiple of eight elements (`Vec`): eight
// neighbours, in 16 B accesses. Others: elements a CTA's width apart, one by one, so that neighbouring threads still read neighbouring elements.
template <bool Vec>
__device__ __forceinline__ int bn_at(int c, int j) {
    return Vec ? (c * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8 + j
               : (c * 8 + j) * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x);
}

template <typename T, bool Vec>
__device__ __forceinline__ void bn_load(const T* row, int hidden, int c, float (&v)[8]) {
    if constexpr (Vec) {
        const int at = bn_at<true>(c, 0);
        alignas(16) T e[8];
        if (at < hidden) {
            #pragma unroll
            for (int q = 0; q < static_cast<int>(sizeof(T)) / 2; ++q)
                reinterpret_cast<uint4*>(e)[q] = *reinterpret_cast<const uint4*>(row + at + q * (16 / static_cast<int>(sizeof(T))));
            #pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = bn_float<T>(e[j]);
        } else {
            #pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        }
    } else {
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int at = bn_at<false>(c, j);
            v[j] = at < hidden ? bn_float<T>(row[at]) : 0.f;
        }
    }
}

template <typename T, bool Vec>
__device__ __forceinline__ void bn_store(T* row, int hidden, int c, const float (&v)[8]) {
    if constexpr (Vec) {
        const int at = bn_at<true>(c, 0);
        if (at >= hidden) return;
        alignas(16) T e[8];
        #pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = bn_round<T>(v[j]);
        #pragma unroll
        for (int q = 0; q < static_cast<int>(sizeof(T)) / 2; ++q)
            *reinterpret_cast<uint4*>(row + at + q * (16 / static_cast<int>(sizeof(T)))) = reinterpret_cast<const uint4*>(e)[q];
    } else {
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int at = bn_at<false>(c, j);
            if (at < hidden) row[at] = bn_round<T>(v[j]);
        }
    }
}

// a weight or gate row that is 32 bits wide or of the activations' type
template <typename X, bool Vec>
__device__ __forceinline__ void bn_load_either(const void* row, int is32, long long at_row, int hidden, int c, float (&v)[8]) {
    if (is32) bn_load<float, Vec>(static_cast<const float*>(row) + at_row, hidden, c, v);
    else bn_load<X, Vec>(static_cast<const X*>(row) + at_row, hidden, c, v);
}

// Sums of N values over the CTA, the same in every thread: shuffles, then each warp's sums through shared memory. `part` is used by turns
// (`turn`), so that a sum needs one barrier: the next one's values go where no thread can still be reading.
template <int N>
__device__ __forceinline__ void bn_sum(float (&v)[N], float (*part)[kBnMaxThreads / 32][4], int& turn) {
    #pragma unroll
    for (int n = 0; n < N; ++n) {
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    }
    const int warps = blockDim.x >> 5;
    if (warps == 1) return;
    float (*p)[4] = part[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
        #pragma unroll
        for (int n = 0; n < N; ++n) p[threadIdx.x >> 5][n] = v[n];
    }
    __syncthreads();
    #pragma unroll
    for (int n = 0; n < N; ++n) v[n] = 0.f;
    for (int w = 0; w < warps; ++w) {
        #pragma unroll
        for (int n = 0; n < N; ++n) v[n] += p[w][n];
    }
}

// scale * gate of a chunk
template <typename X, bool Vec>
__device__ __forceinline__ void bn_gate(const BnParams& q, long long row, int c, float (&g)[8]) {
    if (q.gate_mode == kBnGateNone || q.gate_mode == kBnGateToken) {
        float s = 1.f;
        if (q.gate_mode == kBnGateToken)
            s = q.gate32 ? static_cast<const float*>(q.gate)[row * q.gate_ld] : bn_float<X>(static_cast<const X*>(q.gate)[row * q.gate_ld]);
        #pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = s;
    } else {
        bn_load_either<X, Vec>(q.gate, q.gate32, q.gate_mode == kBnGateElement ? row * q.gate_ld : 0, q.hidden, c, g);
    }
}

template <typename X, typename R, int C, bool Vec>
__global__ void __launch_bounds__(kBnMaxThreads) block_norm_kernel(const BnParams q) {
    __shared__ float part[2][kBnMaxThreads / 32][4];
    int turn = 0;
    const float inv_h = 1.f / static_cast<float>(q.hidden);
    for (long long row = blockIdx.x; row < q.tokens; row += gridDim.x) {
        float r[C][8], u[C][8];
        #pragma unroll
        for (int c = 0; c < C; ++c) bn_load<R, Vec>(static_cast<const R*>(q.residual) + row * q.residual_ld, q.hidden, c, r[c]);
        if (q.y != nullptr) {
            float sum[1] = {0.f};
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                bn_load<X, Vec>(static_cast<const X*>(q.y) + row * q.y_ld, q.hidden, c, u[c]);
                #pragma unroll
                for (int j = 0; j < 8; ++j) sum[0] += u[c][j] * u[c][j];
            }
            float i1 = 1.f;
            if (q.post_w != nullptr) {
                bn_sum<1>(sum, part, turn);
                i1 = rsqrtf(sum[0] * inv_h + q.eps);
            }
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                float g[8], w[8];
                bn_gate<X, Vec>(q, row, c, g);
                if (q.post_w != nullptr) {
                    bn_load_either<X, Vec>(q.post_w, q.weight32, 0, q.hidden, c, w);
                    #pragma unroll
                    for (int j = 0; j < 8; ++j) u[c][j] = u[c][j] * i1 * (w[j] + q.offset);
                }
                #pragma unroll
                for (int j = 0; j < 8; ++j) r[c][j] += q.scale * (u[c][j] * g[j]);
                bn_store<R, Vec>(static_cast<R*>(q.residual_out) + row * q.residual_out_ld, q.hidden, c, r[c]);
            }
        }
        if (q.pre_w != nullptr) {
            float sum[1] = {0.f};
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                #pragma unroll
                for (int j = 0; j < 8; ++j) sum[0] += r[c][j] * r[c][j];
            }
            bn_sum<1>(sum, part, turn);
            const float i2 = rsqrtf(sum[0] * inv_h + q.eps);
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                float w[8];
                bn_load_either<X, Vec>(q.pre_w, q.weight32, 0, q.hidden, c, w);
                #pragma unroll
                for (int j = 0; j < 8; ++j) r[c][j] = r[c][j] * i2 * (w[j] + q.offset);
                bn_store<X, Vec>(static_cast<X*>(q.normed) + row * q.normed_ld, q.hidden, c, r[c]);
            }
        }
    }
}

// Rows are dealt to the CTAs in turn; a thread sums the gradients of its channels' weights over the CTA's rows and leaves them in `partial`,
// which `block_norm_sums_kernel` adds up: always in the same order.
template <typename X, typename R, int C, bool Vec>
__global__ void __launch_bounds__(kBnMaxThreads) block_norm_backward_kernel(const BnParams q) {
    __shared__ float part[2][kBnMaxThreads / 32][4];
    int turn = 0;
    const float inv_h = 1.f / static_cast<float>(q.hidden);
    const bool post = q.post_w != nullptr, pre = q.pre_w != nullptr;
    float acc_pre[C][8] = {}, acc_post[C][8] = {}, acc_gate[C][8] = {};
    for (long long row = blockIdx.x; row < q.tokens; row += gridDim.x) {
        float y[C][8], i1 = 1.f;
        if (q.y != nullptr) {
            float sum[1] = {0.f};
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                bn_load<X, Vec>(static_cast<const X*>(q.y) + row * q.y_ld, q.hidden, c, y[c]);
                #pragma unroll
                for (int j = 0; j < 8; ++j) sum[0] += y[c][j] * y[c][j];
            }
            if (post) {
                bn_sum<1>(sum, part, turn);
                i1 = rsqrtf(sum[0] * inv_h + q.eps);
            }
        }
        float d[C][8];                                       // d_r', then dr
        #pragma unroll
        for (int c = 0; c < C; ++c) {
            if (q.d_residual_out != nullptr) {
                bn_load<R, Vec>(static_cast<const R*>(q.d_residual_out) + row * q.d_residual_out_ld, q.hidden, c, d[c]);
            } else {
                #pragma unroll
                for (int j = 0; j < 8; ++j) d[c][j] = 0.f;
            }
        }
        if (pre) {
            float n[C][8], dh[C][8], sum[2] = {0.f, 0.f};
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                bn_load<R, Vec>(static_cast<const R*>(q.residual) + row * q.residual_ld, q.hidden, c, n[c]);
                bn_load<X, Vec>(static_cast<const X*>(q.d_normed) + row * q.d_normed_ld, q.hidden, c, dh[c]);
                float w[8];
                if (q.y != nullptr) {
                    float g[8];
                    bn_gate<X, Vec>(q, row, c, g);
                    if (post) {
                        bn_load_either<X, Vec>(q.post_w, q.weight32, 0, q.hidden, c, w);
                        #pragma unroll
                        for (int j = 0; j < 8; ++j) n[c][j] += q.scale * (y[c][j] * i1 * (w[j] + q.offset) * g[j]);
                    } else {
                        #pragma unroll
                        for (int j = 0; j < 8; ++j) n[c][j] += q.scale * (y[c][j] * g[j]);
                    }
                }
                bn_load_either<X, Vec>(q.pre_w, q.weight32, 0, q.hidden, c, w);
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    sum[0] += n[c][j] * n[c][j];
                    sum[1] += dh[c][j] * (w[j] + q.offset) * n[c][j];
                }
            }
            bn_sum<2>(sum, part, turn);
            const float i2 = rsqrtf(sum[0] * inv_h + q.eps), mean = sum[1] * i2 * inv_h;
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                float w[8];
                bn_load_either<X, Vec>(q.pre_w, q.weight32, 0, q.hidden, c, w);
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float n2 = n[c][j] * i2;
                    acc_pre[c][j] += dh[c][j] * n2;
                    d[c][j] += i2 * (dh[c][j] * (w[j] + q.offset) - n2 * mean);
                }
            }
        }
        if (q.d_residual != nullptr) {
            #pragma unroll
            for (int c = 0; c < C; ++c) bn_store<R, Vec>(static_cast<R*>(q.d_residual) + row * q.d_residual_ld, q.hidden, c, d[c]);
        }
        if (q.y == nullptr) continue;
        float sum[2] = {0.f, 0.f};
        #pragma unroll
        for (int c = 0; c < C; ++c) {
            float g[8], w[8];
            bn_gate<X, Vec>(q, row, c, g);
            if (post) bn_load_either<X, Vec>(q.post_w, q.weight32, 0, q.hidden, c, w);
            float dg[8];
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float n1 = y[c][j] * i1, w1 = post ? w[j] + q.offset : 1.f, dv = q.scale * d[c][j];
                dg[j] = dv * (n1 * w1);
                const float du = dv * g[j];
                acc_post[c][j] += du * n1;
                d[c][j] = du * w1;
                sum[0] += d[c][j] * n1;
                sum[1] += dg[j];
            }
            if (q.gate_mode == kBnGateChannel) {
                #pragma unroll
                for (int j = 0; j < 8; ++j) acc_gate[c][j] += dg[j];
            } else if (q.gate_mode == kBnGateElement) {
                if (q.gate32) bn_store<float, Vec>(static_cast<float*>(q.d_gate) + row * q.d_gate_ld, q.hidden, c, dg);
                else bn_store<X, Vec>(static_cast<X*>(q.d_gate) + row * q.d_gate_ld, q.hidden, c, dg);
            }
        }
        if (post || q.gate_mode == kBnGateToken) bn_sum<2>(sum, part, turn);
        if (q.gate_mode == kBnGateToken && threadIdx.x == 0) {
            if (q.gate32) static_cast<float*>(q.d_gate)[row * q.d_gate_ld] = sum[1];
            else static_cast<X*>(q.d_gate)[row * q.d_gate_ld] = bn_round<X>(sum[1]);
        }
        const float mean = sum[0] * inv_h;
        #pragma unroll
        for (int c = 0; c < C; ++c) {
            if (post) {
                #pragma unroll
                for (int j = 0; j < 8; ++j) d[c][j] = i1 * (d[c][j] - y[c][j] * i1 * mean);
            }
            bn_store<X, Vec>(static_cast<X*>(q.d_y) + row * q.d_y_ld, q.hidden, c, d[c]);
        }
    }
    float* p = q.partial + static_cast<long long>(blockIdx.x) * q.hidden;
    const long long stride = static_cast<long long>(gridDim.x) * q.hidden;
    #pragma unroll
    for (int c = 0; c < C; ++c) {
        float* to = p;
        if (pre) { bn_store<float, Vec>(to, q.hidden, c, acc_pre[c]); to += stride; }
        if (post) { bn_store<float, Vec>(to, q.hidden, c, acc_post[c]); to += stride; }
        if (q.gate_mode == kBnGateChannel) bn_store<float, Vec>(to, q.hidden, c, acc_gate[c]);
    }
}

struct BnSumsParams {
    const float* partial;                                    // [sums][rows][hidden]
    void* out[3];
    int is32[3];
    int rows, hidden;
};

// Column sums: a block takes 32 channels of one of the (up to three) gradients, a warp every eighth row; added up in shared memory in order.
template <typename X>
__global__ void __launch_bounds__(256) block_norm_sums_kernel(const BnSumsParams q) {
    __shared__ float part[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.x * 32 + lane, which = blockIdx.y;
    float v = 0.f;
    if (h < q.hidden) {
        const float* p = q.partial + static_cast<long long>(which) * q.rows * q.hidden + h;
        for (int r = warp; r < q.rows; r += 8) v += p[static_cast<long long>(r) * q.hidden];
    }
    part[warp][lane] = v;
    __syncthreads();
    if (warp != 0 || h >= q.hidden) return;
    #pragma unroll
    for (int w = 1; w < 8; ++w) v += part[w][lane];
    if (q.is32[which]) static_cast<float*>(q.out[which])[h] = v;
    else static_cast<X*>(q.out[which])[h] = bn_round<X>(v);
}

}  // namespace mm
