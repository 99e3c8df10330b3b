// Routing from logits, the balance loss over the experts, and the gradient of both.
//
// A token's scores over E experts: softmax (mode 0) or sigmoid (mode 1) of its logits. An expert whose logit is -inf or NaN is off for that token;
// +inf counts as the largest finite number.
//
//   route:    the K largest keys (mode 0 the logits, mode 1 sigmoid + bias), ties to the lower expert; weights: scores over the sum of the selected
//             scores, times a scale. Keys of mode 1 are compared in 64 bits: in 32, two experts that differ could tie, or change places.
//   balance:  per sequence of n routed tokens, with c_e the slots routed to expert e and P_e the mean of p_e = score_e / sum of the token's scores:
//             L = sum over e of (E c_e / (K n)) P_e; the loss is the mean of L over the sequences that have tokens, plus the mean square of the
//             logarithm of the sum of exponentials of a token's logits, each times its coefficient.
//   gradient: with q_e = dL/dp_e:  mode 0  p_e (q_e - sum of q p),  mode 1  (1 - s_e) p_e (q_e - sum of q p);  of the routing weights w_k the same
//             over the selected slots; of the square 2 lse softmax_e.
//
// One warp holds a token's logits in registers, expert j * 32 + lane in slot j of a lane.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cfloat>
#include <cstdint>

namespace mm {

constexpr int kRtMaxExperts = 1024, kRtMaxTopk = 32, kRtWarps = 8;
// Sums of probabilities over tokens are kept as multiples of 2^-36 in 64 bits: additions of whole numbers, whose order changes nothing. 2^27 tokens fit.
constexpr double kRtFixed = 68719476736.0;
constexpr int kRtFlushRows = 64;             // rows that a warp sums in 32 bits before they go into the 64-bit sum

struct RtParams {
    const void* logits;
    long long logits_ld;
    const float* bias;
    const uint8_t* valid;
    long long* idx;                          // [T][K]
    float* weights;                          // [T][K]
    const int* cu;                           // [S + 1], or nullptr: one sequence of all tokens
    int T, E, K, S, mode;
    float route_scale, balance_coef, z_coef, d_loss;
    const float* d_loss_ptr;                 // device scalar, or nullptr: d_loss
    const float* d_weights;                  // [T][K] or nullptr
    int* counts;                             // [S][E]
    int* tokens;                             // [S]
    float* mean;                             // [S][E]
    float* losses;                           // loss, balance, z
    unsigned long long* sums;                // [S][E]
    double* z_part;                          // one per warp of the grid
    int z_parts, balance;
    void* d_logits;
    long long d_logits_ld;
};

template <typename L> __device__ __forceinline__ float rt_float(L v);
template <> __device__ __forceinline__ float rt_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float rt_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float rt_float<__half>(__half v) { return __half2float(v); }
template <typename L> __device__ __forceinline__ L rt_round(float v);
template <> __device__ __forceinline__ float rt_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 rt_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half rt_round<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float rt_off() { return -__int_as_float(0x7f800000); }

// a logit as it counts: NaN is an expert that is off, +inf the largest number
__device__ __forceinline__ float rt_logit(float v) { return v > -FLT_MAX ? fminf(v, FLT_MAX) : (v == -FLT_MAX ? v : rt_off()); }

__device__ __forceinline__ float rt_max(float v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float rt_sum(float v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename L, int V>
__device__ __forceinline__ void rt_load(const RtParams& q, int row, uint32_t lane, float (&l)[V]) {
    const L* p = static_cast<const L*>(q.logits) + static_cast<long long>(row) * q.logits_ld;
    #pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = j * 32 + static_cast<int>(lane);
        l[j] = e < q.E ? rt_logit(rt_float<L>(p[e])) : rt_off();
    }
}

// The sequence of a token, S if it is in none. Reads cu alone, whatever it holds.
__device__ __forceinline__ int rt_sequence(const RtParams& q, int row) {
    if (q.cu == nullptr) return 0;
    if (row < q.cu[0]) return q.S;
    int lo = 0, hi = q.S;                    // the number of ends that are <= row
    while (lo < hi) {
        const int m = (lo + hi) >> 1;
        if (q.cu[m + 1] <= row) lo = m + 1; else hi = m;
    }
    return lo;
}

template <typename L, int V>
__global__ void __launch_bounds__(kRtWarps * 32) route_kernel(const RtParams q) {
    const uint32_t lane = threadIdx.x & 31u;
    for (int row = blockIdx.x * kRtWarps + (threadIdx.x >> 5); row < q.T; row += gridDim.x * kRtWarps) {
        long long my_idx = -1;
        float my_score = 0.f, l[V];
        if (q.valid == nullptr || q.valid[row] != 0) {
            rt_load<L, V>(q, row, lane, l);
            double key[V];
            #pragma unroll
            for (int j = 0; j < V; ++j) {
                key[j] = static_cast<double>(l[j]);
                if (q.mode == 1 && l[j] > rt_off())
                    key[j] = 1.0 / (1.0 + exp(-key[j])) + (q.bias != nullptr ? static_cast<double>(q.bias[j * 32 + lane]) : 0.0);
            }
            for (int k = 0; k < q.K; ++k) {
                double best = static_cast<double>(rt_off());
                int at = q.E;
                #pragma unroll
                for (int j = 0; j < V; ++j)
                    if (key[j] > best) { best = key[j]; at = j * 32 + static_cast<int>(lane); }
                #pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const double other = __shfl_xor_sync(0xffffffffu, best, o);
                    const int other_at = __shfl_xor_sync(0xffffffffu, at, o);
                    if (other > best || (other == best && other_at < at)) { best = other; at = other_at; }
                }
                if (at >= q.E) break;                                   // every expert that is on has been taken
                float chosen = 0.f;
                #pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j * 32 + static_cast<int>(lane) == at) { chosen = l[j]; key[j] = static_cast<double>(rt_off()); }
                chosen = __shfl_sync(0xffffffffu, chosen, at & 31);
                if (static_cast<int>(lane) == k) { my_idx = at; my_score = chosen; }
            }
        }
        const bool live = my_idx >= 0;
        float s = 0.f;
        if (q.mode == 1) {
            if (live) s = 1.f / (1.f + expf(-my_score));
        } else {
            const float top = rt_max(live ? my_score : rt_off());
            if (live) s = expf(my_score - top);
        }
        const float total = rt_sum(s);
        if (static_cast<int>(lane) < q.K) {
            q.idx[static_cast<long long>(row) * q.K + lane] = my_idx;
            q.weights[static_cast<long long>(row) * q.K + lane] = total > 0.f ? s / total * q.route_scale : 0.f;
        }
    }
}

// A token's probabilities p, its softmax (which is p in mode 0), its sigmoids (mode 1) and the logarithm of its sum of exponentials.
template <int V>
__device__ __forceinline__ float rt_probabilities(const RtParams& q, const float (&l)[V], float (&p)[V], float (&soft)[V], float (&sig)[V]) {
    float top = rt_off();
    #pragma unroll
    for (int j = 0; j < V; ++j) top = fmaxf(top, l[j]);
    top = rt_max(top);
    if (top == rt_off()) {
        #pragma unroll
        for (int j = 0; j < V; ++j) p[j] = soft[j] = sig[j] = 0.f;
        return 0.f;
    }
    float sum = 0.f, sig_sum = 0.f;
    #pragma unroll
    for (int j = 0; j < V; ++j) {
        soft[j] = expf(l[j] - top);
        sum += soft[j];
        if (q.mode == 1) {
            sig[j] = 1.f / (1.f + expf(-l[j]));
            sig_sum += sig[j];
        }
    }
    sum = rt_sum(sum);
    const float inv = 1.f / sum;
    float sig_inv = 0.f;
    if (q.mode == 1) {
        sig_sum = rt_sum(sig_sum);
        sig_inv = sig_sum > 0.f ? 1.f / sig_sum : 0.f;
    }
    #pragma unroll
    for (int j = 0; j < V; ++j) {
        soft[j] *= inv;
        p[j] = q.mode == 1 ? sig[j] * sig_inv : soft[j];
    }
    return top + logf(sum);
}

// A warp takes consecutive tokens and adds their probabilities up in registers for as long as they are of one sequence.
template <typename L, int V>
__global__ void __launch_bounds__(kRtWarps * 32) balance_kernel(const RtParams q) {
    const uint32_t lane = threadIdx.x & 31u;
    const int warp = blockIdx.x * kRtWarps + (threadIdx.x >> 5), warps = gridDim.x * kRtWarps;
    const int lo = static_cast<int>(static_cast<long long>(q.T) * warp / warps), hi = static_cast<int>(static_cast<long long>(q.T) * (warp + 1) / warps);
    float acc[V] = {};
    double z = 0.0;
    int seq = -1, n = 0, since = 0;
    auto flush = [&]() {
        #pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = j * 32 + static_cast<int>(lane);
            if (e < q.E && acc[j] != 0.f) atomicAdd(q.sums + static_cast<long long>(seq) * q.E + e, static_cast<unsigned long long>(static_cast<double>(acc[j]) * kRtFixed + 0.5));
            acc[j] = 0.f;
        }
        if (lane == 0 && n > 0) atomicAdd(q.tokens + seq, n);
        n = since = 0;
    };
    for (int row = lo; row < hi; ++row) {
        const int s = rt_sequence(q, row);
        if (s >= q.S) continue;
        const long long e = static_cast<int>(lane) < q.K ? q.idx[static_cast<long long>(row) * q.K + lane] : -1;
        const bool slot = e >= 0 && e < q.E;
        if (__ballot_sync(0xffffffffu, slot) == 0u) continue;
        if (s != seq || since == kRtFlushRows) {
            if (seq >= 0) flush();
            seq = s;
        }
        if (slot) atomicAdd(q.counts + static_cast<long long>(seq) * q.E + e, 1);
        float l[V], p[V], soft[V], sig[V];
        rt_load<L, V>(q, row, lane, l);
        const float lse = rt_probabilities<V>(q, l, p, soft, sig);
        #pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += p[j];
        z += static_cast<double>(lse) * static_cast<double>(lse);
        ++n; ++since;
    }
    if (seq >= 0) flush();
    if (lane == 0) q.z_part[warp] = z;
}

// Over the CTA, in a fixed order; the result is thread 0's.
__device__ __forceinline__ double rt_block_sum(double v, double* part) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) v += part[w];
    return v;
}

// Mean probabilities, and the losses from the sums.
__global__ void __launch_bounds__(1024) balance_end_kernel(const RtParams q) {
    __shared__ double part[32];
    double live = 0.0, all = 0.0, z = 0.0, balance = 0.0;
    for (int s = threadIdx.x; s < q.S; s += blockDim.x) {
        live += q.tokens[s] > 0;
        all += q.tokens[s];
    }
    for (int i = threadIdx.x; i < q.z_parts; i += blockDim.x) z += q.z_part[i];
    const long long cells = static_cast<long long>(q.S) * q.E;
    for (long long i = threadIdx.x; i < cells; i += blockDim.x) {
        const int n = q.tokens[i / q.E];
        const double mean = n > 0 ? static_cast<double>(q.sums[i]) / kRtFixed / n : 0.0;
        q.mean[i] = static_cast<float>(mean);
        if (n > 0) balance += static_cast<double>(q.counts[i]) * q.E / (static_cast<double>(q.K) * n) * mean;
    }
    live = rt_block_sum(live, part);
    all = rt_block_sum(all, part);
    z = rt_block_sum(z, part);
    balance = rt_block_sum(balance, part);
    if (threadIdx.x == 0) {
        balance = live > 0.0 ? balance / live : 0.0;
        z = all > 0.0 ? z / all : 0.0;
        q.losses[0] = static_cast<float>(q.balance_coef * balance + q.z_coef * z);
        q.losses[1] = static_cast<float>(balance);
        q.losses[2] = static_cast<float>(z);
    }
}

template <typename L, int V>
__global__ void __launch_bounds__(kRtWarps * 32) router_backward_kernel(const RtParams q) {
    __shared__ int part_live[kRtWarps], part_all_lo[kRtWarps], part_all_hi[kRtWarps];
    const uint32_t lane = threadIdx.x & 31u;
    float live = 1.f, all = 1.f;
    if (q.balance) {
        // sequences that have tokens, and their tokens: whole numbers
        int a = 0;
        long long b = 0;
        for (int s = threadIdx.x; s < q.S; s += blockDim.x) { a += q.tokens[s] > 0; b += q.tokens[s]; }
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
        if (lane == 0) { part_live[threadIdx.x >> 5] = a; part_all_lo[threadIdx.x >> 5] = static_cast<int>(b & 0x7fffffff); part_all_hi[threadIdx.x >> 5] = static_cast<int>(b >> 31); }
        __syncthreads();
        a = 0; b = 0;
        for (int w = 0; w < kRtWarps; ++w) { a += part_live[w]; b += part_all_lo[w] + (static_cast<long long>(part_all_hi[w]) << 31); }
        live = static_cast<float>(a > 0 ? a : 1);
        all = static_cast<float>(b > 0 ? b : 1);
    }
    const float g = q.d_loss_ptr != nullptr ? *q.d_loss_ptr : q.d_loss;
    const int warp = blockIdx.x * kRtWarps + (threadIdx.x >> 5), warps = gridDim.x * kRtWarps;
    const int lo = static_cast<int>(static_cast<long long>(q.T) * warp / warps), hi = static_cast<int>(static_cast<long long>(q.T) * (warp + 1) / warps);
    const float zc = 2.f * q.z_coef * g / all;
    for (int row = lo; row < hi; ++row) {
        const long long e = static_cast<int>(lane) < q.K ? q.idx[static_cast<long long>(row) * q.K + lane] : -1;
        const bool slot = e >= 0 && e < q.E;
        float l[V], d[V] = {};
        rt_load<L, V>(q, row, lane, l);
        if (__ballot_sync(0xffffffffu, slot) != 0u) {
            const int s = q.balance ? rt_sequence(q, row) : q.S;
            if (s < q.S) {
                float p[V], soft[V], sig[V], c[V];
                const float lse = rt_probabilities<V>(q, l, p, soft, sig);
                const float n = static_cast<float>(q.tokens[s]);
                const float f = n > 0.f ? q.balance_coef * g * static_cast<float>(q.E) / (static_cast<float>(q.K) * n * n * live) : 0.f;
                float inner = 0.f;
                #pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int at = j * 32 + static_cast<int>(lane);
                    c[j] = at < q.E ? f * static_cast<float>(q.counts[static_cast<long long>(s) * q.E + at]) : 0.f;
                    inner += c[j] * p[j];
                }
                inner = rt_sum(inner);
                #pragma unroll
                for (int j = 0; j < V; ++j) {
                    d[j] = p[j] * (c[j] - inner);
                    if (q.mode == 1) d[j] *= 1.f - sig[j];
                    d[j] += zc * lse * soft[j];
                }
            }
            if (q.d_weights != nullptr) {
                float dw = slot ? q.d_weights[static_cast<long long>(row) * q.K + lane] * q.route_scale : 0.f;
                // the selected logits, from the lanes that hold them
                float mine = rt_off();
                for (int k = 0; k < q.K; ++k) {
                    const int at = static_cast<int>(__shfl_sync(0xffffffffu, slot ? e : -1ll, k));
                    float v = rt_off();
                    #pragma unroll
                    for (int j = 0; j < V; ++j) if (j * 32 + static_cast<int>(lane) == at) v = l[j];
                    v = __shfl_sync(0xffffffffu, v, at & 31);
                    if (static_cast<int>(lane) == k && slot) mine = v;
                }
                float w = 0.f, rest = 1.f;
                if (q.mode == 1) {
                    if (mine > rt_off()) w = 1.f / (1.f + expf(-mine));
                    rest = 1.f - w;
                } else {
                    const float top = rt_max(mine);
                    if (mine > rt_off()) w = expf(mine - top);
                }
                const float total = rt_sum(w);
                w = total > 0.f ? w / total : 0.f;
                const float inner = rt_sum(w * dw);
                const float dk = w * (dw - inner) * rest;
                for (int k = 0; k < q.K; ++k) {
                    const int at = static_cast<int>(__shfl_sync(0xffffffffu, slot ? e : -1ll, k));
                    const float v = __shfl_sync(0xffffffffu, dk, k);
                    #pragma unroll
                    for (int j = 0; j < V; ++j) if (j * 32 + static_cast<int>(lane) == at) d[j] += v;
                }
            }
        }
        L* to = static_cast<L*>(q.d_logits) + static_cast<long long>(row) * q.d_logits_ld;
        #pragma unroll
        for (int j = 0; j < V; ++j) {
            const int at = j * 32 + static_cast<int>(lane);
            if (at < q.E) to[at] = rt_round<L>(d[j]);
        }
    }
}

}  // namespace mm
