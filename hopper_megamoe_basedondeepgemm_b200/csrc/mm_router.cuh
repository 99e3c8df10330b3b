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
// One warp holds a token's logits in registers, expert j * 32 + lane in slot j of a lane: neighbouring lanes read neighbouring experts wherever a row starts,
// and the order of slots and lanes is that of the experts. Bound by instructions more than by memory: some 300 to 400 a token against 4 bytes an
// expert.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cfloat>
#include <cstdint>

#include "../../include/megamoe_b200.h"
#include "mm_error.h"
#include "mm_router.h"

namespace mm {

// Sums of probabilities over tokens are kept as multiples of 2^-36 in 64 bits: additions of whole numbers, whose order changes nothing. 2^27 tokens fit.
constexpr float kRtFixed = 68719476736.0f;
constexpr int kRtFlushRows = 64;             // rows that a warp sums in 32 bits before they go into the 64-bit sum

template <typename L> __device__ __forceinline__ float rt_float(L v);
template <> __device__ __forceinline__ float rt_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float rt_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float rt_float<__half>(__half v) { return __half2float(v); }
template <typename L> __device__ __forceinline__ L rt_round(float v);
template <> __device__ __forceinline__ float rt_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 rt_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half rt_round<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float rt_off() { return -__int_as_float(0x7f800000); }

// a logit as it counts: NaN is an expert that is off (the maximum with a number is that number), +inf the largest number
__device__ __forceinline__ float rt_logit(float v) { return fminf(fmaxf(v, rt_off()), FLT_MAX); }

// numbers as whole numbers of the same order; 0 is below all of them
__device__ __forceinline__ uint32_t rt_order(float v) {
    const uint32_t b = __float_as_uint(v);
    return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float rt_unorder(uint32_t o) { return __uint_as_float(o ^ (o >> 31 ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ float rt_max(float v) { return rt_unorder(__reduce_max_sync(0xffffffffu, rt_order(v))); }
__device__ __forceinline__ float rt_sum(float v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// sigmoid(v), and 1 - sigmoid(v) without the difference of near numbers
__device__ __forceinline__ float rt_sigmoid(float v) { return __fdividef(1.f, 1.f + expf(-v)); }       // (exp(-v) above 2^126 gives 0)
__device__ __forceinline__ float rt_sigmoid_rest(float v) { return __fdividef(1.f, 1.f + expf(v)); }

template <typename L, int V>
__device__ __forceinline__ void rt_load(const RtParams& q, int row, int lane, float (&l)[V]) {
    const L* p = static_cast<const L*>(q.logits) + static_cast<long long>(row) * q.logits_ld + lane;
    #pragma unroll
    for (int j = 0; j < V; ++j) l[j] = j * 32 + lane < q.E ? rt_float<L>(p[j * 32]) : rt_off();
    #pragma unroll
    for (int j = 0; j < V; ++j) l[j] = rt_logit(l[j]);
}

// The sequence of a token that lies at or behind cu[0]: S if it is behind the last one. Reads cu alone, whatever it holds, and where the result is below S,
// cu[result + 1] is above the token.
__device__ __forceinline__ int rt_sequence(const int* cu, int S, int row) {
    int lo = 0, hi = S;                      // the number of ends that are <= row
    while (lo < hi) {
        const int m = (lo + hi) >> 1;
        if (cu[m + 1] <= row) lo = m + 1; else hi = m;
    }
    return lo;
}

// ----------------------------------------------------------------------------- route
// A row whose candidates do not fit a warp (many equal keys): the largest key, one after the other, over all experts.
template <typename L, int Mode>
__device__ __noinline__ void rt_route_any(const RtParams& q, int row, int* at_out, float* logit_out) {
    const int lane = threadIdx.x & 31;
    const L* p = static_cast<const L*>(q.logits) + static_cast<long long>(row) * q.logits_ld;
    double last = 0.0;
    int last_at = -1, mine = -1;
    float mine_logit = 0.f;
    for (int k = 0; k < q.K; ++k) {
        double best = static_cast<double>(rt_off());
        int at = q.E;
        for (int e = lane; e < q.E; e += 32) {
            const float v = rt_logit(rt_float<L>(p[e]));
            if (v == rt_off()) continue;
            double key = static_cast<double>(v);
            if (Mode == 1) key = 1.0 / (1.0 + exp(-key)) + (q.bias != nullptr ? static_cast<double>(q.bias[e]) : 0.0);
            if (k > 0 && !(key < last || (key == last && e > last_at))) continue;                // taken already
            if (key > best) { best = key; at = e; }
        }
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double other = __shfl_xor_sync(0xffffffffu, best, o);
            const int other_at = __shfl_xor_sync(0xffffffffu, at, o);
            if (other_at < q.E && (at >= q.E || other > best || (other == best && other_at < at))) { best = other; at = other_at; }
        }
        if (at >= q.E) break;
        last = best;
        last_at = at;
        if (lane == k) { mine = at; mine_logit = rt_logit(rt_float<L>(p[at])); }
    }
    *at_out = mine;
    *logit_out = mine_logit;
}

// Twice what a 32-bit key of mode 1 can be off by: 2^-20 for the exponential, the sum and the quotient of a sigmoid, 2^-22 of the key for its last addition.
__device__ __forceinline__ float rt_key_margin(float key) { return 0x1p-19f + fabsf(key) * 0x1p-21f; }

// The K-th largest of the lanes' own maxima is a bound: no key below it is among the K largest. What is not below it, K experts and a few, moves to one per
// lane, and the largest of those are taken by turns. In mode 1 keys are first computed in 32 bits; where two that matter come closer than their
// error, they are computed in 64.
template <typename L, int V, int Mode>
__global__ void __launch_bounds__(kRtWarps * 32) route_kernel(const RtParams q) {
    __shared__ float cand_logit[kRtWarps][32];
    __shared__ int cand_at[kRtWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t below = (1u << lane) - 1u;
    for (int row = blockIdx.x * kRtWarps + warp; row < q.T; row += gridDim.x * kRtWarps) {
        int rank = -1, at = -1;                                          // of the expert that this lane has taken
        float logit = 0.f, top = 0.f;
        int taken = 0;
        if (q.valid == nullptr || q.valid[row] != 0) {
            float l[V];
            uint32_t key[V], best = 0u;
            rt_load<L, V>(q, row, lane, l);
            #pragma unroll
            for (int j = 0; j < V; ++j) {
                float k = l[j];
                if (Mode == 1) {
                    const float b = q.bias != nullptr && j * 32 + lane < q.E ? __ldg(q.bias + j * 32 + lane) : 0.f;
                    k = k == rt_off() ? k : __fdividef(1.f, 1.f + __expf(-k)) + b;
                }
                key[j] = k > rt_off() ? rt_order(k) : 0u;
                best = max(best, key[j]);
            }
            uint32_t bound = 0u, mine = best;
            for (int n = 0; n < q.K;) {
                bound = __reduce_max_sync(0xffffffffu, mine);
                if (bound == 0u) break;
                const bool is = mine == bound;
                n += __popc(__ballot_sync(0xffffffffu, is));
                if (is) mine = 0u;
            }
            if (Mode == 1 && bound != 0u) bound = rt_order(rt_unorder(bound) - rt_key_margin(rt_unorder(bound)));
            if (bound == 0u) bound = 1u;
            int n = 0;
            #pragma unroll
            for (int j = 0; j < V; ++j) {
                const bool is = key[j] >= bound;
                const uint32_t who = __ballot_sync(0xffffffffu, is);
                if (who != 0u) {
                    const int to = n + __popc(who & below);
                    if (is && to < 32) { cand_logit[warp][to] = l[j]; cand_at[warp][to] = j * 32 + lane; }
                    n += __popc(who);
                }
            }
            __syncwarp();
            if (n > 32) {
                rt_route_any<L, Mode>(q, row, &at, &logit);
                rank = at >= 0 ? lane : -1;
                top = rt_max(rank >= 0 ? logit : rt_off());
                taken = __popc(__ballot_sync(0xffffffffu, rank >= 0));
            } else {
                uint32_t hi = 0u, lo = 0u;                               // this lane's candidate, as a key of 32 bits or 64
                float k32 = 0.f;
                if (lane < n) {
                    logit = cand_logit[warp][lane];
                    at = cand_at[warp][lane];
                    k32 = logit;
                    if (Mode == 1) k32 = __fdividef(1.f, 1.f + __expf(-logit)) + (q.bias != nullptr ? __ldg(q.bias + at) : 0.f);
                    hi = rt_order(k32);
                }
                __syncwarp();
                bool close = false;
                if (Mode == 1) {
                    // two of them nearer than the error, or equal?
                    uint32_t left = hi;
                    float last = 0.f;
                    for (int k = 0; k <= q.K && k < n; ++k) {
                        const uint32_t m = __reduce_max_sync(0xffffffffu, left);
                        const float f = rt_unorder(m);
                        const uint32_t who = __ballot_sync(0xffffffffu, left == m);
                        close = close || (k > 0 && last - f <= rt_key_margin(last)) || (who & (who - 1u)) != 0u;
                        last = f;
                        if (left == m) left = 0u;
                    }
                    if (close) {
                        unsigned long long b = 0ull;
                        if (lane < n) {
                            const double key64 = 1.0 / (1.0 + exp(-static_cast<double>(logit))) + (q.bias != nullptr ? static_cast<double>(__ldg(q.bias + at)) : 0.0);
                            b = static_cast<unsigned long long>(__double_as_longlong(key64 == 0.0 ? 0.0 : key64));
                            b ^= static_cast<unsigned long long>(static_cast<long long>(b) >> 63) | 0x8000000000000000ull;
                        }
                        hi = static_cast<uint32_t>(b >> 32);
                        lo = static_cast<uint32_t>(b);
                    }
                }
                const int want = min(q.K, n);
                for (int k = 0; k < want; ++k) {
                    const uint32_t m = __reduce_max_sync(0xffffffffu, hi);
                    bool is = hi == m && m != 0u;
                    if (Mode == 1 && close) {
                        const uint32_t m_lo = __reduce_max_sync(0xffffffffu, is ? lo : 0u);
                        is = is && lo == m_lo;
                    }
                    // (candidates lie in the experts' order: of equal ones the first lane's is the lowest)
                    const uint32_t who = __ballot_sync(0xffffffffu, is);
                    if (is && (who & below) == 0u) { rank = k; hi = lo = 0u; }
                }
                taken = want;
                if (Mode == 0) top = rt_max(rank >= 0 ? logit : rt_off());
            }
        }
        float s = 0.f;
        if (rank >= 0) s = Mode == 1 ? rt_sigmoid(logit) : expf(logit - top);
        const float total = rt_sum(s);
        const long long to = static_cast<long long>(row) * q.K;
        if (rank >= 0) {
            q.idx[to + rank] = at;
            q.weights[to + rank] = total > 0.f ? s / total * q.route_scale : 0.f;
        }
        if (lane >= taken && lane < q.K) {
            q.idx[to + lane] = -1;
            q.weights[to + lane] = 0.f;
        }
    }
}

// ----------------------------------------------------------------------------- balance
// A token's probabilities p; its softmax and the logarithm of its sum of exponentials; mode 1: its sigmoids' complements.
template <int V, int Mode, bool Rest>
__device__ __forceinline__ float rt_probabilities(const float (&l)[V], float (&p)[V], float (&soft)[V], float (&rest)[V]) {
    float top = l[0];
    #pragma unroll
    for (int j = 1; j < V; ++j) top = fmaxf(top, l[j]);
    top = rt_max(top);
    if (top == rt_off()) {
        #pragma unroll
        for (int j = 0; j < V; ++j) p[j] = soft[j] = rest[j] = 0.f;
        return 0.f;
    }
    float sum = 0.f, sig_sum = 0.f, lse = top;
    if (Mode == 1 && top <= 60.f) {
        // exp(l) by itself does not overflow (nor does the sum): it gives the softmax and the sigmoid
        #pragma unroll
        for (int j = 0; j < V; ++j) {
            soft[j] = expf(l[j]);
            rest[j] = __fdividef(1.f, 1.f + soft[j]);
            p[j] = soft[j] * rest[j];
            sum += soft[j];
            sig_sum += p[j];
        }
        if (top >= -40.f) {                                              // (nor do the largest of them get lost)
            lse = 0.f;
        } else {
            sum = 0.f;
            #pragma unroll
            for (int j = 0; j < V; ++j) { soft[j] = expf(l[j] - top); sum += soft[j]; }
        }
    } else {
        #pragma unroll
        for (int j = 0; j < V; ++j) {
            soft[j] = expf(l[j] - top);
            sum += soft[j];
            if (Mode == 1) {
                p[j] = rt_sigmoid(l[j]);
                if (Rest) rest[j] = rt_sigmoid_rest(l[j]);
                sig_sum += p[j];
            }
        }
    }
    sum = rt_sum(sum);
    const float inv = 1.f / sum;
    float sig_inv = 0.f;
    if (Mode == 1) {
        sig_sum = rt_sum(sig_sum);
        sig_inv = sig_sum > 0.f ? 1.f / sig_sum : 0.f;
    }
    #pragma unroll
    for (int j = 0; j < V; ++j) {
        soft[j] *= inv;
        p[j] = Mode == 1 ? p[j] * sig_inv : soft[j];
    }
    return lse + logf(sum);
}

// Over the CTA, in a fixed order; the result is every thread's.
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

// Counts, mean probabilities and losses from the sums, by one CTA.
__device__ __forceinline__ void rt_balance_end(const RtParams& q, int z_parts, double* part) {
    double live = 0.0, all = 0.0, z = 0.0, balance = 0.0;
    for (int s = threadIdx.x; s < q.S; s += blockDim.x) {
        const int n = __ldcg(q.sum_tokens + s);
        q.tokens[s] = n;
        live += n > 0;
        all += n;
    }
    for (int i = threadIdx.x; i < z_parts; i += blockDim.x) z += __ldcg(q.z_part + i);
    for (int s = 0, e = threadIdx.x; ; e += blockDim.x) {
        while (e >= q.E) { e -= q.E; ++s; }
        if (s >= q.S) break;
        const long long i = static_cast<long long>(s) * q.E + e;
        const int n = __ldcg(q.sum_tokens + s), c = __ldcg(q.sum_counts + i);
        const double mean = n > 0 ? static_cast<double>(__ldcg(q.sums + i)) / static_cast<double>(kRtFixed) / n : 0.0;
        q.mean[i] = static_cast<float>(mean);
        q.counts[i] = c;
        if (n > 0) balance += static_cast<double>(c) * q.E / (static_cast<double>(q.K) * n) * mean;
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

// A CTA takes consecutive tokens, piece by piece of one sequence each: its warps add the probabilities up in registers, the CTA adds the warps' sums and puts them to the
// sequence's. The last CTA to end turns the sums into the results where they are few.
template <typename L, int V, int Mode>
__global__ void __launch_bounds__(kRtWarps * 32) balance_kernel(const RtParams q) {
    __shared__ float warp_sum[kRtWarps][V * 32];
    __shared__ int hist[V * 32], warp_tokens[kRtWarps];
    __shared__ double part[kRtWarps];
    __shared__ bool last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lo = static_cast<int>(static_cast<long long>(q.T) * blockIdx.x / gridDim.x), hi = static_cast<int>(static_cast<long long>(q.T) * (blockIdx.x + 1) / gridDim.x);
    for (int e = threadIdx.x; e < V * 32; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    double z = 0.0;
    int row = lo;
    while (row < hi) {
        int s = 0, end = hi;
        if (q.cu != nullptr) {
            const int first = q.cu[0];
            if (row < first) { row = min(first, hi); continue; }
            s = rt_sequence(q.cu, q.S, row);
            if (s >= q.S) break;
            end = min(hi, q.cu[s + 1]);
        }
        end = min(end, row + kRtFlushRows * kRtWarps);
        float acc[V] = {};
        int n = 0;
        for (int r = row + warp; r < end; r += kRtWarps) {
            const long long e = lane < q.K ? q.idx[static_cast<long long>(r) * q.K + lane] : -1;
            const bool slot = e >= 0 && e < q.E;
            float l[V], p[V], soft[V], rest[V];
            rt_load<L, V>(q, r, lane, l);
            if (__ballot_sync(0xffffffffu, slot) == 0u) continue;
            if (slot) atomicAdd(hist + e, 1);
            const float lse = rt_probabilities<V, Mode, false>(l, p, soft, rest);
            #pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += p[j];
            z += static_cast<double>(lse) * static_cast<double>(lse);
            ++n;
        }
        #pragma unroll
        for (int j = 0; j < V; ++j) warp_sum[warp][j * 32 + lane] = acc[j];
        if (lane == 0) warp_tokens[warp] = n;
        __syncthreads();
        for (int e = threadIdx.x; e < q.E; e += blockDim.x) {
            unsigned long long sum = 0ull;
            #pragma unroll
            for (int w = 0; w < kRtWarps; ++w) sum += __float2ull_rn(warp_sum[w][e] * kRtFixed);
            const long long to = static_cast<long long>(s) * q.E + e;
            if (sum != 0ull) atomicAdd(q.sums + to, sum);
            if (hist[e] != 0) { atomicAdd(q.sum_counts + to, hist[e]); hist[e] = 0; }
        }
        if (threadIdx.x == 0) {
            int all = 0;
            #pragma unroll
            for (int w = 0; w < kRtWarps; ++w) all += warp_tokens[w];
            if (all > 0) atomicAdd(q.sum_tokens + s, all);
        }
        __syncthreads();
        row = end;
    }
    z = rt_block_sum(lane == 0 ? z : 0.0, part);
    if (threadIdx.x == 0) {
        q.z_part[blockIdx.x] = z;
        last = false;
    }
    if (static_cast<long long>(q.S) * q.E > kRtEndCells) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(q.ticket, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    rt_balance_end(q, gridDim.x, part);
}

template <typename L>
__global__ void __launch_bounds__(1024) balance_end_kernel(const RtParams q, int z_parts) {
    __shared__ double part[32];
    rt_balance_end(q, z_parts, part);
}

// ----------------------------------------------------------------------------- gradient
// Consecutive tokens to a warp: the factors of a sequence's experts stay in registers. The routes' gradients, one per lane, get to their experts' lanes through a row in
// shared memory that is zero between the tokens.
template <typename L, int V, int Mode>
__global__ void __launch_bounds__(kRtWarps * 32) router_backward_kernel(const RtParams q) {
    __shared__ float rows[kRtWarps][V * 32];
    __shared__ int part_live[kRtWarps];
    __shared__ long long part_all[kRtWarps];
    const int lane = threadIdx.x & 31, warp_in = threadIdx.x >> 5;
    float* buf = rows[warp_in];
    float live = 1.f, all = 1.f;
    #pragma unroll
    for (int j = 0; j < V; ++j) buf[j * 32 + lane] = 0.f;
    __syncwarp();
    if (q.balance) {
        // sequences that have tokens, and their tokens: whole numbers
        int a = 0;
        long long b = 0;
        if (q.S == 1) {
            b = q.tokens[0];
            a = b > 0;
        } else {
            for (int s = threadIdx.x; s < q.S; s += blockDim.x) { a += q.tokens[s] > 0; b += q.tokens[s]; }
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
            if (lane == 0) { part_live[warp_in] = a; part_all[warp_in] = b; }
            __syncthreads();
            a = 0; b = 0;
            for (int w = 0; w < kRtWarps; ++w) { a += part_live[w]; b += part_all[w]; }
        }
        live = static_cast<float>(a > 0 ? a : 1);
        all = static_cast<float>(b > 0 ? b : 1);
    }
    const float g = q.d_loss_ptr != nullptr ? *q.d_loss_ptr : q.d_loss;
    const int warp = blockIdx.x * kRtWarps + warp_in, warps = gridDim.x * kRtWarps;
    const int lo = static_cast<int>(static_cast<long long>(q.T) * warp / warps), hi = static_cast<int>(static_cast<long long>(q.T) * (warp + 1) / warps);
    const float zc = 2.f * q.z_coef * g / all;
    int seq = -1, seq_end = -1;
    float c[V];
    for (int row = lo; row < hi; ++row) {
        float l[V], d[V];
        const long long e64 = lane < q.K ? q.idx[static_cast<long long>(row) * q.K + lane] : -1;
        const float dw_in = q.d_weights != nullptr && lane < q.K ? q.d_weights[static_cast<long long>(row) * q.K + lane] : 0.f;
        rt_load<L, V>(q, row, lane, l);
        const int e = e64 >= 0 && e64 < q.E ? static_cast<int>(e64) : -1;
        const bool routed = __ballot_sync(0xffffffffu, e >= 0) != 0u;
        #pragma unroll
        for (int j = 0; j < V; ++j) d[j] = 0.f;
        if (q.balance && routed) {
            if (row >= seq_end || seq < 0) {
                int s = 0;
                seq_end = q.T;
                if (q.cu != nullptr) {
                    s = row < q.cu[0] ? q.S : rt_sequence(q.cu, q.S, row);
                    seq_end = s < q.S ? q.cu[s + 1] : row + 1;
                }
                seq = s;
                const float n = s < q.S ? static_cast<float>(q.tokens[s]) : 0.f;
                const float f = n > 0.f ? q.balance_coef * g * static_cast<float>(q.E) / (static_cast<float>(q.K) * n * n * live) : 0.f;
                #pragma unroll
                for (int j = 0; j < V; ++j)
                    c[j] = s < q.S && j * 32 + lane < q.E ? f * static_cast<float>(q.counts[static_cast<long long>(s) * q.E + j * 32 + lane]) : 0.f;
            }
            if (seq < q.S) {
                float p[V], soft[V], rest[V];
                const float lse = rt_probabilities<V, Mode, true>(l, p, soft, rest);
                float inner = 0.f;
                #pragma unroll
                for (int j = 0; j < V; ++j) inner += c[j] * p[j];
                inner = rt_sum(inner);
                const float zl = zc * lse;
                #pragma unroll
                for (int j = 0; j < V; ++j) {
                    d[j] = p[j] * (c[j] - inner);
                    if (Mode == 1) d[j] *= rest[j];
                    d[j] += zl * soft[j];
                }
            }
        }
        if (q.d_weights != nullptr && routed) {
            const float dw = e >= 0 ? dw_in * q.route_scale : 0.f;
            const float mine = e >= 0 ? rt_logit(rt_float<L>(static_cast<const L*>(q.logits)[static_cast<long long>(row) * q.logits_ld + e])) : rt_off();
            float w = 0.f, rest = 1.f;
            if (Mode == 1) {
                if (mine > rt_off()) { w = rt_sigmoid(mine); rest = rt_sigmoid_rest(mine); }
            } else {
                const float top = rt_max(mine);
                if (mine > rt_off()) w = expf(mine - top);
            }
            const float total = rt_sum(w);
            w = total > 0.f ? w / total : 0.f;
            const float inner = rt_sum(w * dw);
            const float dk = w * (dw - inner) * rest;
            // an expert that the token names twice shows by the lane that another one's number has taken the place of
            if (e >= 0) buf[e] = __int_as_float(lane);
            __syncwarp();
            const bool twice = __ballot_sync(0xffffffffu, e >= 0 && __float_as_int(buf[e >= 0 ? e : 0]) != lane) != 0u;
            __syncwarp();
            if (!twice) {
                if (e >= 0) buf[e] = dk;
            } else {
                if (e >= 0) buf[e] = 0.f;
                __syncwarp();
                for (int k = 0; k < q.K; ++k) {
                    if (lane == k && e >= 0) buf[e] += dk;
                    __syncwarp();
                }
            }
            __syncwarp();
            #pragma unroll
            for (int j = 0; j < V; ++j) d[j] += buf[j * 32 + lane];
            __syncwarp();
            if (e >= 0) buf[e] = 0.f;
            __syncwarp();
        }
        L* to = static_cast<L*>(q.d_logits) + static_cast<long long>(row) * q.d_logits_ld + lane;
        #pragma unroll
        for (int j = 0; j < V; ++j)
            if (j * 32 + lane < q.E) to[j * 32] = rt_round<L>(d[j]);
    }
}

// ----------------------------------------------------------------------------- launches
template <typename L, int V, int Mode>
int rt_launch_kernel(RtOp op, const RtParams& q, int sms, cudaStream_t stream) {
    const int blocks = (q.T + kRtWarps - 1) / kRtWarps;
    if (op == kRtBalance) {
        // (tokens to spare for each warp's sums: four of them)
        const int want = (blocks + 3) / 4, grid = want < 1 ? 1 : (want < kRtBalanceCtas ? want : kRtBalanceCtas);
        balance_kernel<L, V, Mode><<<grid, kRtWarps * 32, 0, stream>>>(q);
        MM_CUDA(cudaGetLastError());
        if (static_cast<long long>(q.S) * q.E > kRtEndCells) balance_end_kernel<L><<<1, 1024, 0, stream>>>(q, grid);
    } else {
        const int grid = blocks < sms * 8 ? blocks : sms * 8;
        if (op == kRtRoute) route_kernel<L, V, Mode><<<grid, kRtWarps * 32, 0, stream>>>(q);
        else router_backward_kernel<L, V, Mode><<<grid, kRtWarps * 32, 0, stream>>>(q);
    }
    MM_CUDA(cudaGetLastError());
    return MM_OK;
}

template <typename L, int V>
int rt_launch_mode(RtOp op, const RtParams& q, int sms, cudaStream_t stream) {
    return q.mode == 1 ? rt_launch_kernel<L, V, 1>(op, q, sms, stream) : rt_launch_kernel<L, V, 0>(op, q, sms, stream);
}

template <typename L>
int rt_launch(RtOp op, const RtParams& q, int sms, cudaStream_t stream) {
    const int v = (q.E + 31) / 32;
    if (v <= 1) return rt_launch_mode<L, 1>(op, q, sms, stream);
    if (v <= 2) return rt_launch_mode<L, 2>(op, q, sms, stream);
    if (v <= 4) return rt_launch_mode<L, 4>(op, q, sms, stream);
    if (v <= 8) return rt_launch_mode<L, 8>(op, q, sms, stream);
    if (v <= 12) return rt_launch_mode<L, 12>(op, q, sms, stream);
    if (v <= 16) return rt_launch_mode<L, 16>(op, q, sms, stream);
    return rt_launch_mode<L, 32>(op, q, sms, stream);
}

}  // namespace mm
