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
// and the order of slots and lanes is that of the experts. More instructions than memory, against 4 bytes an expert: 690 a token to route one over 384 experts and 406 for
// the gradient, which bound both (64 % of the issue slots); 245 for the balance loss, which its CTAs' barriers and common sums bound (37 %).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cfloat>
#include <cstdint>

#include "../../include/megamoe_b200.h"
#include "mm_error.h"
#include "mm_launch.h"
#include "mm_ptx.cuh"
#include "mm_router.h"

namespace mm {

// Sums of probabilities over tokens are kept as whole numbers of 64 bits, whose additions' order changes nothing: multiples of `q.step`, 2^-63 of the next power of two above
// the number of tokens.
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

// The special function unit's exponential and reciprocal, results below 2^-126 as 0: good to 2^-22 and 2^-23, and an exponent of x log2(e) is off by up to
// 1.5 |x| 2^-24 of its result.
__device__ __forceinline__ float rt_exp2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float rt_rcp(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
constexpr float kRtLog2e = 1.4426950408889634f;
__device__ __forceinline__ float rt_exp(float v) { return rt_exp2(v * kRtLog2e); }
// sigmoid(v), and 1 - sigmoid(v) without the difference of near numbers
__device__ __forceinline__ float rt_sigmoid(float v) { return rt_rcp(1.f + rt_exp(-v)); }
__device__ __forceinline__ float rt_sigmoid_rest(float v) { return rt_rcp(1.f + rt_exp(v)); }
// Scores of which only the ratio counts. Where all of a token's sigmoids are below 2^-24 each is its exponential, as far as 32 bits tell, and is taken relative to the largest one:
// from a logit of -87 on the sigmoid by itself is 0 in 32 bits. Tokens whose logits are all below kRtLowest have scores of 0 in 64 bits, too, and count as such.
constexpr float kRtLowSum = 0x1p-24f, kRtLow = -17.f, kRtLowest = -709.78f;

template <typename L, int V>
__device__ __forceinline__ void rt_fetch(const RtParams& q, int row, int lane, float (&l)[V]) {
    const L* p = static_cast<const L*>(q.logits) + static_cast<long long>(row) * q.logits_ld + lane;
    #pragma unroll
    for (int j = 0; j < V; ++j) l[j] = j * 32 + lane < q.E ? rt_float<L>(p[j * 32]) : rt_off();
}
template <int V>
__device__ __forceinline__ void rt_clean(float (&l)[V]) {
    #pragma unroll
    for (int j = 0; j < V; ++j) l[j] = rt_logit(l[j]);
}

// The first token of a share, of those that the launch deals out.
__device__ __forceinline__ int rt_share(const RtParams& q, int n) { return n * q.share + min(n, q.shares_more); }

// The sequence of a token that lies at or behind cu[0], by a whole warp: S if it is behind the last one. Each step looks at 32 ends at once. Reads cu alone, whatever
// it holds, and where the result is below S, cu[result + 1] is above the token.
__device__ __forceinline__ int rt_sequence(const int* cu, int S, int row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = S;                      // the number of ends that are <= row lies between
    while (lo < hi) {
        const int step = (hi - lo + 31) >> 5, m = lo + lane * step;
        const uint32_t above = __ballot_sync(0xffffffffu, m < hi && cu[min(m, hi - 1) + 1] > row);
        if (above == 0u) {                   // (none of those looked at: behind the last of them)
            lo = lo + (hi - lo - 1) / step * step + 1;
        } else {
            const int f = __ffs(above) - 1;
            hi = lo + f * step;
            lo = f > 0 ? lo + (f - 1) * step + 1 : hi;
        }
    }
    return hi;
}

// ----------------------------------------------------------------------------- route
// A row whose candidates do not fit a warp (many equal keys, or more routes than lanes have experts on top): the largest key, one after the other, over all experts.
// The lane's expert, -1 for none. (A call of its own, by values: a reference to the launch's parameters would have every thread copy them.)
template <typename L, int Mode>
__device__ __noinline__ int rt_route_any(const L* p, const float* bias, int experts, int topk) {
    const int lane = threadIdx.x & 31;
    double last = 0.0;
    int last_at = -1, mine = -1;
    for (int k = 0; k < topk; ++k) {
        double best = static_cast<double>(rt_off());
        int at = experts;
        for (int e = lane; e < experts; e += 32) {
            const float v = rt_logit(rt_float<L>(p[e]));
            double key = static_cast<double>(v);
            if (Mode == 1) key = 1.0 / (1.0 + exp(-key)) + (bias != nullptr ? static_cast<double>(bias[e]) : 0.0);
            const bool open = v != rt_off() && key > static_cast<double>(rt_off()) && (k == 0 || key < last || (key == last && e > last_at));           // on, and not taken already
            if (open && (at == experts || key > best)) { best = key; at = e; }
        }
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double other = __shfl_xor_sync(0xffffffffu, best, o);
            const int other_at = __shfl_xor_sync(0xffffffffu, at, o);
            if (other_at < experts && (at >= experts || other > best || (other == best && other_at < at))) { best = other; at = other_at; }
        }
        if (at >= experts) break;
        last = best;
        last_at = at;
        if (lane == k) mine = at;
    }
    return mine;
}

// Twice what a 32-bit key of mode 1 can be off by: 2^-20 for the exponential, the sum and the quotient of a sigmoid, 2^-22 of the key for its last addition.
__device__ __forceinline__ float rt_key_margin(float key) { return 0x1p-19f + fabsf(key) * 0x1p-21f; }

// The K-th largest of the lanes' own maxima is a bound: no key below it is among the K largest. What is not below it, K experts and a few, moves to one per
// lane, in the experts' order, and a candidate's place is the number of those before it. In mode 1 keys are first computed in 32 bits; where two
// candidates come closer than their error, all of them are computed in 64.
template <typename L, int V, int Mode>
__global__ void __launch_bounds__(kRtWarps * 32) route_kernel(const RtParams q) {
    __shared__ float cand_logit[kRtWarps][32];
    __shared__ __align__(16) float cand_key[kRtWarps][32];
    __shared__ int cand_at[kRtWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t below = (1u << lane) - 1u;
    grid_dependency_wait();
    grid_launch_dependents();
    for (int row = blockIdx.x * kRtWarps + warp; row < q.T; row += gridDim.x * kRtWarps) {
        int rank = q.K, at = -1, taken = 0;                              // this lane's expert and its place
        float logit = rt_off();
        if (q.valid == nullptr || q.valid[row] != 0) {
            float l[V], key[V];
            rt_fetch<L, V>(q, row, lane, l);
            if (Mode == 1) {
                #pragma unroll
                for (int j = 0; j < V; ++j) key[j] = q.bias != nullptr && j * 32 + lane < q.E ? __ldg(q.bias + j * 32 + lane) : 0.f;
            }
            float best = rt_off();                                       // (NaN is no maximum, and not below: not a candidate)
            #pragma unroll
            for (int j = 0; j < V; ++j) {
                key[j] = Mode == 1 ? (l[j] > rt_off() ? rt_sigmoid(l[j]) + key[j] : rt_off()) : l[j];
                best = fmaxf(best, key[j]);
            }
            if (Mode == 0 && rt_max(best) > FLT_MAX) {                   // infinities count as the largest number
                best = fminf(best, FLT_MAX);
                #pragma unroll
                for (int j = 0; j < V; ++j) key[j] = l[j] = rt_logit(l[j]);
            }
            // lanes of one maximum are taken at once: the bound is then lower than it has to be
            uint32_t mine = best == rt_off() ? 0u : rt_order(best), high = 0u;
            for (int k = 0; k < q.K; ++k) {
                high = __reduce_max_sync(0xffffffffu, mine);
                mine = mine == high ? 0u : mine;
            }
            float bound = -FLT_MAX;                                      // (what is on; in mode 1 with an infinite bias, too)
            if (high != 0u) {
                bound = rt_unorder(high);
                if (Mode == 1) bound = fmaxf(bound - rt_key_margin(bound), -FLT_MAX);
            }
            int n = 0;
            #pragma unroll
            for (int j = 0; j < V; ++j) {
                const bool is = key[j] >= bound;
                const uint32_t who = __ballot_sync(0xffffffffu, is);
                if (who != 0u) {
                    const int to = n + __popc(who & below);
                    if (is && to < 32) { cand_key[warp][to] = key[j]; cand_at[warp][to] = j * 32 + lane; if (Mode == 1) cand_logit[warp][to] = l[j]; }
                    n += __popc(who);
                }
            }
            if (lane >= n && lane < ((n + 3) & ~3)) cand_key[warp][lane] = rt_off();       // (goes before none)
            __syncwarp();
            if (n > 32) {
                at = rt_route_any<L, Mode>(static_cast<const L*>(q.logits) + static_cast<long long>(row) * q.logits_ld, q.bias, q.E, q.K);
                if (at >= 0) {
                    rank = lane;
                    logit = rt_logit(rt_float<L>(static_cast<const L*>(q.logits)[static_cast<long long>(row) * q.logits_ld + at]));
                }
                taken = __popc(__ballot_sync(0xffffffffu, at >= 0));
            } else {
                float mine_key = rt_off();
                if (lane < n) { mine_key = cand_key[warp][lane]; at = cand_at[warp][lane]; logit = Mode == 1 ? cand_logit[warp][lane] : mine_key; }
                int before = 0, near = 0;                                // candidates that go before this one; in mode 1 those that may or may not, itself among them
                const float margin = Mode == 1 ? rt_key_margin(mine_key) : 0.f;
                for (int c = 0; c < n; c += 4) {
                    const float4 k4 = *reinterpret_cast<const float4*>(&cand_key[warp][c]);
                    const float ks[4] = {k4.x, k4.y, k4.z, k4.w};
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        before += c + i < lane ? ks[i] >= mine_key : ks[i] > mine_key;
                        if (Mode == 1) near += !(fabsf(ks[i] - mine_key) > margin);
                    }
                }
                const bool close = near != 1;
                if (Mode == 1) {
                    if (__ballot_sync(0xffffffffu, close && lane < n) != 0u) {
                        const double key64 = lane < n ? 1.0 / (1.0 + exp(-static_cast<double>(logit))) + (q.bias != nullptr ? static_cast<double>(__ldg(q.bias + at)) : 0.0) : 0.0;
                        before = 0;
                        for (int c = 0; c < n; ++c) {
                            const double other = __shfl_sync(0xffffffffu, key64, c);
                            before += other > key64 || (other == key64 && c < lane);
                        }
                    }
                }
                __syncwarp();
                taken = min(q.K, n);
                if (lane < n && before < taken) rank = before; else logit = rt_off();
            }
        }
        const bool chosen = rank < q.K;
        float s = 0.f;
        if (Mode == 1) {
            if (chosen) s = rt_sigmoid(logit);
        } else {
            const float top = rt_max(logit);
            if (chosen) s = rt_exp(logit - top);
        }
        float total = rt_sum(s);
        if (Mode == 1 && total < kRtLowSum) {
            const float top = rt_max(logit);
            s = chosen && top >= kRtLowest ? rt_exp(logit - top) : 0.f;
            total = rt_sum(s);
        }
        const long long to = static_cast<long long>(row) * q.K;
        if (chosen) {
            q.idx[to + rank] = at;
            q.weights[to + rank] = total > 0.f ? s * rt_rcp(total) * q.route_scale : 0.f;
        }
        if (lane >= taken && lane < q.K) {
            q.idx[to + lane] = -1;
            q.weights[to + lane] = 0.f;
        }
    }
}

// CTAs of the kernels below that an SM is to hold, and the launches fill: registers for a token's logits, those of the next one and what is made of them. A grid of that size
// has each warp take several tokens, whose sums go out once.
template <int V>
constexpr int rt_ctas() { return V <= 4 ? 5 : (V <= 8 ? 4 : (V <= 12 ? 3 : (V <= 16 ? 2 : 1))); }

// ----------------------------------------------------------------------------- balance
// What a token's logits give, up to factors of the whole token: exp[j] * exp_scale is its softmax; in mode 1 sig[j] * sig_scale are its sigmoids over their sum, and
// 1 - sigmoid is rest[j] (where asked for).
template <int V>
struct RtScores {
    float exp[V], sig[V], rest[V], exp_scale, sig_scale, lse;
};

// `Careful` takes any logits; without it, it says (false) when they hold a NaN, or numbers so large that the result means nothing.
template <int V, int Mode, bool Rest, bool Careful>
__device__ __forceinline__ bool rt_scores_try(const float (&l)[V], RtScores<V>& s) {
    float top = l[0];
    #pragma unroll
    for (int j = 1; j < V; ++j) top = fmaxf(top, l[j]);                  // (NaN is no maximum)
    top = rt_max(top);
    s.exp_scale = s.sig_scale = s.lse = 0.f;
    if (Careful && top == rt_off()) {
        #pragma unroll
        for (int j = 0; j < V; ++j) s.exp[j] = s.sig[j] = s.rest[j] = 0.f;
        return true;
    }
    float sum = 0.f, sig_sum = 0.f;
    // mode 1: exp(l) by itself, where it neither overflows nor loses the largest of them, gives both the softmax and the sigmoid
    const bool plain = Mode == 1 && top >= kRtLow && top <= 40.f;
    const float base = plain ? 0.f : top, shift = base * kRtLog2e;
    #pragma unroll
    for (int j = 0; j < V; ++j) {
        s.exp[j] = Careful ? rt_exp(l[j] - base) : rt_exp2(fmaf(l[j], kRtLog2e, -shift));
        sum += s.exp[j];
    }
    sum = rt_sum(sum);
    if (!Careful && !(sum > 0.f && sum <= FLT_MAX)) return false;
    if (Mode == 1) {
        #pragma unroll
        for (int j = 0; j < V; ++j) {
            if (plain) {
                s.rest[j] = rt_rcp(1.f + s.exp[j]);
                s.sig[j] = s.exp[j] * s.rest[j];
            } else if (top < kRtLow) {
                s.sig[j] = top >= kRtLowest ? s.exp[j] : 0.f;
                s.rest[j] = 1.f;
            } else {
                s.sig[j] = rt_sigmoid(l[j]);
                if (Rest) s.rest[j] = rt_sigmoid_rest(l[j]);
            }
            sig_sum += s.sig[j];
        }
        sig_sum = rt_sum(sig_sum);
        s.sig_scale = sig_sum > 0.f ? rt_rcp(sig_sum) : 0.f;
    }
    s.exp_scale = rt_rcp(sum);
    s.lse = base + __logf(sum);
    return true;
}
template <int V, int Mode, bool Rest>
__device__ __forceinline__ void rt_scores(float (&l)[V], RtScores<V>& s) {
    if (rt_scores_try<V, Mode, Rest, false>(l, s)) return;
    rt_clean<V>(l);
    rt_scores_try<V, Mode, Rest, true>(l, s);
}

// Sums over the CTA, in a fixed order; the results are every thread's.
template <int N, int Warps = kRtWarps>
__device__ __forceinline__ void rt_block_sum(double (&v)[N], double (*part)[N]) {
    #pragma unroll
    for (int n = 0; n < N; ++n) {
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    }
    if ((threadIdx.x & 31) == 0) {
        #pragma unroll
        for (int n = 0; n < N; ++n) part[threadIdx.x >> 5][n] = v[n];
    }
    __syncthreads();
    #pragma unroll
    for (int n = 0; n < N; ++n) {
        v[n] = 0.0;
        #pragma unroll
        for (int w = 0; w < Warps; ++w) v[n] += part[w][n];
    }
}

// Counts and mean probabilities of the cells `first`, `first + stride`, ... (of all threads that take part); what they add to the balance loss.
__device__ __forceinline__ double rt_balance_cells(const RtParams& q, long long first, long long stride) {
    constexpr int kBatch = 6;                // cells in flight
    const long long cells = static_cast<long long>(q.S) * q.E;
    double balance = 0.0;
    for (long long i0 = first; i0 < cells; i0 += kBatch * stride) {
        unsigned long long sum[kBatch];
        int count[kBatch], n[kBatch];
        #pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const long long i = min(i0 + b * stride, cells - 1);
            sum[b] = __ldcg(q.sums + i);
            count[b] = __ldcg(q.sum_counts + i);
            n[b] = __ldcg(q.sum_tokens + (q.S == 1 ? 0 : static_cast<int>(static_cast<uint32_t>(i) / static_cast<uint32_t>(q.E))));
        }
        #pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const long long i = i0 + b * stride;
            if (i >= cells) break;
            const float inv = n[b] > 0 ? 1.f / static_cast<float>(n[b]) : 0.f, mean = static_cast<float>(sum[b]) * q.step * inv;
            q.mean[i] = mean;
            q.counts[i] = count[b];
            balance += static_cast<double>(static_cast<float>(count[b]) * inv) * static_cast<double>(mean);
        }
    }
    return balance;
}

// The results, by one CTA: the losses, and with `cells` all counts and mean probabilities. `balance`: what other CTAs' cells add to the balance loss, in all.
__device__ __forceinline__ void rt_balance_results(const RtParams& q, bool cells, double balance) {
    __shared__ double part[kRtWarps][4];
    double v[4] = {0.0, 0.0, 0.0, balance};                  // sequences with tokens, tokens, squares, balance
    for (int i = threadIdx.x; i < q.z_parts; i += blockDim.x) v[2] += __ldcg(q.z_part + i);
    for (int s = threadIdx.x; s < q.S; s += blockDim.x) {
        const int n = __ldcg(q.sum_tokens + s);
        q.tokens[s] = n;
        v[0] += n > 0;
        v[1] += n;
    }
    if (cells) v[3] += rt_balance_cells(q, threadIdx.x, blockDim.x);
    rt_block_sum<4>(v, part);
    if (threadIdx.x == 0) {
        const double b = v[0] > 0.0 ? v[3] * q.E / q.K / v[0] : 0.0, z = v[1] > 0.0 ? v[2] / v[1] : 0.0;
        q.losses[0] = static_cast<float>(q.balance_coef * b + q.z_coef * z);
        q.losses[1] = static_cast<float>(b);
        q.losses[2] = static_cast<float>(z);
    }
}

// Thread 0 counts this CTA in, behind a barrier that has brought it what the others wrote: whether it is the last of the grid (then what all CTAs wrote is there).
__device__ __forceinline__ bool rt_last_cta(unsigned* ticket, bool* last) {
    if (threadIdx.x == 0) *last = atom_acq_rel_gpu_add(ticket, 1u) == gridDim.x - 1;
    __syncthreads();
    return *last;
}

template <typename L>
__global__ void __launch_bounds__(256) balance_zero_kernel(const RtParams q) {
    grid_dependency_wait();
    grid_launch_dependents();
    unsigned long long* p = q.sums;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < q.zero_words; i += static_cast<long long>(gridDim.x) * blockDim.x) p[i] = 0ull;
}

// The tokens lo to hi - 1, piece by piece of one sequence each: the CTA's warps take them in turn and add up their probabilities in registers, a token's logits asked for while
// the one before is worked on. `count(s, e)` is told every slot; `flush(s, acc, n)` at the end of a piece what a warp has summed, and of how many
// tokens. Returns the warp's sum of squares.
template <typename L, int V, int Mode, int Warps, typename Count, typename Flush>
__device__ __forceinline__ double rt_balance_tokens(const RtParams& q, int lo, int hi, Count count, Flush flush) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float l[V];
    long long route = -1;
    // (a warp's tokens are one in `Warps` of the CTA's, whatever the pieces)
    auto fetch = [&](int r) {
        if (r < hi) {
            rt_fetch<L, V>(q, r, lane, l);
            route = lane < q.K ? q.idx[static_cast<long long>(r) * q.K + lane] : -1;
        }
    };
    int mine = lo + warp;                                                // this warp's next token
    fetch(mine);
    double z = 0.0;
    int row = lo;
    while (row < hi) {
        int s = 0, end = hi;
        if (q.cu != nullptr) {
            const int first = q.cu[0];
            if (row < first) {
                s = -1;
                end = min(hi, first);
            } else {
                s = rt_sequence(q.cu, q.S, row);
                if (s >= q.S) break;
                end = min(hi, max(q.cu[s + 1], row + 1));
            }
        }
        end = min(end, row + kRtFlushRows * Warps);
        float acc[V] = {};
        int n = 0;
        for (; mine < end; mine += Warps) {
            float x[V];
            RtScores<V> scores;
            #pragma unroll
            for (int j = 0; j < V; ++j) x[j] = l[j];
            const long long e = route;
            fetch(mine + Warps);
            const bool slot = s >= 0 && e >= 0 && e < q.E;
            if (__ballot_sync(0xffffffffu, slot) == 0u) continue;
            if (slot) count(s, static_cast<int>(e));
            rt_scores<V, Mode, false>(x, scores);
            #pragma unroll
            for (int j = 0; j < V; ++j) acc[j] = Mode == 1 ? fmaf(scores.sig[j], scores.sig_scale, acc[j]) : fmaf(scores.exp[j], scores.exp_scale, acc[j]);
            z += static_cast<double>(scores.lse) * static_cast<double>(scores.lse);
            ++n;
        }
        row = end;
        if (s >= 0) flush(s, acc, n);
    }
    return z;
}

// Many tokens: a CTA adds its warps' sums up and puts them to the sequence's in memory, which `balance_zero_kernel` has cleared. The last CTA to end turns the
// sums into the results where they are few.
template <typename L, int V, int Mode>
__global__ void __launch_bounds__(kRtWarps * 32, rt_ctas<V>()) balance_kernel(const RtParams q) {
    __shared__ float warp_sum[kRtWarps][V * 32];
    __shared__ int hist[V * 32], warp_tokens[kRtWarps];
    __shared__ double warp_z[kRtWarps];
    __shared__ bool last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lo = rt_share(q, blockIdx.x), hi = rt_share(q, blockIdx.x + 1);
    const float per_one = 1.f / q.step;
    for (int e = threadIdx.x; e < V * 32; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    grid_dependency_wait();                  // (for the cleared sums, and for the logits and routes of kernels ahead of `balance_zero_kernel`: only a grid that waits sees what others wrote)
    grid_launch_dependents();
    const double z = rt_balance_tokens<L, V, Mode, kRtWarps>(
        q, lo, hi, [&](int, int e) { atomicAdd(hist + e, 1); },
        [&](int s, const float (&acc)[V], int n) {
            #pragma unroll
            for (int j = 0; j < V; ++j) warp_sum[warp][j * 32 + lane] = acc[j];
            if (lane == 0) warp_tokens[warp] = n;
            __syncthreads();
            for (int e = threadIdx.x; e < q.E; e += blockDim.x) {
                unsigned long long sum = 0ull;
                #pragma unroll
                for (int w = 0; w < kRtWarps; ++w) sum += __float2ull_rn(warp_sum[w][e] * per_one);
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
        });
    if (lane == 0) warp_z[warp] = z;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        #pragma unroll
        for (int w = 0; w < kRtWarps; ++w) sum += warp_z[w];
        q.z_part[blockIdx.x] = sum;
    }
    if (static_cast<long long>(q.S) * q.E <= kRtEndCells && rt_last_cta(q.ticket, &last)) rt_balance_results(q, true, 0.0);
}

// Few tokens: one cluster, whose CTAs keep their sums in shared memory and add up each other's: one launch, nothing in memory but the results. A call from Python takes
// 2.5 us less of the host than with two launches (with the gradient 12.9 and 15.4 us a pass). On the GPU 16 tokens of 48 experts take 3.2 us, 256 5.4, 384 5.9, and by the two
// launches 385 take 5.9; of 384 experts 4.2, 5.9, 6.5 and 6.2, in five sequences 6.6, 7.8, 8.5 and 9.2: the border is where the GPU begins to lose.
template <typename T>
__device__ __forceinline__ T rt_of_cta(const T* p, uint32_t rank) {      // the same variable of another CTA of the cluster
    static_assert(sizeof(T) == 4 || sizeof(T) == 8);
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    if constexpr (sizeof(T) == 4) {
        uint32_t v;
        asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
        return *reinterpret_cast<T*>(&v);
    } else {
        unsigned long long v;
        asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
        return *reinterpret_cast<T*>(&v);
    }
}

template <typename L, int V, int Mode>
__global__ void __launch_bounds__(kRtSmallWarps * 32) balance_small_kernel(const RtParams q) {
    __shared__ float warp_sum[kRtSmallWarps][V * 32], sums[kRtSmallCells];
    __shared__ int counts[kRtSmallCells], tokens[kRtSmallSequences];
    __shared__ double warp_z[kRtSmallWarps], cta[2], part[kRtSmallWarps][1];       // cta: sum of squares; what its cells add to the balance loss
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = cluster_rank(), ctas = gridDim.x;
    const int cells = q.S * q.E;
    const int lo = rt_share(q, rank), hi = rt_share(q, rank + 1);
    for (int i = threadIdx.x; i < cells; i += blockDim.x) { sums[i] = 0.f; counts[i] = 0; }
    for (int i = threadIdx.x; i < q.S; i += blockDim.x) tokens[i] = 0;
    __syncthreads();
    grid_dependency_wait();
    grid_launch_dependents();
    const double z = rt_balance_tokens<L, V, Mode, kRtSmallWarps>(
        q, lo, hi, [&](int s, int e) { atomicAdd(counts + s * q.E + e, 1); },
        [&](int s, const float (&acc)[V], int n) {
            #pragma unroll
            for (int j = 0; j < V; ++j) warp_sum[warp][j * 32 + lane] = acc[j];
            if (lane == 0 && n > 0) atomicAdd(tokens + s, n);
            __syncthreads();
            for (int e = threadIdx.x; e < q.E; e += blockDim.x) {
                float sum = sums[s * q.E + e];
                #pragma unroll
                for (int w = 0; w < kRtSmallWarps; ++w) sum += warp_sum[w][e];
                sums[s * q.E + e] = sum;
            }
            __syncthreads();
        });
    if (lane == 0) warp_z[warp] = z;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        #pragma unroll
        for (int w = 0; w < kRtSmallWarps; ++w) sum += warp_z[w];
        cta[0] = sum;
    }
    cluster_arrive();
    cluster_wait();
    double balance[1] = {0.0};
    for (int i = static_cast<int>(rank * blockDim.x + threadIdx.x); i < cells; i += static_cast<int>(ctas * blockDim.x)) {
        const int s = q.S == 1 ? 0 : i / q.E;
        float sum = 0.f;
        int count = 0, n = 0;
        for (uint32_t r = 0; r < ctas; ++r) {
            sum += rt_of_cta(sums + i, r);
            count += rt_of_cta(counts + i, r);
            n += rt_of_cta(tokens + s, r);
        }
        const float inv = n > 0 ? 1.f / static_cast<float>(n) : 0.f, mean = sum * inv;
        q.mean[i] = mean;
        q.counts[i] = count;
        balance[0] += static_cast<double>(static_cast<float>(count) * inv) * static_cast<double>(mean);
    }
    rt_block_sum<1, kRtSmallWarps>(balance, part);
    if (threadIdx.x == 0) cta[1] = balance[0];
    cluster_arrive();
    cluster_wait();
    if (rank == 0 && warp == 0) {
        int live = 0, all = 0;
        for (int s = lane; s < q.S; s += 32) {
            int n = 0;
            for (uint32_t r = 0; r < ctas; ++r) n += rt_of_cta(tokens + s, r);
            q.tokens[s] = n;
            live += n > 0;
            all += n;
        }
        live = __reduce_add_sync(0xffffffffu, live);
        all = __reduce_add_sync(0xffffffffu, all);
        if (lane == 0) {
            double b = 0.0, squares = 0.0;
            for (uint32_t r = 0; r < ctas; ++r) { b += rt_of_cta(cta + 1, r); squares += rt_of_cta(cta, r); }
            b = live > 0 ? b * q.E / q.K / live : 0.0;
            squares = all > 0 ? squares / all : 0.0;
            q.losses[0] = static_cast<float>(q.balance_coef * b + q.z_coef * squares);
            q.losses[1] = static_cast<float>(b);
            q.losses[2] = static_cast<float>(squares);
        }
    }
    cluster_arrive();                        // (no CTA leaves while its shared memory is read)
    cluster_wait();
}

// The same for many sums: by as many CTAs as there are thousands of them; the last one adds up what the others found.
template <typename L>
__global__ void __launch_bounds__(kRtWarps * 32) balance_end_kernel(const RtParams q) {
    __shared__ double part[kRtWarps][1];
    __shared__ bool last;
    double balance[1] = {rt_balance_cells(q, static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x, static_cast<long long>(gridDim.x) * blockDim.x)};
    rt_block_sum<1>(balance, part);
    if (threadIdx.x == 0) q.end_part[blockIdx.x] = balance[0];
    if (!rt_last_cta(q.ticket, &last)) return;
    double all = 0.0;
    for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += blockDim.x) all += __ldcg(q.end_part + i);
    rt_balance_results(q, false, all);
}

// ----------------------------------------------------------------------------- gradient
// Consecutive tokens to a warp: the factors of a sequence's experts stay in registers. The routes' gradients, one per lane, get to their experts' lanes through a row in
// shared memory that is zero between the tokens.
template <typename L, int V, int Mode>
__global__ void __launch_bounds__(kRtWarps * 32, rt_ctas<V>()) router_backward_kernel(const RtParams q) {
    __shared__ float rows[kRtWarps][V * 32];
    const int lane = threadIdx.x & 31, warp_in = threadIdx.x >> 5;
    const int lo = rt_share(q, blockIdx.x * kRtWarps + warp_in), hi = rt_share(q, blockIdx.x * kRtWarps + warp_in + 1);
    float* buf = rows[warp_in];
    float c[V], ahead[V], dw_ahead = 0.f;
    long long e_ahead = -1;
    auto fetch = [&](int row) {
        if (row < hi) {
            rt_fetch<L, V>(q, row, lane, ahead);
            e_ahead = lane < q.K ? q.idx[static_cast<long long>(row) * q.K + lane] : -1;
            dw_ahead = q.d_weights != nullptr && lane < q.K ? q.d_weights[static_cast<long long>(row) * q.K + lane] : 0.f;
        }
    };
    grid_dependency_wait();
    grid_launch_dependents();
    fetch(lo);
    const float g = q.d_loss_ptr != nullptr ? *q.d_loss_ptr : q.d_loss;
    float live = 1.f, all = 1.f;
    #pragma unroll
    for (int j = 0; j < V; ++j) buf[j * 32 + lane] = 0.f;
    __syncwarp();
    if (q.balance) {
        // sequences that have tokens, and their tokens: whole numbers, by every warp for itself
        int a = 0;
        long long b = 0;
        for (int s = lane; s < q.S; s += 32) {
            const int n = q.tokens[s];
            a += n > 0;
            b += n;
        }
        a = __reduce_add_sync(0xffffffffu, a);
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) b += __shfl_xor_sync(0xffffffffu, b, o);
        live = static_cast<float>(a > 0 ? a : 1);
        all = static_cast<float>(b > 0 ? b : 1);
    }
    const float zc = 2.f * q.z_coef * g / all;
    int seq = -1, seq_end = -1;
    for (int row = lo; row < hi; ++row) {
        float l[V], d[V];
        #pragma unroll
        for (int j = 0; j < V; ++j) l[j] = ahead[j];
        const long long e64 = e_ahead;
        const float dw_in = dw_ahead;
        fetch(row + 1);
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
                const float f = n > 0.f ? __fdividef(q.balance_coef * g * static_cast<float>(q.E), static_cast<float>(q.K) * n) * __fdividef(1.f, n * live) : 0.f;
                #pragma unroll
                for (int j = 0; j < V; ++j)
                    c[j] = s < q.S && j * 32 + lane < q.E ? f * static_cast<float>(q.counts[static_cast<long long>(s) * q.E + j * 32 + lane]) : 0.f;
            }
            if (seq < q.S) {
                RtScores<V> x;
                rt_scores<V, Mode, true>(l, x);
                float inner = 0.f;
                #pragma unroll
                for (int j = 0; j < V; ++j) inner = fmaf(c[j], Mode == 1 ? x.sig[j] : x.exp[j], inner);
                inner = rt_sum(inner) * (Mode == 1 ? x.sig_scale : x.exp_scale);
                const float zl = zc * x.lse;
                #pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (Mode == 1) d[j] = fmaf(x.sig[j] * x.rest[j], x.sig_scale * (c[j] - inner), x.exp[j] * (x.exp_scale * zl));
                    else d[j] = x.exp[j] * (x.exp_scale * (c[j] - inner + zl));
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
                if (mine > rt_off()) w = rt_exp(mine - top);
            }
            float total = rt_sum(w);
            if (Mode == 1 && total < kRtLowSum) {                        // (then `rest` is 1 to 32 bits)
                const float top = rt_max(mine);
                w = mine > rt_off() && top >= kRtLowest ? rt_exp(mine - top) : 0.f;
                total = rt_sum(w);
            }
            w = total > 0.f ? w * rt_rcp(total) : 0.f;
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
    const int blocks = (q.T + kRtWarps - 1) / kRtWarps, resident = rt_ctas<V>() * sms;
    const int grid = blocks < 1 ? 1 : (blocks < resident ? blocks : resident);
    auto shared_out = [&](int shares) {
        RtParams p = q;
        p.share = q.T / shares;
        p.shares_more = q.T % shares;
        return p;
    };
    if constexpr (V <= kRtSmallExperts / 32) {
        if (op == kRtBalance && q.T <= kRtSmallTokens && static_cast<long long>(q.S) * q.E <= kRtSmallCells && q.S <= kRtSmallSequences) {
            // (sequences: all the CTAs there can be, because each takes its pieces of them one after the other)
            const int want = q.S > 1 ? q.T : (q.T + kRtSmallWarps - 1) / kRtSmallWarps, ctas = want < 1 ? 1 : (want < kRtSmallCtas ? want : kRtSmallCtas);
            MM_CUDA(launch_clusters(balance_small_kernel<L, V, Mode>, ctas, ctas, kRtSmallWarps * 32, stream, shared_out(ctas)));
            return MM_OK;
        }
    }
    if (op == kRtBalance) {
        // one sequence: two CTAs an SM at most, because what each CTA adds to the same sums and counts costs more than its share of the tokens (16384 tokens of 48 experts
        // with the gradient 15.4 us, with five an SM 17.0); several sequences: all that fit, because a CTA takes its pieces of sequences one after the other (12000 tokens of 128
        // experts in 37 sequences 23.5 us, with two an SM 24.6)
        const int most = q.cu == nullptr && 2 * sms < kRtBalanceCtas ? 2 * sms : kRtBalanceCtas;
        const int ctas = grid < most ? grid : most;
        RtParams b = shared_out(ctas);
        b.z_parts = ctas;
        b.step = 0x1p-63f;
        while (b.step * 0x1p63f < static_cast<float>(q.T)) b.step *= 2.f;    // (T as a float may be 2^-24 less: the sums have a bit to spare)
        const long long zero = (b.zero_words + 1023) / 1024;
        MM_CUDA(launch_behind(balance_zero_kernel<L>, static_cast<int>(zero < sms ? zero : sms), 256, stream, b));
        MM_CUDA(launch_behind(balance_kernel<L, V, Mode>, b.z_parts, kRtWarps * 32, stream, b));
        const long long cells = static_cast<long long>(q.S) * q.E;
        if (cells > kRtEndCells) {
            const long long want = cells / 2048;
            MM_CUDA(launch_plain(balance_end_kernel<L>, static_cast<unsigned>(want < kRtBalanceCtas ? want : kRtBalanceCtas), kRtWarps * 32, stream, b));
        }
    } else if (op == kRtRoute) {
        MM_CUDA(launch_behind(route_kernel<L, V, Mode>, blocks < sms * 8 ? blocks : sms * 8, kRtWarps * 32, stream, q));
    } else {
        MM_CUDA(launch_behind(router_backward_kernel<L, V, Mode>, grid, kRtWarps * 32, stream, shared_out(grid * kRtWarps)));
    }
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
