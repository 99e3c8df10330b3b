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
// In the backward pass everything that goes through y is written with the coefficient a = scale * (gate of the channel) * (offset + w_post) and
// v = y i1 a (times the token's or element's gate): then the sum that the norm of y needs is sum of v dr, which with
// dr = d_r' + i2 (dh w2 - m n2),  m = i2 / H * sum of dh w2 r',  falls apart into sums of v d_r', v dh w2 and v r'. They are taken together with
// those of the norm of r', so that a row needs one exchange between its threads. The gradients of a channel's gate and of w_post are one sum over
// the rows, of dr n1 (token's or element's gate), times the other's factor. Rows are multiplied by their root before anything else: powers of i1 and i2 by
// themselves leave the range of 32 bits for streams from 10^12 on, and for rows of zeros with an eps below 10^-25.
//
// A row belongs to one CTA, or with more than 4096 channels to two (a cluster), eight channels to a thread. Bound by memory: the bytes of the rows, in and out. CTAs stay and walk over the rows; a
// thread asks for its part of the next row before it works on the one it has, and while a row's sums are exchanged, the sum of squares of the next row's
// y goes with them: one barrier a row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "../../include/megamoe_b200.h"
#include "mm_block_norm.h"
#include "mm_error.h"
#include "mm_launch.h"
#include "mm_ptx.cuh"

namespace mm {

template <typename T> __device__ __forceinline__ float bn_float(T v);
template <> __device__ __forceinline__ float bn_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float bn_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float bn_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T bn_round(float v);
template <> __device__ __forceinline__ float bn_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 bn_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half bn_round<__half>(float v) { return __float2half_rn(v); }

// How a row lies over the threads. kBnWhole: every row starts on 16 bytes (32-bit elements: 32) and is made of groups of eight channels, of which a thread has one, in one
// access. Otherwise a thread's eight channels lie the threads' number apart, so that neighbouring threads read neighbouring elements wherever the row starts.
// kBnTwo: the row belongs to a cluster of two CTAs (more than 4096 channels).
enum BnLayout { kBnWhole = 1, kBnTwo = 2 };
template <int Lay>
__device__ __forceinline__ int bn_thread() { return static_cast<int>((Lay & kBnTwo) != 0 ? (blockIdx.x & 1u) * blockDim.x + threadIdx.x : threadIdx.x); }
template <int Lay>
__device__ __forceinline__ int bn_width() { return static_cast<int>((Lay & kBnTwo) != 0 ? 2u * blockDim.x : blockDim.x); }

// Sums of N values (a power of two) over the row's threads, the same in every thread. In a warp the values are dealt out while they are added: each step
// halves both the values of a lane and the lanes of a value. Each warp's sums go through shared memory (`part`, all zero at first, of which a turn
// is used at a time: the next sums' values go where no thread can still be reading, so one barrier does), and four lanes add up one value. Two CTAs leave
// their warps' sums in the shared memory of both, each in its half, so both add the same numbers in the same order; no CTA writes to the other behind the last barrier.
constexpr int kBnSumWarps = kBnMaxThreads / 32;
template <int Room, int Lay> using BnSums = float[2][Room][kBnSumWarps * ((Lay & kBnTwo) != 0 ? 2 : 1)];
template <int Lay>
__device__ __forceinline__ void bn_barrier() {
    if constexpr ((Lay & kBnTwo) != 0) { cluster_arrive(); cluster_wait(); } else { __syncthreads(); }
}
template <int N, int Lay, int Room>
__device__ __forceinline__ void bn_sum(float (&v)[N], BnSums<Room, Lay>& part, int& turn) {
    static_assert(N <= Room && N <= 16);
    constexpr bool kTwo = (Lay & kBnTwo) != 0;
    const uint32_t lane = threadIdx.x & 31u;
    float s[N];
    #pragma unroll
    for (int n = 0; n < N; ++n) s[n] = v[n];
    int o = 16;
    #pragma unroll
    for (int half = N / 2; half > 0; half /= 2, o /= 2) {
        #pragma unroll
        for (int n = 0; n < half; ++n) {
            const bool up = (lane & o) != 0u;
            const float keep = up ? s[n + half] : s[n], send = up ? s[n] : s[n + half];
            s[n] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
    #pragma unroll
    for (; o > 0; o /= 2) s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
    const uint32_t mine = lane * N / 32;                     // the value that this lane has the warp's sum of
    if (kTwo || blockDim.x > 32) {
        auto& p = part[turn];
        turn ^= 1;
        if (lane % (32 / N) == 0) {
            if constexpr (kTwo) {
                const uint32_t rank = blockIdx.x & 1u;
                float* at = &p[mine][rank * kBnSumWarps + (threadIdx.x >> 5)];
                *at = s[0];
                st_cluster_f32(at, rank ^ 1u, s[0]);
            } else {
                p[mine][threadIdx.x >> 5] = s[0];
            }
        }
        bn_barrier<Lay>();
        #pragma unroll
        for (int first = 0; first < N; first += 8) {         // eight values at a time
            const float* of = &p[first + (lane >> 2) % (N < 8 ? N : 8)][(lane & 3u) * 4u];
            const float4 w = *reinterpret_cast<const float4*>(of);
            float t = (w.x + w.y) + (w.z + w.w);
            if constexpr (kTwo) {
                const float4 x = *reinterpret_cast<const float4*>(of + kBnSumWarps);
                t += (x.x + x.y) + (x.z + x.w);
            }
            t += __shfl_xor_sync(0xffffffffu, t, 1);
            t += __shfl_xor_sync(0xffffffffu, t, 2);
            #pragma unroll
            for (int n = 0; n < 8 && first + n < N; ++n) v[first + n] = __shfl_sync(0xffffffffu, t, n * 4);
        }
    } else {
        #pragma unroll
        for (int n = 0; n < N; ++n) v[n] = __shfl_sync(0xffffffffu, s[0], n * (32 / N));
    }
}
static_assert(kBnSumWarps == 16, "four lanes read four warps' sums each");

template <int Lay, int Room>
__device__ __forceinline__ void bn_sum_init(BnSums<Room, Lay>& part) {
    if ((Lay & kBnTwo) != 0 || blockDim.x > 32) {
        for (int i = threadIdx.x; i < static_cast<int>(sizeof(part) / 4); i += blockDim.x) (&part[0][0][0])[i] = 0.f;
        bn_barrier<Lay>();
    }
}

// ----------------------------------------------------------------------------- channels of a thread
// Two 32-bit numbers in one register pair: one instruction adds or multiplies both.
__device__ __forceinline__ unsigned long long bn_bits(float2 v) { return *reinterpret_cast<unsigned long long*>(&v); }
__device__ __forceinline__ float2 bn_pair(unsigned long long b) { return *reinterpret_cast<float2*>(&b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bn_bits(a)), "l"(bn_bits(b)), "l"(bn_bits(c)));
    return bn_pair(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bn_bits(a)), "l"(bn_bits(b)));
    return bn_pair(d);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Eight elements as they lie in memory. Loads of them are written down where they are to be issued (volatile), a row ahead of their use.
template <typename T> struct Bn8 { uint32_t w[sizeof(T) * 2]; };

__device__ __forceinline__ void bn_unpack(const Bn8<float>& r, float2 (&v)[4]) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
}
__device__ __forceinline__ void bn_unpack(const Bn8<__nv_bfloat16>& r, float2 (&v)[4]) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(r.w[i] << 16), __uint_as_float(r.w[i] & 0xffff0000u));
}
__device__ __forceinline__ void bn_unpack(const Bn8<__half>& r, float2 (&v)[4]) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
}
__device__ __forceinline__ Bn8<float> bn_pack(const float2 (&v)[4], float) {
    Bn8<float> r;
    #pragma unroll
    for (int i = 0; i < 4; ++i) { r.w[2 * i] = __float_as_uint(v[i].x); r.w[2 * i + 1] = __float_as_uint(v[i].y); }
    return r;
}
__device__ __forceinline__ Bn8<__nv_bfloat16> bn_pack(const float2 (&v)[4], __nv_bfloat16) {
    Bn8<__nv_bfloat16> r;
    #pragma unroll
    for (int i = 0; i < 4; ++i) { const __nv_bfloat162 p = __float22bfloat162_rn(v[i]); r.w[i] = *reinterpret_cast<const uint32_t*>(&p); }
    return r;
}
__device__ __forceinline__ Bn8<__half> bn_pack(const float2 (&v)[4], __half) {
    Bn8<__half> r;
    #pragma unroll
    for (int i = 0; i < 4; ++i) { const __half2 p = __float22half2_rn(v[i]); r.w[i] = *reinterpret_cast<const uint32_t*>(&p); }
    return r;
}

// Eight elements on their way: as they will lie in memory, or one to a register, because putting two of them together waits for both.
template <typename T, int Lay> struct BnAhead { uint32_t w[(Lay & kBnWhole) != 0 || sizeof(T) == 4 ? sizeof(T) * 2 : 8]; };
template <typename T, int Lay>
__device__ __forceinline__ Bn8<T> bn_take(const BnAhead<T, Lay>& a) {
    Bn8<T> r;
    #pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) * 2; ++i) r.w[i] = (Lay & kBnWhole) != 0 || sizeof(T) == 4 ? a.w[i] : (a.w[(2 * i) & 7] | a.w[(2 * i + 1) & 7] << 16);
    return r;
}

// The eight channels of this thread in a row: in one access (of 32 bytes for 32-bit elements: two of 16 would each move half of every 32-byte sector), or one by one.
template <typename T, int Lay>
__device__ __forceinline__ void bn_fetch(const T* row, int hidden, BnAhead<T, Lay>& r) {
    if constexpr ((Lay & kBnWhole) != 0) {
        const T* p = row + bn_thread<Lay>() * 8;
        if constexpr (sizeof(T) == 4)
            asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]),
                         "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7]) : "l"(p) : "memory");
        else
            asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "l"(p) : "memory");
    } else {
        int at = bn_thread<Lay>();
        #pragma unroll
        for (int i = 0; i < 8; ++i, at += bn_width<Lay>()) {
            if constexpr (sizeof(T) == 4)
                asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\tmov.b32 %0, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}" : "=&r"(r.w[i]) : "l"(row + at), "r"(at), "r"(hidden) : "memory");
            else
                asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\tmov.b32 %0, 0;\n\t@p ld.global.u16 %0, [%1];\n\t}" : "=&r"(r.w[i]) : "l"(row + at), "r"(at), "r"(hidden) : "memory");
        }
    }
}
template <typename T, int Lay>
__device__ __forceinline__ void bn_put(T* row, int hidden, const float2 (&v)[4]) {
    const Bn8<T> r = bn_pack(v, T());
    if constexpr ((Lay & kBnWhole) != 0) {
        T* p = row + bn_thread<Lay>() * 8;
        if constexpr (sizeof(T) == 4)
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]),
                         "r"(r.w[7]) : "memory");
        else
            asm volatile("st.global.v4.b32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]) : "memory");
    } else {
        const int at = bn_thread<Lay>(), width = bn_width<Lay>();
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int a = at + 2 * i * width, b = a + width;
            if constexpr (sizeof(T) == 4) {
                if (a < hidden) reinterpret_cast<uint32_t*>(row)[a] = r.w[2 * i];
                if (b < hidden) reinterpret_cast<uint32_t*>(row)[b] = r.w[2 * i + 1];
            } else {
                if (a < hidden) reinterpret_cast<uint16_t*>(row)[a] = static_cast<uint16_t>(r.w[i]);
                if (b < hidden) reinterpret_cast<uint16_t*>(row)[b] = static_cast<uint16_t>(r.w[i] >> 16);
            }
        }
    }
}

// weights and gates of the channels
template <typename X, int Lay>
__device__ __forceinline__ void bn_weight(const void* w, int is32, int hidden, float2 (&v)[4]) {
    if (is32) { BnAhead<float, Lay> r; bn_fetch<float, Lay>(static_cast<const float*>(w), hidden, r); bn_unpack(bn_take(r), v); }
    else { BnAhead<X, Lay> r; bn_fetch<X, Lay>(static_cast<const X*>(w), hidden, r); bn_unpack(bn_take(r), v); }
}
// scale * (channel's gate) * (offset + w_post): the factor of y
template <typename X, int Lay>
__device__ __forceinline__ void bn_y_factor(const BnParams& q, float2 (&a)[4]) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = both(q.scale);
    if (q.post_w != nullptr) {
        float2 w[4];
        bn_weight<X, Lay>(q.post_w, q.weight32, q.hidden, w);
        #pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = make_float2(q.scale * (w[i].x + q.offset), q.scale * (w[i].y + q.offset));
    }
    if (q.gate_mode == kBnGateChannel) {
        float2 g[4];
        bn_weight<X, Lay>(q.gate, q.gate32, q.hidden, g);
        #pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = mul2(a[i], g[i]);
    }
}
template <typename X, int Lay>
__device__ __forceinline__ void bn_pre_factor(const BnParams& q, float2 (&w)[4]) {
    bn_weight<X, Lay>(q.pre_w, q.weight32, q.hidden, w);
    #pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = make_float2(w[i].x + q.offset, w[i].y + q.offset);
}

// A token's gate is asked for a row ahead as it lies in memory, and turned into a number when its row comes: a conversion at the load would wait for it. No
// branches: they would part the work of two rows.
template <typename X>
__device__ __forceinline__ uint32_t bn_gate_bits(const BnParams& q, long long row) {
    uint32_t bits;
    const long long at = row * q.gate_ld;
    if constexpr (sizeof(X) == 4)
        asm volatile("ld.global.b32 %0, [%1];" : "=r"(bits) : "l"(static_cast<const uint32_t*>(q.gate) + at) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\t@p ld.global.b32 %0, [%1];\n\t@!p ld.global.u16 %0, [%1];\n\t}"
                     : "=r"(bits) : "l"(static_cast<const char*>(q.gate) + (at << (q.gate32 ? 2 : 1))), "r"(q.gate32) : "memory");
    return bits;
}
template <typename X>
__device__ __forceinline__ float bn_gate_value(const BnParams& q, uint32_t bits) {
    if constexpr (sizeof(X) == 4) return __uint_as_float(bits);
    const uint16_t half = static_cast<uint16_t>(bits);
    const float narrow = bn_float<X>(*reinterpret_cast<const X*>(&half));
    return q.gate32 ? __uint_as_float(bits) : narrow;
}
// An element's gate: of the activations' type or 32 bits, held in room for the latter. Whole rows: loads under a predicate instead of two branches, behind which the loaded
// numbers would be moved and waited for (8192 x 3072 bf16, gradient 91 us instead of 99). Channels one by one have no registers to spare for that (norm of 8192 x 3001 96 us instead of 88).
template <typename X, int Lay>
__device__ __forceinline__ void bn_fetch_gate(const BnParams& q, long long row, uint32_t (&r)[8]) {
    if constexpr (sizeof(X) == 2 && (Lay & kBnWhole) != 0) {
        const int shift = q.gate32 ? 2 : 1;
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %9, 0;\n\t@p ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
                     "@!p ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%8];\n\t}"
                     : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                     : "l"(static_cast<const char*>(q.gate) + (row * q.gate_ld + bn_thread<Lay>() * 8 << shift)), "r"(q.gate32) : "memory");
    } else if (sizeof(X) == 4 || q.gate32) {
        BnAhead<float, Lay> f;
        bn_fetch<float, Lay>(static_cast<const float*>(q.gate) + row * q.gate_ld, q.hidden, f);
        #pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = f.w[i];
    } else {
        BnAhead<X, Lay> h;
        bn_fetch<X, Lay>(static_cast<const X*>(q.gate) + row * q.gate_ld, q.hidden, h);
        #pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(h.w) / 4); ++i) r[i] = h.w[i];
    }
}
template <typename X, int Lay>
__device__ __forceinline__ void bn_unpack_gate(const BnParams& q, const uint32_t (&r)[8], float2 (&g)[4]) {
    if (sizeof(X) == 4 || q.gate32) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    } else {
        BnAhead<X, Lay> h;
        #pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(h.w) / 4); ++i) h.w[i] = r[i];
        bn_unpack(bn_take(h), g);
    }
}

__device__ __forceinline__ float bn_square(const float2 (&v)[4]) {
    float2 s = mul2(v[0], v[0]);
    #pragma unroll
    for (int i = 1; i < 4; ++i) s = fma2(v[i], v[i], s);
    return s.x + s.y;
}
template <typename T> __device__ __forceinline__ float bn_square(const Bn8<T>& r) { float2 v[4]; bn_unpack(r, v); return bn_square(v); }
template <int N>
__device__ __forceinline__ void bn_clear(uint32_t (&w)[N]) {
    #pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 0u;
}

// What there is in a call, as far as it shapes the loop over the rows.
enum BnKind { kBnPlain = 0 /* no gate, or one that is part of y's factor */, kBnToken = 1, kBnElement = 2, kBnStream = 3 /* no y */ };

// 64 registers a thread, so two CTAs of 512 threads an SM; 16-bit streams 56, so three of 384. 16384 x 4096, 32-bit stream, both norms, channel gate: 127 us (6.3 TB/s); 8192 x
// 3072 in bf16 37 us (5.4). (One CTA of twice the registers an SM 168 us; sixteen channels a thread 134; rows copied ahead into shared memory by cp.async
// 160. y one row ahead, bf16 40 us; two rows ahead with a 32-bit stream, which then has no register left, 137.)
// Rows over two CTAs wait for the cluster's barrier (and for the stores that its release orders): 8192 x 8192 bf16 121 us (4.4 TB/s), 32-bit stream 158 (5.1), 32-bit activations
// 191 (5.6), 4096 x 6144 bf16 47 (64 registers, so two CTAs an SM, 55; one CTA with sixteen channels a thread and nothing in flight ahead 178). Clusters of four are slower: 173,
// 232 with a 32-bit stream, and 76.
template <typename X, typename R, bool Post, bool Pre, int Kind, int Lay>
__global__ void __maxnreg__((sizeof(R) == 2 && (Lay & kBnWhole) != 0 && Kind != kBnElement ? 56 : 64)) block_norm_kernel(const BnParams q) {
    constexpr bool kWhole = (Lay & kBnWhole) != 0, kTwo = (Lay & kBnTwo) != 0;
    __shared__ __align__(16) BnSums<2, Lay> part;
    const float inv_h = 1.f / static_cast<float>(q.hidden);
    constexpr bool kFar = Post && kWhole && sizeof(R) == 2;      // y two rows ahead: its squares are summed a row before its turn
    const int step = kTwo ? gridDim.x >> 1 : gridDim.x, tokens = static_cast<int>(q.tokens);
    const bool on = !kWhole || bn_thread<Lay>() * 8 < q.hidden;
    BnAhead<R, Lay> rr;
    BnAhead<X, Lay> ry, ry_far;
    uint32_t rg[8];
    float2 a[4], w[4];
    uint32_t gate_bits = 0u;
    bn_clear(rr.w);
    bn_clear(ry.w);
    bn_clear(ry_far.w);
    bn_clear(rg);
    #pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = w[i] = both(0.f);
    grid_dependency_wait();
    grid_launch_dependents();
    auto fetch = [&](long long row) {
        if (on) {
            if (kFar) {
                if (row + step < tokens) bn_fetch<X, Lay>(static_cast<const X*>(q.y) + (row + step) * q.y_ld, q.hidden, ry_far);
            } else if (Kind != kBnStream) {
                bn_fetch<X, Lay>(static_cast<const X*>(q.y) + row * q.y_ld, q.hidden, ry);
            }
            bn_fetch<R, Lay>(static_cast<const R*>(q.residual) + row * q.residual_ld, q.hidden, rr);
            if (Kind == kBnElement) bn_fetch_gate<X, Lay>(q, row, rg);
        }
        if (Kind == kBnToken) gate_bits = bn_gate_bits<X>(q, row);
    };
    int row = kTwo ? blockIdx.x >> 1 : blockIdx.x;
    if (kFar && on) bn_fetch<X, Lay>(static_cast<const X*>(q.y) + row * q.y_ld, q.hidden, ry);
    fetch(row);
    if (on) {
        if (Kind != kBnStream) bn_y_factor<X, Lay>(q, a);
        if (Pre) bn_pre_factor<X, Lay>(q, w);
    }
    bn_sum_init<Lay, 2>(part);
    int turn = 0;
    float i1 = 1.f;
    if (Post) {
        float sum[1] = {bn_square(bn_take(ry))};
        bn_sum<1, Lay, 2>(sum, part, turn);
        i1 = rsqrtf(sum[0] * inv_h + q.eps);
    }
    while (true) {
        const bool more = row + step < tokens;
        float2 r[4], v[4], g[4];
        bn_unpack(bn_take(rr), r);
        if (Kind != kBnStream) bn_unpack(bn_take(ry), v);
        if (Kind == kBnElement) bn_unpack_gate<X, Lay>(q, rg, g);
        const float f = Kind == kBnToken ? i1 * bn_gate_value<X>(q, gate_bits) : i1;
        if (kFar) ry = ry_far;
        if (more) fetch(row + step);
        if (Kind != kBnStream) {
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (Post || Kind == kBnToken) v[i] = mul2(v[i], both(f));
                if (Kind == kBnElement) v[i] = mul2(v[i], g[i]);
                r[i] = fma2(v[i], a[i], r[i]);
            }
            if (on) bn_put<R, Lay>(static_cast<R*>(q.residual_out) + row * q.residual_out_ld, q.hidden, r);
        }
        if (Pre) {
            // the sum of the next row's squares goes with this row's
            float sum[2] = {bn_square(r), 0.f};
            if (Post) {
                sum[1] = bn_square(bn_take(ry));
                bn_sum<2, Lay, 2>(sum, part, turn);
                i1 = rsqrtf(sum[1] * inv_h + q.eps);
            } else {
                float only[1] = {sum[0]};
                bn_sum<1, Lay, 2>(only, part, turn);
                sum[0] = only[0];
            }
            const float2 i2 = both(rsqrtf(sum[0] * inv_h + q.eps));
            #pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = mul2(mul2(r[i], i2), w[i]);
            if (on) bn_put<X, Lay>(static_cast<X*>(q.normed) + row * q.normed_ld, q.hidden, r);
        } else if (Post) {
            float sum[1] = {bn_square(bn_take(ry))};
            bn_sum<1, Lay, 2>(sum, part, turn);
            i1 = rsqrtf(sum[0] * inv_h + q.eps);
        }
        if (!more) return;
        row += step;
    }
}

// Rows are dealt to the CTAs in turn; a thread sums what the gradients of its channels' weights are made of over the CTA's rows and leaves it in `partial`, which
// `block_norm_sums_kernel` adds up: always in the same order. Some 330 instructions a warp and row, so the issue slots are half full; what is left is the wait for a row's
// exchange, and registers bound what can go on meanwhile: 128 a thread, a row being worked on and a row on its way, y two rows ahead (its sum of squares goes
// with the exchange of the row before). 8192 x 4096, 32-bit stream, both norms: 100 us (6.0 TB/s); y one row ahead 131.
// Where a CTA of 128 registers a thread leaves an SM's registers half used and no second one fits (more than 256 threads, up to 384: hidden 2056 to 3072, and 4104 to 6144 over two CTAs), it takes two rows
// at a time through one exchange, with 168: 8192 x 3072 in bf16 62 us (one row at a time 67), with a token's gate 64, with a 32-bit stream 78 (81). (With 256 threads
// two CTAs of one row win, 44 us against 46 for 8192 x 2048; with an element's gate, or 32-bit
// activations, two rows do not fit the registers.) With an element's gate one row takes those 168: 128 are too few, and a register that is put away while its load is on its way
// waits for it (8192 x 3072 bf16 82 us instead of 94, 8192 x 3001 134 instead of 370; odd rows without such a gate are faster with 128, 114 against 141).
// Rows over two CTAs: 8192 x 8192 bf16 259 us (3.1 TB/s), 32-bit stream 277 (4.4), 4096 x 6144 bf16, two rows at a time, 87 (one at a time 111; clusters of four 172).
template <typename X, typename R, bool Post, bool Pre, int Kind, int Lay, int Rows, int Most>
__global__ void __launch_bounds__(Most, 1) block_norm_backward_kernel(const BnParams q) {
    constexpr bool kY = Kind != kBnStream, kSumV = Post || Kind == kBnToken;
    constexpr int kSums = (kSumV ? 8 : 2) * Rows;
    constexpr bool kWhole = (Lay & kBnWhole) != 0, kTwo = (Lay & kBnTwo) != 0;
    __shared__ __align__(16) BnSums<kSums, Lay> part;
    const int team = kTwo ? blockIdx.x >> 1 : blockIdx.x, teams = kTwo ? gridDim.x >> 1 : gridDim.x;
    const float inv_h = 1.f / static_cast<float>(q.hidden);
    const int step = teams * Rows, tokens = static_cast<int>(q.tokens);
    const bool on = !kWhole || bn_thread<Lay>() * 8 < q.hidden, sum_y = Post || q.gate_mode == kBnGateChannel, has_d = q.d_residual_out != nullptr;
    BnAhead<R, Lay> rd[Rows], rr[Rows];                      // on their way
    BnAhead<X, Lay> ry_ahead[Rows], rh[Rows];
    Bn8<X> ry[Rows];                                         // norm of y: the next rows'
    uint32_t rg[Rows][8], gate_bits[Rows];
    float2 a[4], w[4], acc_pre[4], acc_y[4];
    #pragma unroll
    for (int n = 0; n < Rows; ++n) {
        bn_clear(rd[n].w);
        bn_clear(rr[n].w);
        bn_clear(ry[n].w);
        bn_clear(rh[n].w);
        bn_clear(ry_ahead[n].w);
        bn_clear(rg[n]);
        gate_bits[n] = 0u;
    }
    #pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = w[i] = acc_pre[i] = acc_y[i] = both(0.f);
    auto fetch_y = [&](int first) {
        #pragma unroll
        for (int n = 0; n < Rows; ++n) {
            const long long row = first + n;
            if (kY && on && row < tokens) bn_fetch<X, Lay>(static_cast<const X*>(q.y) + row * q.y_ld, q.hidden, ry_ahead[n]);
            else bn_clear(ry_ahead[n].w);
        }
    };
    auto fetch = [&](int first) {
        fetch_y(Post ? first + step : first);
        #pragma unroll
        for (int n = 0; n < Rows; ++n) {
            const long long row = first + n;
            if (n > 0 && row >= tokens) {                    // (a pair without its second row works on zeros)
                bn_clear(rr[n].w);
                bn_clear(rh[n].w);
                bn_clear(rd[n].w);
                continue;
            }
            if (on) {
                if (Pre) {
                    bn_fetch<R, Lay>(static_cast<const R*>(q.residual) + row * q.residual_ld, q.hidden, rr[n]);
                    bn_fetch<X, Lay>(static_cast<const X*>(q.d_normed) + row * q.d_normed_ld, q.hidden, rh[n]);
                }
                if (has_d) bn_fetch<R, Lay>(static_cast<const R*>(q.d_residual_out) + row * q.d_residual_out_ld, q.hidden, rd[n]);
                if (Kind == kBnElement) bn_fetch_gate<X, Lay>(q, row, rg[n]);
            }
            if (Kind == kBnToken) gate_bits[n] = bn_gate_bits<X>(q, row);
        }
    };
    int first = team * Rows;
    grid_dependency_wait();
    grid_launch_dependents();                                // (the sums' kernel waits for this one's end by itself)
    if (Post) {
        fetch_y(first);
        #pragma unroll
        for (int n = 0; n < Rows; ++n) ry[n] = bn_take(ry_ahead[n]);
    }
    fetch(first);
    if (on) {
        if (kY) bn_y_factor<X, Lay>(q, a);
        if (Pre) bn_pre_factor<X, Lay>(q, w);
    }
    bn_sum_init<Lay, kSums>(part);
    int turn = 0;
    float i1[Rows];
    #pragma unroll
    for (int n = 0; n < Rows; ++n) i1[n] = 1.f;
    if (Post) {
        float sum[Rows];
        #pragma unroll
        for (int n = 0; n < Rows; ++n) sum[n] = bn_square(ry[n]);
        bn_sum<Rows, Lay, kSums>(sum, part, turn);
        #pragma unroll
        for (int n = 0; n < Rows; ++n) i1[n] = rsqrtf(sum[n] * inv_h + q.eps);
    }
    while (true) {
        const bool more = first + step < tokens;
        Bn8<R> cd[Rows];
        Bn8<X> cy[Rows], ch[Rows];
        uint32_t cg[Rows][8];
        float2 r[Rows][4];
        float gate[Rows];
        #pragma unroll
        for (int n = 0; n < Rows; ++n) {
            cd[n] = bn_take(rd[n]);
            cy[n] = Post ? ry[n] : bn_take(ry_ahead[n]);
            ch[n] = bn_take(rh[n]);
            #pragma unroll
            for (int i = 0; i < 8; ++i) cg[n][i] = rg[n][i];
            if (Pre) bn_unpack(bn_take(rr[n]), r[n]);
            if (Post) ry[n] = bn_take(ry_ahead[n]);
            gate[n] = Kind == kBnToken ? bn_gate_value<X>(q, gate_bits[n]) : 1.f;
        }
        if (more) fetch(first + step);
        float sum[kSums];                                    // of each row: r' r', dh w2 r'; v d, v dh w2, v r' (v without a token's gate), next y's squares
        #pragma unroll
        for (int n = 0; n < Rows; ++n) {
            float2 v[4], dh[4], d[4], g[4], t[5];
            #pragma unroll
            for (int k = 0; k < 5; ++k) t[k] = both(0.f);
            if (kY) bn_unpack(cy[n], v);
            if (Kind == kBnElement) bn_unpack_gate<X, Lay>(q, cg[n], g);
            if (Pre) bn_unpack(ch[n], dh);
            if (kSumV) bn_unpack(cd[n], d);
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (kY) {
                    v[i] = mul2(Post ? mul2(v[i], both(i1[n])) : v[i], a[i]);
                    if (Kind == kBnElement) v[i] = mul2(v[i], g[i]);
                }
                if (Pre) {
                    if (kY) r[n][i] = fma2(v[i], both(gate[n]), r[n][i]);
                    dh[i] = mul2(dh[i], w[i]);
                    t[0] = fma2(r[n][i], r[n][i], t[0]);
                    t[1] = fma2(dh[i], r[n][i], t[1]);
                }
                if (kSumV) {
                    t[2] = fma2(v[i], d[i], t[2]);
                    if (Pre) { t[3] = fma2(v[i], dh[i], t[3]); t[4] = fma2(v[i], r[n][i], t[4]); }
                }
            }
            float* to = sum + n * (kSums / Rows);
            to[0] = t[0].x + t[0].y;
            to[1] = t[1].x + t[1].y;
            if (kSumV) {
                #pragma unroll
                for (int k = 2; k < 5; ++k) to[k] = t[k].x + t[k].y;
                to[5] = Post ? bn_square(ry[n]) : 0.f;
                to[6] = to[7] = 0.f;
            }
        }
        if (kSumV || Pre) bn_sum<kSums, Lay, kSums>(sum, part, turn);
        float gate_back[Rows];
        #pragma unroll
        for (int n = 0; n < Rows; ++n) {
            const long long row = first + n;
            const bool there = n == 0 || row < tokens;
            const float* of = sum + n * (kSums / Rows);
            const float i2 = Pre ? rsqrtf(of[0] * inv_h + q.eps) : 0.f, mean = Pre ? i2 * of[1] * inv_h : 0.f;       // mean: of dh w2 n2
            const float vd = kSumV ? (Pre ? of[2] + i2 * (of[3] - mean * (i2 * of[4])) : of[2]) : 0.f;
            gate_back[n] = vd;
            float2 d[4];
            bn_unpack(cd[n], d);
            if (Pre) {
                float2 dh[4];
                bn_unpack(ch[n], dh);
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // (i2 ahead of w: dh w once more would be kept from above, eight registers a row that two rows do not have, 72 us for 64 with a token's gate)
                    const float2 h2 = mul2(dh[i], both(i2)), n2 = mul2(r[n][i], both(i2));
                    acc_pre[i] = fma2(dh[i], n2, acc_pre[i]);
                    d[i] = fma2(h2, w[i], fma2(n2, both(-i2 * mean), d[i]));
                }
            }
            if (on && there) bn_put<R, Lay>(static_cast<R*>(q.d_residual) + row * q.d_residual_ld, q.hidden, d);
            if (kY) {
                const float2 y_back = both(-gate[n] * inv_h * vd);
                float2 y[4];                                 // n1 with a norm of y
                bn_unpack(cy[n], y);
                if (Post) {
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = mul2(y[i], both(i1[n]));
                }
                if (Kind == kBnElement) {
                    float2 g[4], dg[4];
                    bn_unpack_gate<X, Lay>(q, cg[n], g);
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        dg[i] = mul2(mul2(y[i], a[i]), d[i]);
                        d[i] = mul2(d[i], g[i]);
                    }
                    if (on && there) {
                        const long long at = row * q.d_gate_ld;
                        if (sizeof(X) == 4 || q.gate32) bn_put<float, Lay>(static_cast<float*>(q.d_gate) + at, q.hidden, dg);
                        else bn_put<X, Lay>(static_cast<X*>(q.d_gate) + at, q.hidden, dg);
                    }
                }
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 du = Kind == kBnToken ? mul2(d[i], both(gate[n])) : d[i];
                    acc_y[i] = fma2(du, y[i], acc_y[i]);
                    d[i] = Post ? mul2(fma2(y[i], y_back, mul2(du, a[i])), both(i1[n])) : mul2(du, a[i]);
                }
                if (on && there) bn_put<X, Lay>(static_cast<X*>(q.d_y) + row * q.d_y_ld, q.hidden, d);
            }
            if (Post) i1[n] = rsqrtf(of[5] * inv_h + q.eps);
        }
        if (Kind == kBnToken && (!kTwo || (blockIdx.x & 1u) == 0u) && threadIdx.x < Rows && first + static_cast<int>(threadIdx.x) < tokens) {
            const long long at = (first + static_cast<int>(threadIdx.x)) * q.d_gate_ld;
            const float of = Rows == 2 && threadIdx.x == 1 ? gate_back[Rows - 1] : gate_back[0];
            if (sizeof(X) == 4 || q.gate32) static_cast<float*>(q.d_gate)[at] = of;
            else static_cast<X*>(q.d_gate)[at] = bn_round<X>(of);
        }
        if (!more) break;
        first += step;
    }
    if (!on) return;
    float* p = q.partial + static_cast<long long>(team) * q.hidden;
    if (Pre) bn_put<float, Lay>(p, q.hidden, acc_pre);
    if (sum_y) bn_put<float, Lay>(Pre ? p + static_cast<long long>(teams) * q.hidden : p, q.hidden, acc_y);
}

// Column sums of the CTAs' partial sums: a block takes 32 channels of one of the two, a thread every 128th row of four channels, a few loads that are all on their way at
// once; added up over a warp's four rows by shuffles, then over the warps in order. 148 to 1184 rows that lie in the L2.
constexpr int kBnSumThreads = 1024;
template <typename X>
__global__ void __launch_bounds__(kBnSumThreads) block_norm_sums_kernel(const BnSumsParams q) {
    __shared__ float part[kBnSumThreads / 32][33];
    const int col = (threadIdx.x & 7) * 4, group = threadIdx.x >> 3, blocks = (q.hidden + 31) / 32, which = blockIdx.x / blocks, h0 = (blockIdx.x - which * blocks) * 32;
    const bool of_pre = q.d_pre_w != nullptr && which == 0;
    float v[4] = {};
    const float* p = q.partial + static_cast<long long>(which) * q.rows * q.hidden + h0 + col;
    grid_dependency_wait();
    grid_launch_dependents();
    if ((q.hidden & 3) == 0) {
        if (h0 + col < q.hidden) {
            #pragma unroll 5
            for (int r = group; r < q.rows; r += kBnSumThreads / 8) {
                const float4 f = *reinterpret_cast<const float4*>(p + static_cast<long long>(r) * q.hidden);
                v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
            }
        }
    } else {
        #pragma unroll 5
        for (int r = group; r < q.rows; r += kBnSumThreads / 8) {
            #pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += h0 + col + i < q.hidden ? p[static_cast<long long>(r) * q.hidden + i] : 0.f;
        }
    }
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] += __shfl_xor_sync(0xffffffffu, v[i], 8);
        v[i] += __shfl_xor_sync(0xffffffffu, v[i], 16);
        if ((threadIdx.x & 31) < 8) part[threadIdx.x >> 5][col + i] = v[i];
    }
    __syncthreads();
    const int h = h0 + static_cast<int>(threadIdx.x);
    if (threadIdx.x >= 32 || h >= q.hidden) return;
    float sum = 0.f;
    #pragma unroll
    for (int g = 0; g < kBnSumThreads / 32; ++g) sum += part[g][threadIdx.x];
    auto put = [&](void* to, int is32, float x) {
        if (is32) static_cast<float*>(to)[h] = x; else static_cast<X*>(to)[h] = bn_round<X>(x);
    };
    auto get = [&](const void* from, int is32) { return is32 ? static_cast<const float*>(from)[h] : bn_float<X>(static_cast<const X*>(from)[h]); };
    if (of_pre) { put(q.d_pre_w, q.weight32, sum); return; }
    if (q.d_post_w != nullptr) put(q.d_post_w, q.weight32, q.scale * (q.gate != nullptr ? get(q.gate, q.gate32) : 1.f) * sum);
    if (q.d_gate != nullptr) put(q.d_gate, q.gate32, q.scale * (q.post_w != nullptr ? get(q.post_w, q.weight32) + q.offset : 1.f) * sum);
}

// ----------------------------------------------------------------------------- launches
// `teams`: CTAs, or pairs of them, that rows are dealt to
template <auto Kernel, int Lay>
int bn_start(const BnParams& q, int teams, cudaStream_t stream) {
    if constexpr ((Lay & kBnTwo) != 0) MM_CUDA(launch_clusters(Kernel, 2u * teams, 2, bn_threads(q.hidden), stream, q));
    else MM_CUDA(launch_behind(Kernel, teams, bn_threads(q.hidden), stream, q));
    return MM_OK;
}

// CTAs of a kernel that an SM holds; asked for once per CTA size and kernel (the answer is the binary's and the GPU's, of which there is one kind).
template <auto Kernel>
int bn_per_sm(int threads, int* per) {
    static std::atomic<int> known[kBnMaxThreads / 32 + 1] = {};
    const int k = known[threads / 32].load(std::memory_order_relaxed);
    if (k > 0) { *per = k; return MM_OK; }
    int n = 0;
    MM_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, threads, 0));
    *per = n > 0 ? n : 1;
    known[threads / 32].store(*per, std::memory_order_relaxed);
    return MM_OK;
}

template <typename X, typename R, bool Post, bool Pre, int Kind, int Lay>
int bn_launch_kind(const BnParams& q, const BnLaunch& how, cudaStream_t stream) {
    if (how.backward) {
        constexpr bool kPairs = (Lay & kBnWhole) != 0 && Kind != kBnElement && sizeof(X) == 2, kMore = Kind == kBnElement;
        const int threads = bn_threads(q.hidden);
        if (threads > kBnMaxThreads / 2 && threads <= kBnPairThreads) {
            if constexpr (kPairs) {
                if (q.tokens >= 2ll * how.teams) return bn_start<block_norm_backward_kernel<X, R, Post, Pre, Kind, Lay, 2, kBnPairThreads>, Lay>(q, how.teams, stream);
            }
            if constexpr (kMore) return bn_start<block_norm_backward_kernel<X, R, Post, Pre, Kind, Lay, 1, kBnPairThreads>, Lay>(q, how.teams, stream);
        }
        return bn_start<block_norm_backward_kernel<X, R, Post, Pre, Kind, Lay, 1, kBnMaxThreads>, Lay>(q, how.teams, stream);
    }
    int per = 0;
    const int st = bn_per_sm<block_norm_kernel<X, R, Post, Pre, Kind, Lay>>(bn_threads(q.hidden), &per);
    if (st != MM_OK) return st;
    const long long most = static_cast<long long>(per) * how.sms / ((Lay & kBnTwo) != 0 ? 2 : 1);
    return bn_start<block_norm_kernel<X, R, Post, Pre, Kind, Lay>, Lay>(q, static_cast<int>(q.tokens < most ? q.tokens : most), stream);
}

template <typename X, typename R, int Lay>
int bn_launch_rows(const BnParams& q, const BnLaunch& how, cudaStream_t stream) {
    const bool post = q.post_w != nullptr, pre = q.pre_w != nullptr;
    if (q.y == nullptr) return bn_launch_kind<X, R, false, true, kBnStream, Lay>(q, how, stream);
    auto by_kind = [&](auto p, auto n) {
        constexpr bool kPost = decltype(p)::value, kPre = decltype(n)::value;
        if (q.gate_mode == kBnGateToken) return bn_launch_kind<X, R, kPost, kPre, kBnToken, Lay>(q, how, stream);
        if (q.gate_mode == kBnGateElement) return bn_launch_kind<X, R, kPost, kPre, kBnElement, Lay>(q, how, stream);
        return bn_launch_kind<X, R, kPost, kPre, kBnPlain, Lay>(q, how, stream);
    };
    using std::false_type;
    using std::true_type;
    return post ? (pre ? by_kind(true_type{}, true_type{}) : by_kind(true_type{}, false_type{}))
                : (pre ? by_kind(false_type{}, true_type{}) : by_kind(false_type{}, false_type{}));
}

// Two: rows of more than 4096 channels (compiled in files of their own)
template <typename X, typename R, bool Two>
int bn_launch(const BnParams& q, const BnLaunch& how, cudaStream_t stream) {
    constexpr int two = Two ? kBnTwo : 0;
    return how.aligned ? bn_launch_rows<X, R, two | kBnWhole>(q, how, stream) : bn_launch_rows<X, R, two>(q, how, stream);
}

template <typename X>
int bn_launch_sums(const BnSumsParams& q, cudaStream_t stream) {
    MM_CUDA(launch_behind(block_norm_sums_kernel<X>, (q.hidden + 31) / 32 * q.sums, kBnSumThreads, stream, q));
    return MM_OK;
}

}  // namespace mm
