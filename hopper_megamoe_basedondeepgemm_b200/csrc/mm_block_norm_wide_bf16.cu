// The norms of a transformer block, bf16 activations, rows of more than 4096 channels.
#include "mm_block_norm.cuh"

namespace mm {

int launch_block_norm_wide_bf16(const BnParams& q, const BnLaunch& how, cudaStream_t stream) {
    return how.stream32 ? bn_launch<__nv_bfloat16, float, true>(q, how, stream) : bn_launch<__nv_bfloat16, __nv_bfloat16, true>(q, how, stream);
}

}  // namespace mm
