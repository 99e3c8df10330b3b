// The norms of a transformer block, fp16 activations, rows of more than 4096 channels.
#include "mm_block_norm.cuh"

namespace mm {

int launch_block_norm_wide_fp16(const BnParams& q, const BnLaunch& how, cudaStream_t stream) {
    return how.stream32 ? bn_launch<__half, float, true>(q, how, stream) : bn_launch<__half, __half, true>(q, how, stream);
}

}  // namespace mm
