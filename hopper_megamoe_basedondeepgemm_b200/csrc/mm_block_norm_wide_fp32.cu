// The norms of a transformer block, fp32 activations, rows of more than 4096 channels.
#include "mm_block_norm.cuh"

namespace mm {

int launch_block_norm_wide_fp32(const BnParams& q, const BnLaunch& how, cudaStream_t stream) {
    return bn_launch<float, float, true>(q, how, stream);
}

}  // namespace mm
