// The norms of a transformer block, fp32 activations.
#include "mm_block_norm.cuh"

namespace mm {

int launch_block_norm_fp32(const BnParams& q, const BnLaunch& how, cudaStream_t stream) {
    if (q.hidden > kBnOneHidden) return launch_block_norm_wide_fp32(q, how, stream);
    return bn_launch<float, float, false>(q, how, stream);
}
int launch_block_norm_sums_fp32(const BnSumsParams& q, cudaStream_t stream) { return bn_launch_sums<float>(q, stream); }

}  // namespace mm
