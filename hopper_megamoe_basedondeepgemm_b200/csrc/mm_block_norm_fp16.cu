// The norms of a transformer block, fp16 activations.
#include "mm_block_norm.cuh"

namespace mm {

int launch_block_norm_fp16(const BnParams& q, const BnLaunch& how, cudaStream_t stream) {
    if (q.hidden > kBnOneHidden) return launch_block_norm_wide_fp16(q, how, stream);
    return how.stream32 ? bn_launch<__half, float, false>(q, how, stream) : bn_launch<__half, __half, false>(q, how, stream);
}
int launch_block_norm_sums_fp16(const BnSumsParams& q, cudaStream_t stream) { return bn_launch_sums<__half>(q, stream); }

}  // namespace mm
