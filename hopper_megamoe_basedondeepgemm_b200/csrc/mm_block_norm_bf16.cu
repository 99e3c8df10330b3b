// The norms of a transformer block, bf16 activations.
#include "mm_block_norm.cuh"

namespace mm {

int launch_block_norm_bf16(const BnParams& q, const BnLaunch& how, cudaStream_t stream) {
    if (q.hidden > kBnOneHidden) return launch_block_norm_wide_bf16(q, how, stream);
    return how.stream32 ? bn_launch<__nv_bfloat16, float, false>(q, how, stream) : bn_launch<__nv_bfloat16, __nv_bfloat16, false>(q, how, stream);
}
int launch_block_norm_sums_bf16(const BnSumsParams& q, cudaStream_t stream) { return bn_launch_sums<__nv_bfloat16>(q, stream); }

}  // namespace mm
