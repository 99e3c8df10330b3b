// Routing from bf16 logits, the balance loss and their gradient.
#include "mm_router.cuh"

namespace mm {

int launch_router_bf16(RtOp op, const RtParams& q, int sms, cudaStream_t stream) { return rt_launch<__nv_bfloat16>(op, q, sms, stream); }

}  // namespace mm
