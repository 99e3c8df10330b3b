// Routing from fp32 logits, the balance loss and their gradient.
#include "mm_router.cuh"

namespace mm {

int launch_router_fp32(RtOp op, const RtParams& q, int sms, cudaStream_t stream) { return rt_launch<float>(op, q, sms, stream); }

}  // namespace mm
