// Routing from fp16 logits, the balance loss and their gradient.
#include "mm_router.cuh"

namespace mm {

int launch_router_fp16(RtOp op, const RtParams& q, int sms, cudaStream_t stream) { return rt_launch<__half>(op, q, sms, stream); }

}  // namespace mm
