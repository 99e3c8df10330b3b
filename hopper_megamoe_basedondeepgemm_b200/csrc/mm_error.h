// The last CUDA error of a thread as text (`mm_last_cuda_error`), shared by the library's source files.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace mm {

constexpr int kErrorBytes = 256;
extern thread_local char g_cuda_error[kErrorBytes];
int cuda_fail(cudaError_t e, const char* what);          // notes the error, returns MM_ERR_CUDA

}  // namespace mm

#define MM_CUDA(call) do { cudaError_t e_ = (call); if (e_ != cudaSuccess) return mm::cuda_fail(e_, #call); } while (0)
