// Tensor-core (tcgen05) prefill GEMM for M > 32 tokens.
#pragma once
#include <cuda.h>

#include "nxq_internal.h"

namespace nxq {

int context_sm_count();
DeviceStatus* context_status();

// Kernel attributes and driver entry points; NXQ_PREFILL_KERNEL=simt selects
// the CUDA-core kernel instead (for comparisons).
int gemm_init(int device);
bool gemm_supported(const TiledShape& s, int64_t M);
void gemm_kernel_name(const TiledShape& s, int64_t M, char* buf, size_t n);
// y = x W^T; NXQ_ERR_UNSUPPORTED to decline.
int gemm_qmatmul(const Weight* w, const void* x, int x_dtype, void* y, int y_dtype, int64_t M, cudaStream_t st);

// Tensor map of f16 activations [rows][K] (16-byte aligned) for boxes of 64 k x
// box_rows rows, 128-byte swizzle; needs gemm_init with the kernel enabled.
int gemm_activation_map(CUtensorMap* tmap, const void* xh, int64_t rows, int64_t K, int box_rows);

// Whether tensor maps can be made (not with NXQ_PREFILL_KERNEL=simt), and one of 16-bit
// elements for boxes with a 128-byte swizzle: 0, or the driver's error.  `rank`
// dimensions, the first contiguous; `strides` of the others in bytes.
bool tensor_maps();
int tensor_map_16(CUtensorMap* tmap, bool bf16, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                  const uint32_t* box);

}  // namespace nxq
