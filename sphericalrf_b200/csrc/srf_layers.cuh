// srf_layers.cuh -- launch wrappers of the layer operators (srf_grouped.cu, srf_grouped_fp8.cu, srf_quantize.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/srf_abi.h"

namespace srf {

// NULL on success, else a static text of what went wrong.
const char* launch_grouped_matmul(const srf_grouped_t& p, const uint64_t* offsets, const void* x, const void* w, void* y,
                                  unsigned int* error_flags, cudaStream_t stream);
const char* launch_grouped_input_grad(const srf_grouped_t& p, const uint64_t* offsets, const void* dy, const void* w,
                                      const void* gate, void* dx, unsigned int* error_flags, cudaStream_t stream);
size_t grouped_weight_grad_workspace(const srf_grouped_t& p, int n_sms);
const char* launch_grouped_weight_grad(const srf_grouped_t& p, const uint64_t* offsets, const void* dy, const void* x, void* dw,
                                       void* workspace, unsigned int* error_flags, cudaStream_t stream);
const char* launch_grouped_matmul_fp8(const srf_grouped_t& p, const uint64_t* offsets, const void* x, const float* x_scales,
                                      const void* w, const float* w_scales, void* y, unsigned int* error_flags,
                                      cudaStream_t stream);
void launch_quantize_rows(int type, uint64_t n_rows, const uint64_t* n_rows_used, uint32_t n_cols, const void* in, uint64_t ld_in,
                          void* out, uint64_t ld_out, float* scales, cudaStream_t stream);
void launch_quantize_weights(int type, uint32_t n_matrices, uint32_t n_rows, uint32_t n_cols, const void* in, uint64_t ld_in,
                             uint64_t stride_in, void* out, uint64_t ld_out, uint64_t stride_out, float* scales, cudaStream_t stream);

// Host side of the tensor maps: element size 1 or 2, dims/strides innermost first, 128-byte swizzle, box {128 bytes,
// box_rows, 1}.  False when the driver refuses.
bool make_operand_map(void* map, const void* base, int type, uint64_t cols, uint64_t rows, uint64_t ld, uint64_t n_matrices,
                      uint64_t matrix_stride, uint32_t box_rows);
int sm_count();

}  // namespace srf
