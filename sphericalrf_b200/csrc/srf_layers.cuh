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
const char* launch_quantize_rows(int type, uint64_t n_rows, const uint64_t* n_rows_used, uint32_t n_cols, const void* in, uint64_t ld_in,
                          void* out, uint64_t ld_out, float* scales, cudaStream_t stream);
const char* launch_quantize_weights(int type, uint32_t n_matrices, uint32_t n_rows, uint32_t n_cols, const void* in, uint64_t ld_in,
                             uint64_t stride_in, void* out, uint64_t ld_out, uint64_t stride_out, float* scales, cudaStream_t stream);

// Host side of the tensor maps: element size 1 or 2, dims/strides innermost first, 128-byte swizzle, box {128 bytes,
// box_rows, 1}.  False when the driver refuses.
bool make_operand_map(void* map, const void* base, int type, uint64_t cols, uint64_t rows, uint64_t ld, uint64_t n_matrices,
                      uint64_t matrix_stride, uint32_t box_rows);
int sm_count();

// Row tiles of `height` that n_rows samples in n_groups groups can have at most.
uint64_t max_row_tiles(const srf_grouped_t& p, uint64_t height);
// Output tiles of a layer or an input gradient with `cols` columns: CG*128 samples x BN columns on CG CTAs.  A single CTA
// loads its samples in boxes of kRowBox rows, as many as the tile has.
constexpr uint32_t kRowBox = 32;
struct TileShape { int bn, cg; };
// `cols_step`: 32 where a pair's tiles may be narrower than 256 (8-bit tiles may not: their halves are scale blocks).
TileShape pick_tile(const srf_grouped_t& p, uint32_t cols, int sms, int smallest, int cols_step);
// CTAs for them: one per SM, no more than there can be tiles.
uint32_t tile_grid(const srf_grouped_t& p, uint32_t cols, TileShape t, int sms);

// One launch of a layer kernel; `cg` CTAs to a cluster.  The kernel may be set up while the one in front of it in the stream
// still runs (it waits for that one before it touches memory): layers follow one another in chains, and for a few
// samples the set-up is most of a layer's time.
template <class Kernel, class... Args>
const char* launch_layer(Kernel kernel, int smem, int threads, int cg, dim3 grid, cudaStream_t stream, const Args&... args) {
    if (smem > 48 * 1024 && cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return "cudaFuncSetAttribute failed";
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cg;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cg > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? nullptr : "the layer kernel did not launch";
}

}  // namespace srf
