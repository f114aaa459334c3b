// The linears behind atlas_qlinear_gemv and atlas_qlinear_gemm, with an epilogue and a second weight.
#pragma once
#include <cuda_runtime.h>

#include "epilogue.cuh"

namespace atlas {

// Rows of x up to which a linear with an epilogue goes to the per-strip kernel, as one without does (16 rows a pass over the weight).
constexpr int STRIP_MAX_ROWS = 16;

// `up`: the second weight of act(x W^T + b) * (x V^T + c), or null.
int qlinear_gemv(const void *x, int dtype, int64_t m, int64_t ldx, const uint8_t *tiles, const void *scales_tiled,
                 const int32_t *outlier_chunk_ptr, const uint32_t *outlier_entries, const void *outlier_vals_sorted,
                 int64_t n_rows, int64_t n_cols, int block_size, const void *bias, void *y, int64_t ldy, cudaStream_t st, const Epilogue &epi,
                 const AtlasWeight *up);
int qlinear_gemm(const void *x, int dtype, int64_t m, int64_t ldx, const uint8_t *tiles, const void *scales_tiled,
                 const int32_t *outlier_chunk_ptr, const uint32_t *outlier_entries, const void *outlier_vals_sorted,
                 int64_t n_rows, int64_t n_cols, int block_size, const void *bias, void *y, int64_t ldy, void *workspace,
                 size_t workspace_bytes, int32_t *status, void *stream, const AtlasPeerGather *gather, const Epilogue &epi, const AtlasWeight *up);
size_t qlinear_gemm_workspace_bytes(int64_t m, int64_t n_rows, int64_t n_cols, bool two);

}  // namespace atlas
