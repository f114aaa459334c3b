// Quantized linears with an epilogue (epilogue.cuh): argument checks, and which kernel.
//
// As the linears without an epilogue: the per-strip kernel (gemv.cu) up to 16 rows of x, above that the tcgen05 kernels
// (gemm_tile.cu, gemm.cu).  The epilogue stands where they round their sums.
#include "common.cuh"
#include "linear.cuh"

namespace atlas {
namespace {

// What the kernels take for granted of a weight's buffers: codes are read, and scales copied, 16 bytes at a time.
bool aligned(const AtlasWeight &w) {
    return !(((uintptr_t)w.tiles | (uintptr_t)w.scales_tiled) & 15) && !(((uintptr_t)w.outlier_chunk_ptr | (uintptr_t)w.outlier_entries) & 3) &&
           !(((uintptr_t)w.outlier_vals_sorted | (uintptr_t)w.bias) & 1);
}

int check(const AtlasFusedLinear *p) {
    const char *what = "atlas_fused_linear";
    ATLAS_RETURN_IF(!p, ATLAS_ERR_BAD_ARGUMENT, "%s: no arguments", what);
    ATLAS_RETURN_IF(p->activation < ATLAS_ACT_NONE || p->activation > ATLAS_ACT_GELU_TANH, ATLAS_ERR_BAD_ARGUMENT, "%s: activation %d", what, p->activation);
    ATLAS_RETURN_IF(p->m < 0 || p->n_rows <= 0 || p->n_cols <= 0, ATLAS_ERR_BAD_ARGUMENT, "%s: m=%lld n_rows=%lld n_cols=%lld", what, (long long)p->m,
                    (long long)p->n_rows, (long long)p->n_cols);
    ATLAS_RETURN_IF(p->residual && p->m > 1 && p->ldr < p->n_rows, ATLAS_ERR_BAD_ARGUMENT, "%s: residual rows %lld apart", what, (long long)p->ldr);
    ATLAS_RETURN_IF(p->up.tiles && (!p->up.scales_tiled || !p->up.outlier_chunk_ptr), ATLAS_ERR_BAD_ARGUMENT, "%s: the second weight lacks a buffer", what);
    ATLAS_RETURN_IF(!aligned(p->weight) || (p->up.tiles && !aligned(p->up)), ATLAS_ERR_BAD_ARGUMENT,
                    "%s: tiles and scales must be 16-byte aligned, a weight's other buffers to their types", what);
    ATLAS_RETURN_IF(((uintptr_t)p->x | (uintptr_t)p->y | (uintptr_t)p->residual) & 1, ATLAS_ERR_BAD_ARGUMENT, "%s: x, y or residual is not aligned to its type", what);
    ATLAS_RETURN_IF((uintptr_t)p->status & 3, ATLAS_ERR_BAD_ARGUMENT, "%s: status is not aligned to its type", what);
    return ATLAS_OK;
}

// Gate and up with 9 to 16 rows: two token tiles of strips leave no room for both weights' strips in one CTA, so pairs of CTAs
// are only better than the tcgen05 kernel while all of them run at once (2 x 1000 x 1024 4.3 us, 5.5; 2 x 2048 x 1024 4.7, 7.7;
// 2 x 5504 x 2048 17.7, 12.0; 2 x 11008 x 4096 44.4, 36.4).  Up to 8 rows strips are ahead everywhere (2 x 11008 x 4096 22.7 to
// 26.2, 34.8 to 35.6; 2 x 8192 x 2048 12.2 to 13.6, 13.7 to 14.0).  What a tile gives away to the joined linear alone, which strips
// serve: 2 x 11008 x 4096 at 9 and 16 fp16 rows 35.4 and 35.7 us, 28.8 and 33.4; 2 x 8192 x 2048 14.3 and 14.5, 14.8 and 16.7.  The
// joined linear with silu and the product behind it, as modules compute it, takes longer: 12 bf16 rows of the former 38.4, 35.7 here.
bool by_strips(const AtlasFusedLinear *p) {
    return p->m <= STRIP_MAX_ROWS && (!p->up.tiles || p->m <= 8 || 2 * ceil_div_i64(p->n_rows, 16) <= 2 * 148);
}

}  // namespace
}  // namespace atlas

extern "C" size_t atlas_fused_linear_workspace_bytes(const AtlasFusedLinear *p) {
    using namespace atlas;
    if (check(p) != ATLAS_OK || by_strips(p)) return 0;
    return qlinear_gemm_workspace_bytes(p->m, p->n_rows, p->n_cols, p->up.tiles != nullptr);
}

extern "C" int atlas_fused_linear(const AtlasFusedLinear *p, void *stream) {
    using namespace atlas;
    clear_error();
    const int rc = check(p);
    if (rc != ATLAS_OK) return rc;
    if (p->m == 0) return ATLAS_OK;
    const Epilogue epi = make_epilogue(p->residual, p->ldr, p->scale, p->activation);
    const AtlasWeight &w = p->weight, *up = p->up.tiles ? &p->up : nullptr;
    if (by_strips(p))
        return qlinear_gemv(p->x, p->dtype, p->m, p->ldx, w.tiles, w.scales_tiled, w.outlier_chunk_ptr, w.outlier_entries, w.outlier_vals_sorted, p->n_rows,
                            p->n_cols, p->block_size, w.bias, p->y, p->ldy, (cudaStream_t)stream, epi, up);
    return qlinear_gemm(p->x, p->dtype, p->m, p->ldx, w.tiles, w.scales_tiled, w.outlier_chunk_ptr, w.outlier_entries, w.outlier_vals_sorted, p->n_rows, p->n_cols,
                        p->block_size, w.bias, p->y, p->ldy, p->workspace, p->workspace_bytes, p->status, stream, nullptr, epi, up);
}
