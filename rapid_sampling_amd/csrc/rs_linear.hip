// Instantiations, launchers and C entry points of the quantisers and the product in 8 bits.
#include "rs_linear.h"

namespace rs {

template <int DT>
static void launch_quantize(const QuantParams &p, bool tiles, hipStream_t st)
{
    if (tiles) hipLaunchKernelGGL(quantize_tiles_kernel<DT>, dim3((p.R + kFpBlock - 1) / kFpBlock * p.blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL(quantize_rows_kernel<DT>, dim3((uint32_t)(((uint64_t)p.R * p.blocks + 15) / 16)), dim3(256), 0, st, p);
}

template <int DT, int WN, int WM, int MT, int STAGES, bool EXACT>
static hipError_t launch_tiles(const LinearParams &p, hipStream_t st)
{
    using L = LinearTile<WN, WM, MT, STAGES, EXACT>;
    const uint64_t tiles = (uint64_t)((p.M + L::kTileM - 1) / L::kTileM) * ((p.N + L::kTileN - 1) / L::kTileN);
    if (tiles > 0x7FFFFFFF) return hipErrorInvalidValue;
    hipLaunchKernelGGL((linear_tile_kernel<DT, WN, WM, MT, STAGES, EXACT>), dim3((uint32_t)tiles), dim3(L::kThreads), L::kLds, st, p);
    return hipGetLastError();
}

template <int DT, int MT, int NT>
static hipError_t launch_few(const LinearParams &p, hipStream_t st)
{
    const uint32_t waves = p.blocks >= 8 ? 8 : p.blocks >= 4 ? 4 : p.blocks >= 2 ? 2 : 1;
    hipLaunchKernelGGL((linear_few_kernel<DT, MT, NT>), dim3((p.N + 16 * NT - 1) / (16 * NT), (p.M + 16 * MT - 1) / (16 * MT)), dim3(64 * waves), 0, st, p);
    return hipGetLastError();
}

template <int DT>
static hipError_t launch_linear(const LinearParams &p, hipStream_t st)
{
    // (the tiles' kernel reaches its rows with 32 bits)
    if (p.M <= 16 || p.x_stride > kTileStride || p.w_stride > kTileStride) return launch_few<DT, 1, 2>(p, st);
    constexpr bool kExact = DT == RS_DTYPE_F32;
    if (p.M <= 64) return launch_tiles<DT, 1, 4, 1, 3, true>(p, st);
    if constexpr (kExact) return launch_tiles<DT, 2, 4, 2, 3, true>(p, st);
    else return p.M <= 128 ? launch_tiles<DT, 2, 4, 2, 3, false>(p, st) : launch_tiles<DT, 2, 4, 4, 2, false>(p, st);
}

static bool known(int32_t dtype) { return dtype == RS_DTYPE_F32 || dtype == RS_DTYPE_BF16 || dtype == RS_DTYPE_F16; }

}  // namespace rs

using namespace rs;

extern "C" {

int rs_quantize_blocks(const void *x, int32_t dtype, int64_t x_row_stride, int32_t block_rows, int32_t R, int32_t K,
                       void *q, int64_t q_row_stride, float *scale, void *stream)
{
    if (!x || !q || !scale) return RS_ERR_NULL;
    if (!known(dtype) || (block_rows != 1 && block_rows != kFpBlock)) return RS_ERR_ARG;
    if (R <= 0 || K <= 0 || K > RS_LINEAR_MAX || (R > 1 && x_row_stride < 0)) return RS_ERR_SHAPE;
    if (q_row_stride < ((int64_t)K + 15) / 16 * 16) return RS_ERR_SHAPE;
    if (((uintptr_t)x & (dtype == RS_DTYPE_F32 ? 3 : 1)) || ((uintptr_t)q & 15) || (q_row_stride & 15) || ((uintptr_t)scale & 3)) return RS_ERR_ALIGN;
    QuantParams p;
    p.x = x; p.x_stride = x_row_stride; p.q = (uint8_t *)q; p.q_stride = q_row_stride; p.scale = scale;
    p.R = (uint32_t)R; p.K = (uint32_t)K; p.blocks = ((uint32_t)K + kFpBlock - 1) / kFpBlock;
    p.q_cols = (uint32_t)(q_row_stride < (int64_t)p.blocks * kFpBlock ? q_row_stride : (int64_t)p.blocks * kFpBlock);
    const hipStream_t st = (hipStream_t)stream;
    const bool tiles = block_rows != 1;
    if (dtype == RS_DTYPE_F32) launch_quantize<RS_DTYPE_F32>(p, tiles, st);
    else if (dtype == RS_DTYPE_BF16) launch_quantize<RS_DTYPE_BF16>(p, tiles, st);
    else launch_quantize<RS_DTYPE_F16>(p, tiles, st);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

int rs_linear_blocks(const void *x, int64_t x_row_stride, const float *x_scale,
                     const void *w, int64_t w_row_stride, const float *w_scale,
                     int32_t M, int32_t N, int32_t K, void *y, int32_t y_dtype, int64_t y_row_stride, void *stream)
{
    if (!x || !x_scale || !w || !w_scale || !y) return RS_ERR_NULL;
    if (!known(y_dtype)) return RS_ERR_ARG;
    if (M <= 0 || N <= 0 || K <= 0 || M > RS_LINEAR_MAX || N > RS_LINEAR_MAX || K > RS_LINEAR_MAX) return RS_ERR_SHAPE;
    if ((M > 1 && x_row_stride < K) || (N > 1 && w_row_stride < K) || (M > 1 && y_row_stride < N)) return RS_ERR_SHAPE;
    if (((uintptr_t)x & 15) || (M > 1 && (x_row_stride & 15)) || ((uintptr_t)w & 15) || (N > 1 && (w_row_stride & 15)) ||
        ((uintptr_t)x_scale & 3) || ((uintptr_t)w_scale & 3) || ((uintptr_t)y & (y_dtype == RS_DTYPE_F32 ? 3 : 1)))
        return RS_ERR_ALIGN;
    LinearParams p;
    p.x = (const uint8_t *)x; p.x_stride = x_row_stride; p.x_scale = x_scale;
    p.w = (const uint8_t *)w; p.w_stride = w_row_stride; p.w_scale = w_scale;
    p.y = y; p.y_stride = y_row_stride;
    p.M = (uint32_t)M; p.N = (uint32_t)N; p.K = (uint32_t)K; p.blocks = ((uint32_t)K + kFpBlock - 1) / kFpBlock;
    const hipStream_t st = (hipStream_t)stream;
    const hipError_t e = y_dtype == RS_DTYPE_F32 ? launch_linear<RS_DTYPE_F32>(p, st)
                       : y_dtype == RS_DTYPE_BF16 ? launch_linear<RS_DTYPE_BF16>(p, st) : launch_linear<RS_DTYPE_F16>(p, st);
    return e == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

}  // extern "C"
