// Instantiations, launchers and C entry points of the quantisers and the product in 8 bits.
#include "rs_linear.h"

#include <algorithm>

namespace rs {

// As many rows at a time as a launch holds: a workgroup of 256 makes a block of 128 x 128, or 16 of 1 x 128.
template <int DT>
static void launch_quantize(QuantParams p, bool tiles, hipStream_t st)
{
    constexpr uint32_t kGroups = kGridThreads / 256u;
    const uint32_t R = p.R, most = std::min<uint64_t>(R, (uint64_t)kGroups * (tiles ? 1 : 16) / p.blocks * (tiles ? kFpBlock : 1));
    for (uint32_t done = 0; done < R; done += p.R) {
        p.R = std::min(most, R - done);
        if (tiles) hipLaunchKernelGGL(quantize_tiles_kernel<DT>, dim3((uint32_t)(((uint64_t)p.R + kFpBlock - 1) / kFpBlock) * p.blocks), dim3(256), 0, st, p);
        else hipLaunchKernelGGL(quantize_rows_kernel<DT>, dim3((uint32_t)(((uint64_t)p.R * p.blocks + 15) / 16)), dim3(256), 0, st, p);
        p.x = (const char *)p.x + (int64_t)p.R * p.x_stride * (DT == RS_DTYPE_F32 ? 4 : 2);
        p.q += (int64_t)p.R * p.q_stride;
        p.scale += (size_t)(tiles ? p.R / kFpBlock : p.R) * p.blocks;
    }
}

// SPLIT: where there are few tiles their blocks of columns are shared out, for up to one workgroup to a compute unit.  Leaving and
// adding up the parts costs about 2 us, a block 0.9: four blocks to each at least (64 x 1024 x 4096: 30.7 us whole, 12.9 in eight;
// 64 x 4096 x 512: 6.5 whole, 8.0 in two).
template <int DT, int WN, int WM, int NU, int MT, int STAGES, bool SPLIT>
static hipError_t launch_tiles(LinearParams p, hipStream_t st)
{
    using L = LinearTile<WN, WM, NU, MT, STAGES>;
    static_assert(!SPLIT || L::kTileN * L::kTileM * 4 <= kPartBytes, "a tile's sums fit the workspace");
    const uint64_t tiles = (uint64_t)((p.M + L::kTileM - 1) / L::kTileM) * ((p.N + L::kTileN - 1) / L::kTileN);
    p.split = SPLIT ? (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({kPartTiles / tiles, p.blocks / 4, 8})) : 1;
    hipLaunchKernelGGL((linear_tile_kernel<DT, WN, WM, NU, MT, STAGES, SPLIT>), dim3((uint32_t)tiles * p.split), dim3(L::kThreads), L::kLds, st, p);
    return hipGetLastError();
}

template <int DT, int XT, int NT>
static hipError_t launch_few(const LinearParams &p, hipStream_t st)
{
    const uint32_t waves = p.blocks >= 8 ? 8 : p.blocks >= 4 ? 4 : p.blocks >= 2 ? 2 : 1;
    const uint32_t lds = XT < 0 ? 0 : p.M * p.blocks * (kFpBlock + 4);
    hipLaunchKernelGGL((linear_few_kernel<DT, XT, NT>), dim3((p.N + 16 * NT - 1) / (16 * NT), (p.M + 15) / 16), dim3(64 * waves), lds, st, p);
    return hipGetLastError();
}

// 32 rows of w to a workgroup, 16 where there are few (x in 8 bits, 1 x 1024 x 8192: 13.9 us against 10.1; 1 x 8192 x 4096: 9.6
// against 9.4; 1 x 16384 x 4096: 15.3 against 16.5; 1 x 65536 x 4096: 50.8 against 59.1).
template <int DT, int XT>
static hipError_t launch_few(const LinearParams &p, hipStream_t st)
{
    return p.N <= 8192 ? launch_few<DT, XT, 1>(p, st) : launch_few<DT, XT, 2>(p, st);
}

template <int DT>
static hipError_t launch_rows(const LinearParams &p, int32_t x_dtype, hipStream_t st)
{
    return x_dtype == RS_DTYPE_F32 ? launch_few<DT, RS_DTYPE_F32>(p, st) : x_dtype == RS_DTYPE_BF16 ? launch_few<DT, RS_DTYPE_BF16>(p, st) : launch_few<DT, RS_DTYPE_F16>(p, st);
}

// Times in us on one card, weights beyond its caches unless said otherwise.
template <int DT>
static hipError_t launch_linear(const LinearParams &p, hipStream_t st)
{
    // Up to 16 rows one 16 x 16 product holds them all, and nothing but w is worth staging (1 x 131072 x 4096: 98, 5.5 TB/s).
    // (The tiles' kernel reaches its rows with 32 bits.)
    if (p.M <= 16 || p.x_stride > kTileStride || p.w_stride > kTileStride) return launch_few<DT, -1>(p, st);
    // Tiles of 128 x 64 (rows of w x rows of x) for up to 64 rows, and wherever those of 128 x 128 would not give every compute unit
    // its own (100 x 8192 x 4096: 21.8 against 40.6; 1000 x 4096 x 4096: 46.6 against 47.3).  Two waves share w's rows and two x's,
    // since both have to be widened (64 x 131072 x 4096: 118.6 against 121.5 with four and one).
    const uint64_t n128 = (p.N + 127) / 128, m128 = (p.M + 127) / 128;
    if (p.M <= 64 || n128 * m128 <= 256) return launch_tiles<DT, 2, 2, 4, 2, 3, true>(p, st);
    // 128 x 128: 4096 x 32768 x 4096 in 1105, 1055 into bfloat16 (1.0 PFLOP/s), against 1329 and 1257 in tiles of 128 x 64; 300 x 16384
    // x 4096 in 69.6 against 72.5
    return launch_tiles<DT, 1, 4, 8, 2, 2, false>(p, st);
}

static LinearParams linear_params(const void *x, int64_t x_stride, const float *x_scale, const void *w, int64_t w_stride, const float *w_scale,
                                  int32_t M, int32_t N, int32_t K, void *y, int64_t y_stride, void *workspace)
{
    // (the distance to the next row of a single one is not looked at by the checks, and a tile's other rows must lie behind it)
    const int64_t alone = ((int64_t)K + 15) / 16 * 16;
    LinearParams p;
    p.x = (const uint8_t *)x; p.x_stride = M > 1 ? x_stride : alone; p.x_scale = x_scale;
    p.w = (const uint8_t *)w; p.w_stride = N > 1 ? w_stride : alone; p.w_scale = w_scale;
    p.y = y; p.y_stride = y_stride;
    p.M = (uint32_t)M; p.N = (uint32_t)N; p.K = (uint32_t)K; p.blocks = ((uint32_t)K + kFpBlock - 1) / kFpBlock;
    p.split = 1;
    p.arrived = (uint32_t *)workspace;
    p.parts = workspace ? (float *)((char *)workspace + 16 * kPartTiles) : nullptr;
    return p;
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

size_t rs_linear_workspace_bytes(void) { return kPartTiles * (kPartBytes + 16); }

int rs_linear_blocks(const void *x, int64_t x_row_stride, const float *x_scale,
                     const void *w, int64_t w_row_stride, const float *w_scale,
                     int32_t M, int32_t N, int32_t K, void *y, int32_t y_dtype, int64_t y_row_stride,
                     void *workspace, size_t workspace_bytes, void *stream)
{
    if (!x || !x_scale || !w || !w_scale || !y || !workspace) return RS_ERR_NULL;
    if (workspace_bytes < rs_linear_workspace_bytes() || ((uintptr_t)workspace & 255)) return RS_ERR_WORKSPACE;
    if (!known(y_dtype)) return RS_ERR_ARG;
    if (M <= 0 || N <= 0 || K <= 0 || M > RS_LINEAR_MAX || N > RS_LINEAR_MAX || K > RS_LINEAR_MAX) return RS_ERR_SHAPE;
    if ((M > 1 && x_row_stride < K) || (N > 1 && w_row_stride < K) || (M > 1 && y_row_stride < N)) return RS_ERR_SHAPE;
    if (((int64_t)M + 127) / 128 * (((int64_t)N + 127) / 128) > (int64_t)(kGridThreads / 256u)) return RS_ERR_SHAPE;    // workgroups of a launch
    if (((uintptr_t)x & 15) || (M > 1 && (x_row_stride & 15)) || ((uintptr_t)w & 15) || (N > 1 && (w_row_stride & 15)) ||
        ((uintptr_t)x_scale & 3) || ((uintptr_t)w_scale & 3) || ((uintptr_t)y & (y_dtype == RS_DTYPE_F32 ? 3 : 1)))
        return RS_ERR_ALIGN;
    const LinearParams p = linear_params(x, x_row_stride, x_scale, w, w_row_stride, w_scale, M, N, K, y, y_row_stride, workspace);
    const hipStream_t st = (hipStream_t)stream;
    const hipError_t e = y_dtype == RS_DTYPE_F32 ? launch_linear<RS_DTYPE_F32>(p, st)
                       : y_dtype == RS_DTYPE_BF16 ? launch_linear<RS_DTYPE_BF16>(p, st) : launch_linear<RS_DTYPE_F16>(p, st);
    return e == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

int rs_linear_rows(const void *x, int32_t x_dtype, int64_t x_row_stride, const void *w, int64_t w_row_stride, const float *w_scale,
                   int32_t M, int32_t N, int32_t K, void *y, int32_t y_dtype, int64_t y_row_stride, void *stream)
{
    if (!x || !w || !w_scale || !y) return RS_ERR_NULL;
    if (!known(x_dtype) || !known(y_dtype)) return RS_ERR_ARG;
    if (M <= 0 || N <= 0 || K <= 0 || M > RS_LINEAR_ROWS_MAX || N > RS_LINEAR_MAX || K > RS_LINEAR_ROWS_COLUMNS_MAX) return RS_ERR_SHAPE;
    if ((N > 1 && w_row_stride < K) || (M > 1 && y_row_stride < N)) return RS_ERR_SHAPE;
    if (((uintptr_t)x & (x_dtype == RS_DTYPE_F32 ? 3 : 1)) || ((uintptr_t)w & 15) || (N > 1 && (w_row_stride & 15)) || ((uintptr_t)w_scale & 3) ||
        ((uintptr_t)y & (y_dtype == RS_DTYPE_F32 ? 3 : 1)))
        return RS_ERR_ALIGN;
    const LinearParams p = linear_params(x, x_row_stride, nullptr, w, w_row_stride, w_scale, M, N, K, y, y_row_stride, nullptr);
    const hipStream_t st = (hipStream_t)stream;
    const hipError_t e = y_dtype == RS_DTYPE_F32 ? launch_rows<RS_DTYPE_F32>(p, x_dtype, st)
                       : y_dtype == RS_DTYPE_BF16 ? launch_rows<RS_DTYPE_BF16>(p, x_dtype, st) : launch_rows<RS_DTYPE_F16>(p, x_dtype, st);
    return e == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

}  // extern "C"
