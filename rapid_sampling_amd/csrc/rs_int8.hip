// Instantiations, launchers and C entry points of the product in 8-bit integers.
#include "rs_int8.h"

namespace rs {

// As many rows at a time as a launch holds; a wave to a row of up to 2048 columns, a workgroup to a longer one.
template <int DT, int LANES, int PIECES> static void launch_rows(Int8Rows p, hipStream_t st)
{
    constexpr uint32_t kRows = 256u / LANES, kMost = kGridThreads / 256u;
    const uint32_t R = p.R, most = (uint32_t)std::min<uint64_t>(R, (uint64_t)kMost * kRows);
    for (uint32_t done = 0; done < R; done += p.R) {
        p.R = std::min(most, R - done);
        hipLaunchKernelGGL((int8_rows_kernel<DT, LANES, PIECES>), dim3((p.R + kRows - 1) / kRows), dim3(256), 0, st, p);
        p.x = (const char *)p.x + (int64_t)p.R * p.x_stride * kSize<DT>;
        p.q += (int64_t)p.R * p.q_stride;
        p.scale += p.R;
    }
}
template <int DT> static void launch_rows(const Int8Rows &p, hipStream_t st)
{
    if (p.K <= 512) launch_rows<DT, 64, 1>(p, st);
    else if (p.K <= 2048) launch_rows<DT, 64, 4>(p, st);
    else launch_rows<DT, 256, 4>(p, st);
}

// Workgroups that round x for themselves: three to a compute unit at a time (1 row, weights beyond the caches: 65536 x 2048 33.7 us with one to
// each stretch of w, 31.7 with two to a compute unit, 28.7 with three; 65536 x 4096 53.0, 48.8 and 48.1; 65536 x 8192 105, 104.7 and 104).
constexpr uint32_t kAtATime = 768;

template <int DT, int XT, int NT> static void launch_few(const Int8Params &p, hipStream_t st)
{
    const uint32_t blocks = (p.K + 127) / 128, waves = blocks >= 8 ? 8 : blocks >= 4 ? 4 : blocks >= 2 ? 2 : 1;
    const uint32_t lds = XT < 0 ? 0 : p.M * blocks * 128, stretches = (p.N + 16 * NT - 1) / (16 * NT);
    hipLaunchKernelGGL((int8_few_kernel<DT, XT, NT>), dim3(XT < 0 ? stretches : std::min(stretches, kAtATime), (p.M + 15) / 16), dim3(64 * waves), lds, st, p);
}
template <int DT, int XT> static void launch_few(const Int8Params &p, hipStream_t st)
{
    if (p.N <= 8192) launch_few<DT, XT, 1>(p, st);
    else launch_few<DT, XT, 2>(p, st);
}
template <int DT> static void launch_few(const Int8Params &p, int32_t x_dtype, hipStream_t st)
{
    if (x_dtype == RS_DTYPE_F32) launch_few<DT, RS_DTYPE_F32>(p, st);
    else if (x_dtype == RS_DTYPE_BF16) launch_few<DT, RS_DTYPE_BF16>(p, st);
    else launch_few<DT, RS_DTYPE_F16>(p, st);
}

template <int DT, int WN, int WM, int NU, int MT, int STAGES, bool SPLIT> static void launch_tiles(Int8Params p, hipStream_t st)
{
    using T = Int8Tile<DT, WN, WM, NU, MT, STAGES>;
    const uint64_t tiles = (uint64_t)((p.M + T::kTileM - 1) / T::kTileM) * ((p.N + T::kTileN - 1) / T::kTileN);
    p.a.split = SPLIT ? (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({kPartTiles / tiles, (p.K + 127) / 128 / 4, 8})) : 1;
    hipLaunchKernelGGL((int8_tile_kernel<DT, WN, WM, NU, MT, STAGES, SPLIT>), dim3((uint32_t)(tiles * p.a.split)), dim3(T::kThreads), T::kLds, st, p);
}

// (instantiated by name: the compiler leaves some of those that are only launched without their host side)
#define RS_KERNELS(DT)                                                                     \
    template __global__ void int8_tile_kernel<DT, 2, 4, 8, 4, 2, false>(Int8Params);        \
    template __global__ void int8_tile_kernel<DT, 2, 2, 4, 4, 2, false>(Int8Params);        \
    template __global__ void int8_tile_kernel<DT, 2, 2, 4, 2, 3, true>(Int8Params);
RS_KERNELS(RS_DTYPE_F32)
RS_KERNELS(RS_DTYPE_BF16)
RS_KERNELS(RS_DTYPE_F16)

static bool near(const Int8Params &p) { return p.x_stride <= kTileStride && p.w_stride <= kTileStride; }

template <int DT> static void launch_product(const Int8Params &p, hipStream_t st)
{
    // Sixteen rows by sixteen of w, whose whole rows a workgroup reads and with nothing to join, where there are no more of them than the chip has
    // places for and not many columns; up to 16 rows w is read once all the same, but the tiles' loads, whole lines of 128 bytes, read a large
    // one faster.  (us, weights beyond the caches, few against tiles.  1, 16 rows, K = 4096: N = 4096 6.8, 7.3 and 13.9, 14.1; 16384 17.1, 19.4
    // and 21.2, 19.8; 65536 54.4, 67 and 52.8, 52.6; 16 rows, K = 14336: N = 4096 18.6 and 21, 8192 37.6 and 28.  32, 64 rows, K = 1024: N = 4096
    // 5.3, 7.0 and 8.3, 8.3; 8192 7.7, 12.2 and 8.9, 8.9; K = 4096: 1024 6.7, 6.7 and 12, 12; 4096 12.1, 21.2 and 14.7, 14.7; K = 14336, 17
    // rows: 4096 32.8 and 21.)  (The tiles' kernel reaches its rows with 32 bits.)
    const uint64_t blocks = tiles_of(p.M, p.N, 16, 16), most = blocks * p.K;
    if ((p.M <= 16 ? most <= 96u << 16 : blocks <= 1024 && most <= 32u << 16) || !near(p)) return launch_few<DT, -1>(p, st);
    // Where there are few tiles they are small ones, and their columns are shared out.
    const TileSize size = tiles_of(p.M, p.N, 128, 128) < 192 ? kSmall : tile_size(p.M, p.N);
    if (size == kLarge) launch_tiles<DT, 2, 4, 8, 4, 2, false>(p, st);
    else if (size == kMiddle) launch_tiles<DT, 2, 2, 4, 4, 2, false>(p, st);
    else launch_tiles<DT, 2, 2, 4, 2, 3, true>(p, st);
}

static Int8Params int8_params(const void *x, int64_t x_stride, const float *x_scale, const int8_t *w, int64_t w_stride, const float *w_scale, int32_t M, int32_t N,
                              int32_t K, void *y, int64_t y_stride, void *workspace)
{
    // (the distance to the next row of a single one is not looked at by the checks)
    const int64_t alone = ((int64_t)K + 15) / 16 * 16;
    Int8Params p = {};
    p.x = x; p.x_stride = M > 1 ? x_stride : alone; p.x_scale = x_scale;
    p.w = w; p.w_stride = N > 1 ? w_stride : alone; p.w_scale = w_scale;
    p.y = y; p.y_stride = y_stride;
    p.M = (uint32_t)M; p.N = (uint32_t)N; p.K = (uint32_t)K;
    p.a = Product{Operand{(const char *)w, (uint32_t)p.w_stride, p.N}, Operand{(const char *)x, (uint32_t)p.x_stride, p.M}, p.K, 1};
    p.arrived = (uint32_t *)workspace;
    p.parts = workspace ? (int *)((char *)workspace + 16 * kPartTiles) : nullptr;
    return p;
}

static bool known(int32_t dtype) { return dtype == RS_DTYPE_F32 || dtype == RS_DTYPE_BF16 || dtype == RS_DTYPE_F16; }

}  // namespace rs

using namespace rs;

extern "C" {

int rs_quantize_rows(const void *x, int32_t dtype, int64_t x_row_stride, int32_t R, int32_t K, int8_t *q, int64_t q_row_stride, float *scale, void *stream)
{
    if (!x || !q || !scale) return RS_ERR_NULL;
    if (!known(dtype)) return RS_ERR_ARG;
    if (R <= 0 || K <= 0 || K > RS_LINEAR_MAX || (R > 1 && x_row_stride < 0)) return RS_ERR_SHAPE;
    if (q_row_stride < K || q_row_stride > RS_LINEAR_MAX) return RS_ERR_SHAPE;
    if (((uintptr_t)x & (dtype == RS_DTYPE_F32 ? 3 : 1)) || ((uintptr_t)q & 15) || (q_row_stride & 15) || ((uintptr_t)scale & 3)) return RS_ERR_ALIGN;
    Int8Rows p;
    p.x = x; p.x_stride = x_row_stride; p.q = q; p.q_stride = q_row_stride; p.scale = scale;
    p.R = (uint32_t)R; p.K = (uint32_t)K;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == RS_DTYPE_F32) launch_rows<RS_DTYPE_F32>(p, st);
    else if (dtype == RS_DTYPE_BF16) launch_rows<RS_DTYPE_BF16>(p, st);
    else launch_rows<RS_DTYPE_F16>(p, st);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

int rs_linear_int8(const int8_t *x, int64_t x_row_stride, const float *x_scale, const int8_t *w, int64_t w_row_stride, const float *w_scale,
                   int32_t M, int32_t N, int32_t K, void *y, int32_t y_dtype, int64_t y_row_stride, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!x || !x_scale || !w || !w_scale || !y || !workspace) return RS_ERR_NULL;
    if (workspace_bytes < rs_linear_workspace_bytes() || ((uintptr_t)workspace & 255)) return RS_ERR_WORKSPACE;
    if (!known(y_dtype)) return RS_ERR_ARG;
    if (M <= 0 || N <= 0 || K <= 0 || M > RS_LINEAR_MAX || N > RS_LINEAR_MAX || K > RS_LINEAR_INT8_COLUMNS_MAX) return RS_ERR_SHAPE;
    if ((M > 1 && x_row_stride < K) || (N > 1 && w_row_stride < K) || (M > 1 && y_row_stride < N)) return RS_ERR_SHAPE;
    if (((int64_t)M + 63) / 64 * (((int64_t)N + 127) / 128) > (int64_t)(kGridThreads / 256u)) return RS_ERR_SHAPE;    // workgroups of a launch
    if (((uintptr_t)x & 15) || (M > 1 && (x_row_stride & 15)) || ((uintptr_t)w & 15) || (N > 1 && (w_row_stride & 15)) ||
        ((uintptr_t)x_scale & 3) || ((uintptr_t)w_scale & 3) || ((uintptr_t)y & (y_dtype == RS_DTYPE_F32 ? 3 : 1)))
        return RS_ERR_ALIGN;
    const Int8Params p = int8_params(x, x_row_stride, x_scale, w, w_row_stride, w_scale, M, N, K, y, y_row_stride, workspace);
    if (!near(p) && M > 1 << 19) return RS_ERR_SHAPE;                                // (the second axis of a launch)
    const hipStream_t st = (hipStream_t)stream;
    if (y_dtype == RS_DTYPE_F32) launch_product<RS_DTYPE_F32>(p, st);
    else if (y_dtype == RS_DTYPE_BF16) launch_product<RS_DTYPE_BF16>(p, st);
    else launch_product<RS_DTYPE_F16>(p, st);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

int rs_linear_int8_rows(const void *x, int32_t x_dtype, int64_t x_row_stride, const int8_t *w, int64_t w_row_stride, const float *w_scale,
                        int32_t M, int32_t N, int32_t K, void *y, int32_t y_dtype, int64_t y_row_stride, void *stream)
{
    if (!x || !w || !w_scale || !y) return RS_ERR_NULL;
    if (!known(x_dtype) || !known(y_dtype)) return RS_ERR_ARG;
    if (M <= 0 || N <= 0 || K <= 0 || M > RS_LINEAR_ROWS_MAX || N > RS_LINEAR_MAX || K > RS_LINEAR_ROWS_COLUMNS_MAX) return RS_ERR_SHAPE;
    if ((N > 1 && w_row_stride < K) || (M > 1 && (y_row_stride < N || x_row_stride < 0))) return RS_ERR_SHAPE;
    if (((uintptr_t)x & (x_dtype == RS_DTYPE_F32 ? 3 : 1)) || ((uintptr_t)w & 15) || (N > 1 && (w_row_stride & 15)) || ((uintptr_t)w_scale & 3) ||
        ((uintptr_t)y & (y_dtype == RS_DTYPE_F32 ? 3 : 1)))
        return RS_ERR_ALIGN;
    const Int8Params p = int8_params(x, x_row_stride, nullptr, w, w_row_stride, w_scale, M, N, K, y, y_row_stride, nullptr);
    const hipStream_t st = (hipStream_t)stream;
    if (y_dtype == RS_DTYPE_F32) launch_few<RS_DTYPE_F32>(p, x_dtype, st);
    else if (y_dtype == RS_DTYPE_BF16) launch_few<RS_DTYPE_BF16>(p, x_dtype, st);
    else launch_few<RS_DTYPE_F16>(p, x_dtype, st);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

}  // extern "C"
