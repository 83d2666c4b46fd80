// Instantiations, launchers and C entry points of the cross entropy over a vocabulary without its logits.
#include "rs_loss.h"

namespace rs {

static uint32_t size_of(int32_t dtype) { return dtype == RS_DTYPE_F32 ? 4 : 2; }

// Where a call's scratch lies.  The same sizes give the same places.
struct LossSpace {
    uint64_t parts = 0, target = 0;                     // forward
    uint64_t scale = 0, rows = 0, grad = 0, dx = 0;     // backward
    uint64_t twice = 0;                                 // x's rows two times over
    uint32_t high = 0;                                  // rows of G: x's, or twice as many (see loss_scale_kernel)
    uint64_t bytes = 0;
    uint32_t piece = 0, split = 1;                      // tokens of a piece; shares of dx's reduction
    uint64_t grad_stride = 0;
    uint32_t shares = 1;                                // of the product's reduction
    uint64_t sums = 0, sum_stride = 0;
    uint64_t hit = 0, order = 0, starts = 0;
    SortSpace sort = {};                                // of more than kCountRows rows, in the place of order
    uint32_t n_starts = 0;                              // 0: what G's rounding leaves at the tokens is not made up for by itself
    uint64_t take(uint64_t n) { const uint64_t at = bytes; bytes += up(n, 256); return at; }
};

// dx has few tiles: where those of 256 x 256 do not go round, others, whose reduction over the piece is shared out among up to two workgroups
// to a compute unit (385 rows of 2000 and a piece of 50257 in float16: 128 x 64 164 us, 128 x 128 111).
static TileSize dx_size(uint64_t rows, uint64_t columns) { return rows <= 64 ? kSmall : tiles_of(rows, columns, 256, 256) >= 192 ? kLarge : kMiddle; }

// Workgroups that share a tile of x w^T: where the tiles leave much of the chip idle and a tile's columns take long.  (Forward, and with gradients, us, in
// one and shared.  bfloat16: 64 x 1000 x 4096 31.8, 77.5 and 11.4, 39.0; 4 x 16000 x 4096 31.4, 120 and 29.6, 116; 64 x 1000 x 1024 14.7,
// 40.2 and 10.4, 35.4; of 188 tiles, 64 x 24000 x 4096, 35.7, 172 and 43.2, 193.  float32, whose tiles take four times as long: 64 x 1000 x 4096 148, 321
// and 18.8, 62.1; 64 x 8000 x 1024 44.5, 118 and 23.9, 77.8; of 188 tiles 156, 511 and 127, 483; of 243, 64 x 31000 x 1024, 45.7, 171 and
// 44.1, 170, with products that took up to 3 % less than they do.)
static uint32_t product_shares(uint64_t M, uint64_t V, uint64_t K, int32_t dtype)
{
    const uint64_t tiles = tiles_of(M, V, 64, 128);
    if (tiles >= (dtype == RS_DTYPE_F32 ? 256 : 128)) return 1;
    return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({512 / tiles, K * size_of(dtype) / kRowBytes / 8, 32}));
}

// A piece of the vocabulary: 128 MB of G, half of the last cache, in steps of 256 tokens and at least 8192, so that the sums of dx that each piece reads and
// writes again (8 bytes) are little next to its products.  For many rows the piece's weights stay there with it (8192 tokens of 4096 columns are 64 MB); for
// up to a few hundred the piece is most of the vocabulary or all of it, and weights beyond the cache are read from memory by each of the products.
static LossSpace loss_space(int32_t M, int32_t V, int32_t K, int32_t dtype, bool backward)
{
    LossSpace s;
    const uint64_t size = size_of(dtype);
    s.shares = product_shares(M, V, K, dtype);
    if (s.shares > 1) {
        s.sum_stride = up(V, 4);
        s.sums = s.take(s.shares * s.sum_stride * M * 4);
    }
    if (!backward) {
        s.parts = s.take((up(V, 64) / 64) * (uint64_t)M * sizeof(float2));
        s.target = s.take((uint64_t)M * 4);
        return s;
    }
    s.high = (M <= (int32_t)kFewRows || (M <= (int32_t)(2 * kFewRows) && 16 * M > V)) && dtype != RS_DTYPE_F32 ? 2 * M : M;
    if (s.high > (uint32_t)M) s.twice = s.take(s.high * up((uint64_t)K * size, 16));
    else if (dtype != RS_DTYPE_F32) {
        s.n_starts = (uint32_t)(up(V, kStretch) / kStretch) + 1;
        s.hit = s.take((uint64_t)M * 4);
        if (M <= (int32_t)kCountRows) s.order = s.take((uint64_t)M * 8);
        else s.sort = sort_space((uint32_t)M, (uint32_t)V, s.bytes);
        s.starts = s.take((uint64_t)s.n_starts * 4);
    }
    s.scale = s.take(8);
    s.rows = s.take((uint64_t)M * sizeof(LossRow));
    s.piece = (uint32_t)std::min<uint64_t>(up(V, 256), std::max<uint64_t>(8192, ((1ull << 27) / (s.high * size)) / 256 * 256));
    s.grad_stride = s.piece * size + 256;              // (not a power of two: rows would share their memory channels)
    s.grad = s.take((uint64_t)s.high * s.grad_stride);
    const TileSize tile = dx_size(s.high, K);
    const uint64_t tiles = tile == kLarge ? tiles_of(s.high, K, 256, 256) : tiles_of(s.high, K, tile == kMiddle ? 128 : 64, 128), stages = s.piece * size / kRowBytes;
    s.split = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({(tile == kLarge ? 256 : 512) / tiles, stages / 8, 32}));
    s.dx = s.take((uint64_t)s.split * s.high * K * 4);
    return s;
}

// 256 x 256 by eight waves (2 x 4 of them, and 4 x 2 in dx of 16 bits, whose first operand alone costs two reads from LDS for a
// fragment: 540 us for a piece of 8192 tokens with 8192 rows of 4096, and 512), 128 x 128 and 128 x 64 by four.
template <int DT, bool TP, bool TQ> constexpr bool kTurned = TP && !TQ && DT != RS_DTYPE_F32;
template <int DT, bool TP, bool TQ>
using LargeTile = Tile<DT, TP, TQ, !TP && DT != RS_DTYPE_F32, kTurned<DT, TP, TQ> ? 4 : 2, kTurned<DT, TP, TQ> ? 2 : 4, kTurned<DT, TP, TQ> ? 4 : 8, kTurned<DT, TP, TQ> ? 8 : 4, 2>;
template <int DT, bool TP, bool TQ> using MiddleTile = Tile<DT, TP, TQ, !TP && DT != RS_DTYPE_F32, 2, 2, 4, 4, 2>;
template <int DT, bool TP, bool TQ> using SmallTile = Tile<DT, TP, TQ, !TP && DT != RS_DTYPE_F32, 2, 2, 4, 2, 3>;

// float32 and up to 16 rows: 128 x 16 by two waves, which take a row of x apart once for four of w's and make no products for rows that are not there.
// (Forward, and with gradients, us, 128 x 64 and so: 1 x 50000 x 1024 57.6, 219 and 44.1, 183; 16 x 24000 x 4096 112, 414 and 93, 378; 16 x 100000 x 4096
// 417, 1544 and 342, 1325, with products that took up to 3 % less.  128 x 32 for up to 32 rows would save 2 to 10 of 100 more.)
constexpr uint32_t kNarrowRows = 16;
template <int DT, bool TP, bool TQ> using NarrowTile = Tile<DT, TP, TQ, false, 2, 1, 4, 1, 4>;
static bool narrow(int32_t dtype, uint32_t rows) { return dtype == RS_DTYPE_F32 && rows <= kNarrowRows; }

template <class T, class K, class A> static void launch_tiles(K kernel, const A &p, hipStream_t st)
{
    const uint64_t tiles = (uint64_t)((p.a.q.rows + T::kTileM - 1) / T::kTileM) * ((p.a.p.rows + T::kTileN - 1) / T::kTileN);
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(tiles * p.a.split)), dim3(T::kThreads), T::kLds, st, p);
}

// (instantiated by name: the compiler leaves some of those that are only launched without their host side)
#define RS_KERNELS(DT, TILE)                                                                                            \
    template __global__ void loss_tile_kernel<TILE<DT, false, false>>(LossParams);                                      \
    template __global__ void loss_grad_kernel<TILE<DT, false, false>>(LossParams);                                      \
    template __global__ void loss_dx_kernel<TILE<DT, true, false>>(GradParams);                                         \
    template __global__ void loss_dw_kernel<TILE<DT, true, true>>(GradParams);
#define RS_TYPES(TILE) RS_KERNELS(RS_DTYPE_F32, TILE) RS_KERNELS(RS_DTYPE_BF16, TILE) RS_KERNELS(RS_DTYPE_F16, TILE)
#define RS_SHARED(DT)                                                                                                   \
    template __global__ void loss_dx_kernel<SmallTile<DT, false, false>>(GradParams);                                   \
    template __global__ void loss_shares_grad_kernel<DT>(LossParams);
RS_SHARED(RS_DTYPE_F32) RS_SHARED(RS_DTYPE_BF16) RS_SHARED(RS_DTYPE_F16)
template __global__ void loss_tile_kernel<NarrowTile<RS_DTYPE_F32, false, false>>(LossParams);
template __global__ void loss_grad_kernel<NarrowTile<RS_DTYPE_F32, false, false>>(LossParams);
template __global__ void loss_dx_kernel<NarrowTile<RS_DTYPE_F32, false, false>>(GradParams);
template __global__ void loss_dx_kernel<NarrowTile<RS_DTYPE_F32, true, false>>(GradParams);
RS_TYPES(SmallTile)
RS_TYPES(MiddleTile)
RS_TYPES(LargeTile)

#define RS_LAUNCH(size, kernel, TP, TQ)                                                                                 \
    switch (size(p.a.q.rows, p.a.p.rows)) {                                                                             \
    case kLarge:  launch_tiles<LargeTile<DT, TP, TQ>>(kernel<LargeTile<DT, TP, TQ>>, p, st); break;                     \
    case kMiddle: launch_tiles<MiddleTile<DT, TP, TQ>>(kernel<MiddleTile<DT, TP, TQ>>, p, st); break;                   \
    default:      launch_tiles<SmallTile<DT, TP, TQ>>(kernel<SmallTile<DT, TP, TQ>>, p, st); break;                     \
    }
#define RS_NARROW(kernel, TP, TQ)                                                                                       \
    if constexpr (DT == RS_DTYPE_F32)                                                                                   \
        if (narrow(DT, p.a.q.rows)) return launch_tiles<NarrowTile<DT, TP, TQ>>(kernel<NarrowTile<DT, TP, TQ>>, p, st);
template <int DT> static void launch_forward(const LossParams &p, hipStream_t st)
{
    RS_NARROW(loss_tile_kernel, false, false)
    RS_LAUNCH(tile_size, loss_tile_kernel, false, false)
}
template <int DT> static void launch_grad(const LossParams &p, hipStream_t st)
{
    RS_NARROW(loss_grad_kernel, false, false)
    RS_LAUNCH(tile_size, loss_grad_kernel, false, false)
}
template <int DT> static void launch_dx(const GradParams &p, hipStream_t st)
{
    RS_NARROW(loss_dx_kernel, true, false)
    RS_LAUNCH(dx_size, loss_dx_kernel, true, false)
}
// (for few rows dw is all stores, and two workgroups to a compute unit hide more of them: 48 rows of 4096 over 131072 in bfloat16 1083 us with
// its forward pass, 966 so; 385 rows of 2000 over 50257 the same either way)
template <int DT> static void launch_dw(const GradParams &p, hipStream_t st)
{
    if (p.a.red <= 256) launch_tiles<MiddleTile<DT, true, true>>(loss_dw_kernel<MiddleTile<DT, true, true>>, p, st);
    else RS_LAUNCH(tile_size, loss_dw_kernel, true, true)
}

template <int DT> static void launch_product(const GradParams &p, hipStream_t st)
{
    RS_NARROW(loss_dx_kernel, false, false)
    launch_tiles<SmallTile<DT, false, false>>(loss_dx_kernel<SmallTile<DT, false, false>>, p, st);
}

// The product's sums by shares of its reduction.
template <int DT> static void launch_shares(LossParams &p, const LossSpace &s, char *ws, hipStream_t st)
{
    GradParams g = {};
    g.a = p.a;
    g.a.split = s.shares;
    g.y = ws + s.sums;
    g.y_stride = (int64_t)s.sum_stride;
    g.part_stride = (int64_t)s.sum_stride * p.M;
    launch_product<DT>(g, st);
    p.sums = (const float *)(ws + s.sums);
    p.sum_stride = (uint32_t)s.sum_stride;
    p.shares = s.shares;
}

static bool known(int32_t dtype) { return dtype == RS_DTYPE_F32 || dtype == RS_DTYPE_BF16 || dtype == RS_DTYPE_F16; }

static int check(const void *x, int64_t x_stride, const void *w, int64_t w_stride, int32_t dtype, const void *tokens, int32_t tokens_64, int32_t M, int32_t V,
                 int32_t K, double temperature, const void *workspace)
{
    if (!x || !w || !tokens || !workspace) return RS_ERR_NULL;
    if (!known(dtype) || (tokens_64 != 0 && tokens_64 != 1)) return RS_ERR_ARG;
    if (M <= 0 || V <= 0 || K <= 0 || M > RS_LINEAR_MAX || V > 1048576 || K > RS_LOSS_COLUMNS_MAX) return RS_ERR_SHAPE;
    // workgroups of a launch, of 256 threads (those of 512 make tiles four times as large)
    const uint64_t most = kGridThreads / 256u;
    if (tiles_of(M, V, 64, 128) > most || tiles_of(M, K, 64, 128) > most || tiles_of(V, K, 128, 128) > most) return RS_ERR_SHAPE;
    if (!(temperature >= 0.001 && temperature <= 1000)) return RS_ERR_TEMPERATURE;
    const int64_t size = size_of(dtype), far = kTileStride / size;
    if ((M > 1 && (x_stride < K || x_stride > far)) || (V > 1 && (w_stride < K || w_stride > far))) return RS_ERR_SHAPE;
    if (((uintptr_t)x & 15) || ((uintptr_t)w & 15) || (M > 1 && (x_stride * size & 15)) || (V > 1 && (w_stride * size & 15)) ||
        ((uintptr_t)tokens & (tokens_64 ? 7 : 3)))
        return RS_ERR_ALIGN;
    return RS_OK;
}

// (the distance to the next row of a single one is not looked at by the checks)
static Operand rows_of(const void *x, int64_t stride, int32_t rows, int32_t K, uint32_t size)
{
    return Operand{(const char *)x, (uint32_t)(rows > 1 ? stride * size : up((uint64_t)K * size, 16)), (uint32_t)rows};
}

static void launch_lay_out(const void *x, int64_t x_bytes, void *y, int64_t y_bytes, int64_t rows, int64_t source, uint32_t bytes, hipStream_t st)
{
    const uint64_t groups = ((uint64_t)rows * (y_bytes / 16) + 255) / 256;
    hipLaunchKernelGGL(lay_out_rows_kernel, dim3((uint32_t)std::min<uint64_t>(groups, 1u << 16)), dim3(256), 0, st, (const char *)x, x_bytes, (char *)y, y_bytes, rows,
                       source, bytes);
}

template <int DT>
static void backward(LossParams p, const LossSpace &s, Operand x, Operand w, uint32_t K, void *grad_x, void *grad_w, char *ws, hipStream_t st)
{
    constexpr uint32_t size = kSize<DT>;
    if (DT == RS_DTYPE_F16) hipLaunchKernelGGL(loss_scale_kernel, dim3(1), dim3(1024), 0, st, p);
    else p.scale = nullptr;
    uint2 *counted = nullptr;
    if (s.n_starts) {
        p.hit = (float *)(ws + s.hit);
        if (grad_w) {
            p.starts = (uint32_t *)(ws + s.starts); p.n_starts = s.n_starts;
            if (p.M <= kCountRows) p.order = counted = (uint2 *)(ws + s.order);
            else {
                p.order = launch_sort(TokenList{p.tokens, p.token_stride, p.tokens_64}, p.M, p.V, s.sort, ws, nullptr, 0, st);
                hipLaunchKernelGGL(loss_starts_kernel, dim3((p.n_starts + 255) / 256), dim3(256), 0, st, p);
            }
        }
    }
    hipLaunchKernelGGL(loss_rows_kernel, dim3(counted ? (p.M + 63) / 64 + (p.n_starts + 63) / 64 : (p.M + 255) / 256), dim3(256), 0, st, p, counted);
    Operand xs = x;
    if (s.high > p.M) {
        p.rest = p.M;
        if (grad_w) {
            xs = Operand{ws + s.twice, (uint32_t)up((uint64_t)K * size, 16), s.high};
            launch_lay_out(x.at, x.stride, (char *)ws + s.twice, xs.stride, s.high, p.M, K * size, st);
        }
    }
    for (uint32_t v0 = 0; v0 < p.V; v0 += s.piece) {
        const uint32_t n = std::min(s.piece, p.V - v0);
        const char *piece = w.at + (int64_t)v0 * w.stride;
        p.v0 = v0;
        p.a = Product{Operand{piece, w.stride, n}, x, K, 1};
        if (s.shares > 1) {
            launch_shares<DT>(p, s, ws, st);
            hipLaunchKernelGGL(loss_shares_grad_kernel<DT>, dim3((p.V + kShared - 1) / kShared, p.M), dim3(256), 0, st, p);
        } else launch_grad<DT>(p, st);
        GradParams g = {};
        g.scale = p.scale;
        if (grad_x) {
            g.a = Product{Operand{piece, w.stride, K}, Operand{(const char *)p.grad, p.grad_stride, s.high}, n, s.split};
            g.y = ws + s.dx;
            g.y_stride = K;
            g.part_stride = (int64_t)s.high * K;
            g.add = v0 > 0;
            launch_dx<DT>(g, st);
        }
        if (grad_w) {
            g.a = Product{Operand{xs.at, xs.stride, K}, Operand{(const char *)p.grad, p.grad_stride, n}, s.high, 1};
            g.y = (char *)grad_w + (int64_t)v0 * K * size;
            g.y_stride = K;
            g.part_stride = 0;
            g.add = 0;
            g.hit = p.hit; g.order = p.order; g.starts = p.starts; g.n_starts = p.n_starts; g.v0 = v0; g.x = x;
            launch_dw<DT>(g, st);
        }
    }
    if (grad_x) {
        RoundParams r = {};
        r.count = (int64_t)p.M * K;
        r.sums = (const float *)(ws + s.dx); r.part_stride = r.count; r.parts = s.split * (s.high / p.M);
        r.y = grad_x; r.scale = p.scale; r.hit = p.hit; r.rows = p.rows; r.w = w; r.K = K;
        hipLaunchKernelGGL(loss_round_kernel<DT>, dim3((uint32_t)std::min<int64_t>((r.count + 1023) / 1024, 1 << 16)), dim3(256), 0, st, r);
    }
}

}  // namespace rs

using namespace rs;

extern "C" {

int rs_lay_out_rows(const void *x, int64_t x_row_stride, int32_t size, int64_t R, int32_t K, void *y, int64_t y_row_stride, void *stream)
{
    if (!x || !y) return RS_ERR_NULL;
    if (size != 2 && size != 4) return RS_ERR_ARG;
    if (R <= 0 || K <= 0 || K > RS_LINEAR_MAX || x_row_stride < 0 || y_row_stride < K || R > (1ll << 40) / y_row_stride) return RS_ERR_SHAPE;
    if (((uintptr_t)x & (size - 1)) || ((uintptr_t)y & 15) || (y_row_stride * size & 15)) return RS_ERR_ALIGN;
    launch_lay_out(x, x_row_stride * size, y, y_row_stride * size, R, R, (uint32_t)(K * size), (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

size_t rs_linear_cross_entropy_workspace_bytes(int32_t M, int32_t V, int32_t K, int32_t dtype, int32_t backward)
{
    if (M <= 0 || V <= 0 || K <= 0 || !known(dtype)) return 0;
    return loss_space(M, V, K, dtype, backward != 0).bytes;
}

int rs_linear_cross_entropy(const void *x, int64_t x_stride, const void *w, int64_t w_stride, int32_t dtype, const void *tokens, int32_t tokens_64,
                            int64_t token_stride, int32_t M, int32_t V, int32_t K, double temperature, float *loss, float *lse, float *stats, void *workspace,
                            size_t workspace_bytes, void *stream)
{
    const int rc = check(x, x_stride, w, w_stride, dtype, tokens, tokens_64, M, V, K, temperature, workspace);
    if (rc != RS_OK) return rc;
    if (!loss || !lse) return RS_ERR_NULL;
    if (((uintptr_t)loss & 3) || ((uintptr_t)lse & 3) || ((uintptr_t)stats & 7)) return RS_ERR_ALIGN;
    const uint32_t size = size_of(dtype);
    const LossSpace s = loss_space(M, V, K, dtype, false);
    if (workspace_bytes < s.bytes || ((uintptr_t)workspace & 255)) return RS_ERR_WORKSPACE;
    char *ws = (char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    LossParams p = {};
    p.a = Product{rows_of(w, w_stride, V, K, size), rows_of(x, x_stride, M, K, size), (uint32_t)K, 1};
    p.tokens = tokens; p.token_stride = token_stride; p.tokens_64 = tokens_64;
    p.V = (uint32_t)V; p.M = (uint32_t)M;
    p.c = (float)(1.4426950408889634 / temperature); p.inv_t = (float)(1.0 / temperature);
    p.parts = (float2 *)(ws + s.parts); p.target = (float *)(ws + s.target);
    p.loss = loss; p.lse = lse; p.stats = (float2 *)stats;
    if (s.shares > 1) {
        if (dtype == RS_DTYPE_F32) launch_shares<RS_DTYPE_F32>(p, s, ws, st);
        else if (dtype == RS_DTYPE_BF16) launch_shares<RS_DTYPE_BF16>(p, s, ws, st);
        else launch_shares<RS_DTYPE_F16>(p, s, ws, st);
        p.n_parts = (p.V + kShared - 1) / kShared;
        hipLaunchKernelGGL(loss_shares_kernel, dim3(p.n_parts, p.M), dim3(256), 0, st, p);
        if (p.n_parts == 1) return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
    } else {
        const uint32_t stretch = tile_size(M, V) == kLarge ? 128 : 64;
        p.n_parts = (p.V + stretch - 1) / stretch;
        if (dtype == RS_DTYPE_F32) launch_forward<RS_DTYPE_F32>(p, st);
        else if (dtype == RS_DTYPE_BF16) launch_forward<RS_DTYPE_BF16>(p, st);
        else launch_forward<RS_DTYPE_F16>(p, st);
    }
    uint32_t width = 0;                                  // rows of a workgroup: as many as leave every compute unit one
    while (width < 6 && ((uint32_t)M >> (width + 1)) >= 256) ++width;
    hipLaunchKernelGGL(loss_join_kernel, dim3(((uint32_t)M + (1u << width) - 1) >> width), dim3(256), 0, st, p, width);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

int rs_linear_cross_entropy_backward(const void *x, int64_t x_stride, const void *w, int64_t w_stride, int32_t dtype, const void *tokens, int32_t tokens_64,
                                     int64_t token_stride, int32_t M, int32_t V, int32_t K, double temperature, const float *stats,
                                     const float *grad_loss, int32_t grad_loss_stride, const float *grad_lse, int32_t grad_lse_stride,
                                     void *grad_x, void *grad_w, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = check(x, x_stride, w, w_stride, dtype, tokens, tokens_64, M, V, K, temperature, workspace);
    if (rc != RS_OK) return rc;
    if (!stats || (!grad_x && !grad_w)) return RS_ERR_NULL;
    if ((grad_loss_stride | grad_lse_stride) & ~1) return RS_ERR_ARG;
    const uint32_t size = size_of(dtype);
    if (((uintptr_t)stats & 7) || ((uintptr_t)grad_loss & 3) || ((uintptr_t)grad_lse & 3) || ((uintptr_t)grad_x & (size - 1)) || ((uintptr_t)grad_w & (size - 1)))
        return RS_ERR_ALIGN;
    const LossSpace s = loss_space(M, V, K, dtype, true);
    if (workspace_bytes < s.bytes || ((uintptr_t)workspace & 255)) return RS_ERR_WORKSPACE;
    char *ws = (char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    const Operand q = rows_of(x, x_stride, M, K, size), r = rows_of(w, w_stride, V, K, size);
    LossParams p = {};
    p.tokens = tokens; p.token_stride = token_stride; p.tokens_64 = tokens_64;
    p.V = (uint32_t)V; p.M = (uint32_t)M;
    p.c = (float)(1.4426950408889634 / temperature); p.inv_t = (float)(1.0 / temperature);
    p.stats = (float2 *)stats;
    p.g = grad_loss; p.g_stride = grad_loss_stride; p.h = grad_lse; p.h_stride = grad_lse_stride;
    p.scale = (float *)(ws + s.scale); p.rows = (LossRow *)(ws + s.rows);
    p.grad = ws + s.grad; p.grad_stride = (uint32_t)s.grad_stride;
    if (dtype == RS_DTYPE_F32) backward<RS_DTYPE_F32>(p, s, q, r, (uint32_t)K, grad_x, grad_w, ws, st);
    else if (dtype == RS_DTYPE_BF16) backward<RS_DTYPE_BF16>(p, s, q, r, (uint32_t)K, grad_x, grad_w, ws, st);
    else backward<RS_DTYPE_F16>(p, s, q, r, (uint32_t)K, grad_x, grad_w, ws, st);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

}  // extern "C"
