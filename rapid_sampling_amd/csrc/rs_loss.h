// Cross entropy of tokens under softmax(x w^T / T) without the logits, and its gradients.
//
//   z[m, v] = x_m . w_v     M_m = max_v z[m, v]     S_m = sum_v 2^(c (z[m, v] - M_m)), c = log2(e) / T
//   lse_m = M_m / T + ln S_m                        loss_m = (M_m - z[m, t_m]) / T + ln S_m
//   G[m, v] = ((g_m + h_m) 2^(c (z[m, v] - M_m)) / S_m - g_m [v = t_m]) / T        dx = G w        dw = G^T x
//
// with g the gradient of the losses and h that of the lse.  Forward: a product whose tiles leave a maximum and a sum of each row in
// the place of their logits, and a pass that joins these.  Backward, for a piece of the vocabulary at a time: the piece's product once
// more, with G in the place of the logits, and the two products with it.  Three products are what the gradients cannot do without,
// the fourth is the price of the logits that are not kept.
#pragma once

#include "rs_product.h"
#include "rs_sort.h"

namespace rs {

constexpr uint32_t kFewRows = 32, kCountRows = 2048;         // see G's rounding

struct LossRow {                     // of one row, for G
    float   max, a, b;               // M, (g + h) / (S T), g / T
    int32_t token;
};

struct LossParams {
    Product     a;                   // P: weights, Q: x
    const void *tokens;
    int64_t     token_stride;
    int32_t     tokens_64;
    uint32_t    V, M;                // of the whole call
    uint32_t    v0;                  // the piece's first token
    float       c, inv_t;
    float2     *parts;               // [stretches of the vocabulary][M]: maximum, sum
    uint32_t    n_parts;
    float      *target;              // z of the row's token
    float      *loss, *lse;
    float2     *stats;               // maximum, sum; kept for the gradient
    const float *g, *h;
    int32_t     g_stride, h_stride;
    LossRow    *rows;
    float      *scale;               // null, or [0] what G is multiplied with, [1] what the products are
    void       *grad;                // G: rows of grad_stride bytes
    uint32_t    grad_stride;
    uint32_t    rest;                // 0, or rows from one of G to what its rounding left, rounded too
    const float *sums;               // [share of the reduction][M][sum_stride] of the product, where it is shared out
    uint32_t    sum_stride, shares;
    float      *hit;                 // null, or what G's rounding left at each row's token
    const uint2 *order;              // null, or (token, row), by token and row
    uint32_t   *starts;              // ... and the first place of a token from kStretch s on, for every s
    uint32_t    n_starts;
};
constexpr uint32_t kStretch = 64, kNoToken = 1u << 20;

__device__ __forceinline__ int64_t loss_token(const LossParams &p, uint32_t m)
{
    return p.tokens_64 ? ((const int64_t *)p.tokens)[(int64_t)m * p.token_stride] : ((const int32_t *)p.tokens)[(int64_t)m * p.token_stride];
}

// Bound by the product, or for few rows by reading w: 8192 x 131072 x 4096 in bfloat16 6.3 ms (1.40 PFLOP/s), 1 x 65536 x 4096 90 us (6.0 TB/s).
template <class T>
__global__ __launch_bounds__(T::kThreads, 2) void loss_tile_kernel(LossParams p)
{
    extern __shared__ char lds[];
    T tile;
    tile.choose(p.a, blockIdx.x);
    typename T::Acc acc;
    tile.make(p.a, 0, lds, acc);
    const uint32_t V = p.V, stretch = tile.n0 / (16u * T::NU) + wave_id() % T::WN;
    const bool whole = (stretch + 1u) * (16u * T::NU) <= V;
#pragma unroll
    for (int t = 0; t < T::MT; ++t) {
        const uint32_t m = tile.m(t);
        const int64_t token = m < p.M ? loss_token(p, m) : -1;
        float top = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < T::NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[u][t][j] = whole || tile.n(u) + j < V ? acc[u][t][j] : -__builtin_inff();
                top = fmaxf(top, acc[u][t][j]);
            }
        // (few stretches hold the token of any of their rows)
        const bool here = token >= 0 && token < (int64_t)V && (uint32_t)token / (16u * T::NU) == stretch;
        if (__any(here)) {
            float z = 0.0f;
            bool mine = false;
#pragma unroll
            for (int u = 0; u < T::NU; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool it = here && tile.n(u) + j == (uint32_t)token;
                    z = it ? acc[u][t][j] : z;
                    mine = mine || it;
                }
            if (mine) p.target[m] = z;
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float from = top == -__builtin_inff() ? 0.0f : top;
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < T::NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) s += __builtin_amdgcn_exp2f((acc[u][t][j] - from) * p.c);
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (m < p.M && threadIdx.x % 64u < 16u && stretch < p.n_parts) p.parts[(size_t)stretch * p.M + m] = make_float2(top, s);
    }
}

__device__ __forceinline__ float2 join_sums(float2 a, float2 b, float c)
{
    const float top = fmaxf(a.x, b.x), from = top == -__builtin_inff() ? 0.0f : top;
    return make_float2(top, a.y * __builtin_amdgcn_exp2f((a.x - from) * c) + b.y * __builtin_amdgcn_exp2f((b.x - from) * c));
}

// The row's results, from its maximum, its sum, and the logit of its token if it has one.
__device__ __forceinline__ void finish_row(const LossParams &p, uint32_t m, float2 sum, float target)
{
    const bool none = sum.x == -__builtin_inff() && sum.y == 0.0f;             // no logit above -inf
    const float ln_s = none ? 0.0f : 0.693147180559945309f * __builtin_log2f(sum.y);
    const int64_t token = loss_token(p, m);
    p.lse[m] = none ? -__builtin_inff() : sum.x * p.inv_t + ln_s;
    float loss = 0.0f;
    if (token >= (int64_t)p.V) loss = __builtin_nanf("");
    else if (token >= 0) loss = none ? __builtin_inff() : (sum.x - target) * p.inv_t + ln_s;
    p.loss[m] = loss;
    if (p.stats) p.stats[m] = none ? make_float2(0.0f, __builtin_inff()) : sum;
}

// 2^WIDTH rows to a workgroup, 256 / 2^WIDTH threads to a row (8192 rows of 1024 stretches 60 us, one row 4).
__global__ __launch_bounds__(256) void loss_join_kernel(LossParams p, uint32_t width)
{
    __shared__ float2 held[256];
    const uint32_t m = (blockIdx.x << width) + (threadIdx.x & ((1u << width) - 1u)), k = threadIdx.x >> width, many = 256u >> width;
    float2 sum = make_float2(-__builtin_inff(), 0.0f);
    if (m < p.M)
        for (uint32_t s = k; s < p.n_parts; s += many) sum = join_sums(sum, p.parts[(size_t)s * p.M + m], p.c);
    held[threadIdx.x] = sum;
    for (uint32_t d = 128u; d >= 1u << width; d >>= 1) {
        __syncthreads();
        if (threadIdx.x < d) held[threadIdx.x] = join_sums(held[threadIdx.x], held[threadIdx.x + d], p.c);
    }
    if (!k && m < p.M) finish_row(p, m, held[threadIdx.x], p.target[m]);
}

// Where the product has few tiles and a long reduction, workgroups share it out and leave sums (loss_dx_kernel); there are few logits then, and
// these take up where the tiles end otherwise.  The logits from column v on, a multiple of 4:
__device__ __forceinline__ v4f shared_sums(const LossParams &p, uint32_t m, uint32_t v)
{
    const float *at = p.sums + (int64_t)m * p.sum_stride + v;
    v4f z = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (uint32_t k = 0; k < p.shares; ++k) z += *(const v4f *)(at + (int64_t)k * p.M * p.sum_stride);
    return z;
}
// Forward: a workgroup to kShared columns of a row (with the product, 64 x 1000 x 4096 in bfloat16, 11.4 us; by tiles alone 31.8).
constexpr uint32_t kShared = 1024;
__global__ __launch_bounds__(256) void loss_shares_kernel(LossParams p)
{
    __shared__ float2 held[256];
    __shared__ float target;
    const uint32_t m = blockIdx.y, v = blockIdx.x * kShared + threadIdx.x * 4u;
    const int64_t token = loss_token(p, m);
    float2 sum = make_float2(-__builtin_inff(), 0.0f);
    if (v < p.V) {
        const v4f z = shared_sums(p, m, v);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (v + j >= p.V) break;
            sum = join_sums(sum, make_float2(z[j], 1.0f), p.c);
            if ((int64_t)(v + j) == token) p.target[m] = target = z[j];
        }
    }
    held[threadIdx.x] = sum;
    for (uint32_t d = 128u; d; d >>= 1) {
        __syncthreads();
        if (threadIdx.x < d) held[threadIdx.x] = join_sums(held[threadIdx.x], held[threadIdx.x + d], p.c);
    }
    if (threadIdx.x) return;
    if (gridDim.x > 1u) p.parts[(size_t)blockIdx.x * p.M + m] = held[0];
    else finish_row(p, m, held[0], target);
}

// ---------------------------------------------------------------- gradients --
// G in 16 bits is rounded, to bfloat16 with 8 bits of its own size; in float16 it is made so large first (by a power of two, the same
// for the whole call) that the largest possible is below 2^15, and a probability's share of it is lost from 2^-39 on.  That would add to the
// gradients' own rounding another of its size (a row's or a column's many are off in all directions: 1.41 times as much in all).  So what the
// rounding left is made up for.  Of up to kFewRows rows (twice as many over less than sixteen times as many tokens) all of it is kept, as
// rows of their own behind G's: the products are then of twice as many rows, and wait for memory all the same (forward and gradients of 1 row
// of 4096 over 131072 in bfloat16 876 us without, 890 with; of 48 rows it would be 907 and 1012).  Of more rows that of each row at its own
// token, the largest of the row as long as it is not learnt, is added to the two products' sums (loss_round_kernel, add_hits): errors are 1.00 to 1.05 times
// the result's own rounding (1.07 over 100 tokens; 1.03 to 1.14 at a temperature of 0.5, where other tokens have much of a row too).  (us without and with it: 8192 x 131072 x 4096 in bfloat16 28620 and 28750, 4096 x
// 50257 x 1024 in float16 1810 and 1860, 8192 x 8000 x 4096 1840 and 1920, 2000 x 7900 x 4096 476 and 528, 8192 x 512 x 4096 290 and 348.)
__global__ __launch_bounds__(1024) void loss_scale_kernel(LossParams p)
{
    __shared__ float tops[16];
    float top = 0.0f;
    for (uint32_t m = threadIdx.x; m < p.M; m += 1024u) {
        // (what loss_rows_kernel leaves out may not make the others small: the g of a row without a token, and both of one without a finite logit)
        const int64_t token = loss_token(p, m);
        const bool looked_at = token >= 0 && token < (int64_t)p.V;
        const float g = p.g && looked_at ? fabsf(p.g[(int64_t)m * p.g_stride]) : 0.0f, h = p.h ? fabsf(p.h[(int64_t)m * p.h_stride]) : 0.0f;
        const float v = p.stats[m].y < __builtin_inff() ? (g + h) * p.inv_t : 0.0f;
        if (v < __builtin_inff()) top = fmaxf(top, v);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (threadIdx.x % 64u == 0) tops[threadIdx.x / 64u] = top;
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < 16; ++i) top = fmaxf(top, tops[i]);
    const int e = top > 0.0f ? min(max(14 - ((int)(__float_as_uint(top) >> 23) - 127), -100), 100) : 0;
    p.scale[0] = __builtin_ldexpf(1.0f, e);
    p.scale[1] = __builtin_ldexpf(1.0f, -e);
}

// The order of up to kCountRows rows, and then where stretches of the vocabulary begin in it: the number of (token, row) that come before, counted one by one
// by four threads (2000 rows over 32000 tokens 10 us; sorting them would be launches of its own).
__device__ __forceinline__ void loss_order(const LossParams &p, uint2 *order)
{
    __shared__ uint4 held[kCountRows / 4u];
    constexpr uint32_t kRowBits = 11;
    static_assert(kCountRows == 1u << kRowBits, "token (20 bits, or none) and row in 32 bits");
#pragma unroll
    for (uint32_t e = 0; e < kCountRows / 256u; ++e) {
        const uint32_t j = e * 256u + threadIdx.x;
        if (e * 256u >= p.M) break;
        uint32_t pair = 0xFFFFFFFFu;
        if (j < p.M) {
            const int64_t t = loss_token(p, j);
            pair = (t >= 0 && t < (int64_t)p.V ? (uint32_t)t : kNoToken) << kRowBits | j;
        }
        ((uint32_t *)held)[j] = pair;
    }
    __syncthreads();
    const uint32_t row_groups = (p.M + 63u) / 64u, quarter = threadIdx.x % 4u, id = blockIdx.x * 64u + threadIdx.x / 4u;
    const bool is_row = blockIdx.x < row_groups;
    const uint32_t m = is_row ? id : id - row_groups * 64u;                     // or the stretch
    const uint32_t pair = is_row ? ((const uint32_t *)held)[min(m, p.M - 1u)] : (m * kStretch) << kRowBits;
    uint32_t before = 0;
#pragma unroll 4
    for (uint32_t q = quarter; q < (p.M + 3u) / 4u; q += 4u) {
        const uint4 k = held[q];
        before += (k.x < pair) + (k.y < pair) + (k.z < pair) + (k.w < pair);
    }
    before += __shfl_xor(before, 1);
    before += __shfl_xor(before, 2);
    if (quarter) return;
    if (!is_row) {
        if (m < p.n_starts) p.starts[m] = before;
    } else if (m < p.M) order[before] = make_uint2(pair >> kRowBits, m);
}
// More rows are sorted (rs_sort.h), and the stretches' beginnings looked for.
__global__ __launch_bounds__(256) void loss_starts_kernel(LossParams p)
{
    const uint32_t s = blockIdx.x * 256u + threadIdx.x;
    if (s >= p.n_starts) return;
    uint32_t from = 0, to = p.M;                         // the first place whose token is not below is not before `from`, nor behind `to`
    while (from < to) {
        const uint32_t i = (from + to) / 2u, token = p.order[i].x;
        if (token < p.V && token < s * kStretch) from = i + 1u;
        else to = i;
    }
    p.starts[s] = from;
}

// (order: null, or where to put it)
__global__ __launch_bounds__(256) void loss_rows_kernel(LossParams p, uint2 *order)
{
    if (order) loss_order(p, order);
    const uint32_t m = blockIdx.x * 256u + threadIdx.x;
    if (m >= p.M) return;
    const float2 st = p.stats[m];
    const int64_t token = loss_token(p, m);
    const float f = p.scale ? p.inv_t * p.scale[0] : p.inv_t, h = p.h ? p.h[(int64_t)m * p.h_stride] : 0.0f;
    float g = p.g && token >= 0 ? p.g[(int64_t)m * p.g_stride] : 0.0f;
    if (p.g && token >= (int64_t)p.V) g = __builtin_nanf("");                  // its loss is NaN
    LossRow r;
    r.max = st.x;
    r.a = (g + h) * f / st.y;
    r.b = st.y == __builtin_inff() ? 0.0f : g * f;
    r.token = token >= 0 && token < (int64_t)p.V ? (int32_t)token : -1;
    p.rows[m] = r;
}

// What is left of a number when it is rounded to 16 bits; nothing of one that is none.
template <int DT> __device__ __forceinline__ float rounding_left(float v)
{
    float d = 0.0f;
    if constexpr (DT == RS_DTYPE_BF16) d = v - (float)(__bf16)v;
    if constexpr (DT == RS_DTYPE_F16) d = v - (float)(_Float16)v;
    return d == d ? d : 0.0f;
}

// (8192 rows, a piece of 8192 tokens, 4096 columns in bfloat16: 401 us, 1.37 PFLOP/s)
template <class T>
__global__ __launch_bounds__(T::kThreads, 2) void loss_grad_kernel(LossParams p)
{
    extern __shared__ char lds[];
    T tile;
    tile.choose(p.a, blockIdx.x);
    typename T::Acc acc;
    tile.make(p.a, 0, lds, acc);
    const uint32_t from = p.v0 + tile.n0 + wave_id() % T::WN * (16u * T::NU);             // the wave's first token
    auto row_of = [&](int t, v4f (&v)[T::NU]) {
        const LossRow r = p.rows[min(tile.m(t), p.M - 1u)];
#pragma unroll
        for (int u = 0; u < T::NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][j] = r.a * __builtin_amdgcn_exp2f((acc[u][t][j] - r.max) * p.c);
        // (few waves have the token of any of their rows)
        if (!__any((uint32_t)r.token - from < 16u * T::NU)) return;
#pragma unroll
        for (int u = 0; u < T::NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if ((int32_t)(tile.n(u) + p.v0 + j) == r.token) {
                    v[u][j] -= r.b;
                    if (T::DT != RS_DTYPE_F32 && p.hit && tile.m(t) < p.M) p.hit[tile.m(t)] = rounding_left<T::DT>(v[u][j]);
                }
    };
    if constexpr (T::DT == RS_DTYPE_F32) {
#pragma unroll
        for (int t = 0; t < T::MT; ++t) {
            v4f v[T::NU];
            row_of(t, v);
            const uint32_t m = tile.m(t);
            if (m < p.M)
#pragma unroll
                for (int u = 0; u < T::NU; ++u) store_row<T::DT>((char *)p.grad + (int64_t)m * p.grad_stride, 0, tile.n(u), p.a.p.rows, v[u]);
        }
    } else {
        const TileStore<T::DT, T> out(lds);
#pragma unroll
        for (int t = 0; t < T::MT; ++t) {
            v4f v[T::NU];
            row_of(t, v);
            out.put(t, v);
        }
        out.flush(tile, p.grad, p.grad_stride / 2u, p.M, p.a.p.rows);
        if constexpr (T::kTileM <= kFewRows * 2u) {
            if (!p.rest) return;
#pragma unroll
            for (int t = 0; t < T::MT; ++t) {
                v4f v[T::NU];
                row_of(t, v);
#pragma unroll
                for (int u = 0; u < T::NU; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[u][j] = rounding_left<T::DT>(v[u][j]);
                out.put(t, v);
            }
            out.flush(tile, (char *)p.grad + (int64_t)p.rest * p.grad_stride, p.grad_stride / 2u, p.M, p.a.p.rows);
        }
    }
}

// The same from shared-out sums: four columns to a thread.
template <int DT>
__global__ __launch_bounds__(256) void loss_shares_grad_kernel(LossParams p)
{
    const uint32_t m = blockIdx.y, v = blockIdx.x * kShared + threadIdx.x * 4u;
    if (v >= p.V) return;
    const LossRow r = p.rows[m];
    v4f g = shared_sums(p, m, v);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        g[j] = r.a * __builtin_amdgcn_exp2f((g[j] - r.max) * p.c);
        if ((int32_t)(v + j) == r.token) {
            g[j] -= r.b;
            if (p.hit) p.hit[m] = rounding_left<DT>(g[j]);
        }
    }
    char *row = (char *)p.grad + (int64_t)m * p.grad_stride;
    store_row<DT>(row, 0, v, p.V, g);
    if constexpr (DT != RS_DTYPE_F32) {
        if (!p.rest) return;
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = rounding_left<DT>(g[j]);
        store_row<DT>(row + (int64_t)p.rest * p.grad_stride, 0, v, p.V, g);
    }
}

struct GradParams {
    Product      a;                  // P: the output's columns, Q: its rows
    void        *y;                  // (rows, columns)
    int64_t      y_stride;           // elements
    const float *scale;              // null, or [1]: factor of the result
    int32_t      add;                // to what is there
    int64_t      part_stride;        // elements between the sums of the workgroups that share the reduction
    const float *hit;                // dw: null, or as in LossParams, with x and the piece's first token
    const uint2 *order;
    const uint32_t *starts;
    uint32_t     n_starts, v0;
    Operand      x;
};

// dx's sums of one piece of the vocabulary, in float32; every share of the reduction has sums of its own.  (The same piece: 458 us, 1.2 PFLOP/s.  w's
// rows are turned by their reads from LDS, two in the place of one.)
template <class T>
__global__ __launch_bounds__(T::kThreads, 2) void loss_dx_kernel(GradParams p)
{
    extern __shared__ char lds[];
    T tile;
    const uint32_t part = tile.choose(p.a, blockIdx.x);
    typename T::Acc acc;
    tile.make(p.a, part, lds, acc);
    float *y = (float *)p.y + (int64_t)part * p.part_stride;
#pragma unroll
    for (int t = 0; t < T::MT; ++t) {
        const uint32_t m = tile.m(t);
        if (m >= p.a.q.rows) continue;
#pragma unroll
        for (int u = 0; u < T::NU; ++u) {
            const uint32_t n = tile.n(u);
            v4f v = acc[u][t];
            float *at = y + (int64_t)m * p.y_stride;
            if (p.add) {
                if (n + 4u <= p.a.p.rows) { v4f old; __builtin_memcpy(&old, at + n, 16); v += old; }
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j) if (n + j < p.a.p.rows) v[j] += at[n + j];
            }
            store_row<RS_DTYPE_F32>(at, 0, n, p.a.p.rows, v);
        }
    }
}

template <int DT> __device__ __forceinline__ float widen16(uint32_t v)
{
    if constexpr (DT == RS_DTYPE_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)v);
    else return __uint_as_float(v << 16);
}

// What G's rounding left at the tokens of a tile of dw, added to its sums: for the rows whose token the tile holds, which lie side by side in the rows' order,
// stages more of the same product, of those rows of x and a G that is 0 but at each row's token.  What is left is rounded as well, and what that leaves,
// from a second such G: all of float32's 24 bits.  Half a stage for up to 32 rows; the next 64 are on their way while the last half is multiplied, and where they
// are has been read before.  (Places behind the last row hold it once more, with a G of 0: an x that is no number has made its column of the tile none already.)
template <class T> __device__ __forceinline__ void add_hits(const GradParams &p, const T &tile, char *lds, typename T::Acc &acc)
{
    constexpr uint32_t kX = T::P::kBytes, kG = T::Q::kBytes, kLoads = T::P::kLoads, kMany = T::kRed;
    static_assert(2u * kX + 2u * kG <= T::kLds && kMany == 64u && T::kTileM % kStretch == 0u, "where the stages were");
    const uint32_t s = (p.v0 + tile.m0) / kStretch;
    const uint32_t first = p.starts[s], last = p.starts[min(s + T::kTileM / kStretch, p.n_starts - 1u)];
    if (first >= last) return;
    char *const g_at = lds + 2u * kX;
    const typename T::P::Reader rp(wave_id() % T::WN * (16u * T::NU));
    const typename T::Q::Reader rq(wave_id() / T::WN * (16u * T::MT));
    // the thread's pieces of 16 bytes of x's rows, as far as the rows go; what the last one holds behind a row's end belongs to columns that are not there
    uint32_t rows[kLoads];
    auto pair_of = [&](uint32_t e) { return p.order[min(e, last - 1u)]; };
    auto ask = [&](uint32_t e0) {
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            uint32_t e, byte;
            T::P::source_of(T::P::place(i), e, byte);
            rows[i] = pair_of(e0 + e).y;
        }
    };
    auto fetch = [&](char *to) {
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            uint32_t e, byte;
            T::P::source_of(T::P::place(i), e, byte);
            const uint32_t k = tile.n0 * 2u + byte;
            const char *from = p.x.at + (int64_t)rows[i] * p.x.stride + (k < p.a.p.rows * 2u ? k : 0u);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (LdsPtr)(to + (i * T::kWaves + wave_id()) * 1024u), 16, 0, 0);
        }
    };
    // a row of G to a thread: (token, row), what is left there, and its place
    const uint32_t lane = threadIdx.x % kMany;
    uint2 pair = pair_of(first + lane), next = pair_of(first + kMany + lane);
    auto place_of = [&](uint32_t token) { return T::Q::place_of(lane, (token - p.v0 - tile.m0) * 2u); };
    auto set = [&](uint32_t at, float v) {
        put<T::DT>(g_at + at, 0, v);
        put<T::DT>(g_at + kG + at, 0, rounding_left<T::DT>(v));
    };
    ask(first);
    float left = p.hit[pair.y];
    stage_barrier<0>();
    for (uint32_t i = threadIdx.x * 16u; i < 2u * kG; i += T::kThreads * 16u) *(v4i *)(g_at + i) = v4i{0, 0, 0, 0};
    fetch(lds);
    ask(first + kMany);
    stage_barrier<0>();
    uint32_t now = 0;
    for (uint32_t e0 = first; ; e0 += kMany) {
        const uint32_t many = min(last - e0, kMany), at = place_of(pair.x);
        if (threadIdx.x < many) set(at, left);
        stage_barrier<0>();
        v4i x[T::NU], g[T::MT], rest[T::MT];
        auto read = [&](int half) {
#pragma unroll
            for (int u = 0; u < T::NU; ++u) x[u] = rp(lds + now, u, half);
#pragma unroll
            for (int t = 0; t < T::MT; ++t) { g[t] = rq(g_at, t, half); rest[t] = rq(g_at + kG, t, half); }
        };
        auto multiply_read = [&]() {
            multiply_all<T::DT>(x, g, acc);
            multiply_all<T::DT>(x, rest, acc);
        };
        read(0);
        if (many > kMany / 2u) {
            multiply_read();
            read(1);
        }
        if (e0 + kMany < last) fetch(lds + (now ^ kX));
        ask(e0 + 2u * kMany);
        pair = next;
        left = p.hit[pair.y];
        next = pair_of(e0 + 2u * kMany + lane);
        asm volatile("" ::: "memory");                           // (asked for before the products, not behind them)
        multiply_read();
        if (e0 + kMany >= last) return;
        now ^= kX;
        stage_barrier<63>();                                     // all have read G, and x may still be on its way
        if (threadIdx.x < kMany) set(at, 0.0f);
    }
}

// dw of one piece, whole.  (The same piece: 470 us; both operands are turned.)
template <class T>
__global__ __launch_bounds__(T::kThreads, 2) void loss_dw_kernel(GradParams p)
{
    extern __shared__ char lds[];
    T tile;
    tile.choose(p.a, blockIdx.x);
    typename T::Acc acc;
    tile.make(p.a, 0, lds, acc);
    const float f = p.scale ? p.scale[1] : 1.0f;
    if constexpr (T::DT != RS_DTYPE_F32) if (p.hit) add_hits(p, tile, lds, acc);
    if constexpr (T::DT == RS_DTYPE_F32) {
#pragma unroll
        for (int t = 0; t < T::MT; ++t) {
            const uint32_t m = tile.m(t);
            if (m < p.a.q.rows)
#pragma unroll
                for (int u = 0; u < T::NU; ++u) store_row<T::DT>(p.y, (int64_t)m * p.y_stride, tile.n(u), p.a.p.rows, acc[u][t] * f);
        }
    } else {
        const TileStore<T::DT, T> out(lds);
#pragma unroll
        for (int t = 0; t < T::MT; ++t) {
            v4f v[T::NU];
#pragma unroll
            for (int u = 0; u < T::NU; ++u) v[u] = acc[u][t] * f;
            out.put(t, v);
        }
        out.flush(tile, p.y, p.y_stride, p.a.q.rows, p.a.p.rows);
    }
}

// dx (rows, K) from the sums of the shares, and what G's rounding left at the token, rounded once
struct RoundParams {
    const float   *sums;
    int64_t        part_stride, count;
    void          *y;
    const float   *scale, *hit;      // hit: null, or as in LossParams
    const LossRow *rows;
    Operand        w;
    uint32_t       parts, K;
};
template <int DT>
__global__ __launch_bounds__(256) void loss_round_kernel(RoundParams p)
{
    const float f = p.scale ? p.scale[1] : 1.0f;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < p.count; i += (int64_t)gridDim.x * 1024) {
        v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
        const bool whole = i + 4 <= p.count;
        if (whole) {
#pragma unroll 8
            for (uint32_t k = 0; k < p.parts; ++k) {
                v4f v;
                __builtin_memcpy(&v, p.sums + k * p.part_stride + i, 16);        // (part_stride is any number)
                s += v;
            }
        } else
#pragma unroll
            for (int j = 0; j < 4; ++j)
                for (uint32_t k = 0; i + j < p.count && k < p.parts; ++k) s[j] += p.sums[k * p.part_stride + i + j];
        if (DT != RS_DTYPE_F32 && p.hit) {
            int64_t m = p.count >> 32 ? i / p.K : (uint32_t)i / p.K;
            uint32_t k = (uint32_t)(i - m * p.K);
            auto row_of = [&](int32_t token) { return (const uint16_t *)(p.w.at + (int64_t)token * p.w.stride); };
            if (k + 4u <= p.K) {
                const int32_t token = p.rows[m].token;
                if (token >= 0) {
                    uint2 w;
                    __builtin_memcpy(&w, row_of(token) + k, 8);
                    const float left = p.hit[m];
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[j] += left * widen16<DT>((j < 2 ? w.x : w.y) >> (16 * (j % 2)) & 0xFFFFu);
                }
            } else
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int32_t token = i + j < p.count ? p.rows[m].token : -1;
                    if (token >= 0) s[j] += p.hit[m] * widen16<DT>(row_of(token)[k]);
                    if (++k == p.K) { k = 0; ++m; }
                }
        }
        s *= f;
        if (whole) put_four<DT>(p.y, i, s);
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) if (i + j < p.count) put<DT>(p.y, i + j, s[j]);
    }
}

// Rows laid out in multiples of 16 bytes, for those that are not (or, `source` of them, several times over): 16 bytes to a thread.
__global__ __launch_bounds__(256) void lay_out_rows_kernel(const char *x, int64_t x_stride, char *y, int64_t y_stride, int64_t rows, int64_t source, uint32_t bytes)
{
    const uint32_t pieces = (uint32_t)(y_stride / 16);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * pieces; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / pieces;
        const char *from = x + (r < source ? r : r - source) * x_stride;
        const uint32_t at = (uint32_t)(i - r * pieces) * 16u;
        v4i v = {0, 0, 0, 0};
        if (at + 16u <= bytes) __builtin_memcpy(&v, from + at, 16);
        else {
            uint16_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) if (at + 2u * j < bytes) w[j] = *(const uint16_t *)(from + at + 2u * j);
            __builtin_memcpy(&v, w, 16);
        }
        *(v4i *)(y + r * y_stride + at) = v;
    }
}

}  // namespace rs
