// Values in 8 bits (e4m3fn) with a float32 scale for each block of 128 along the rows, and their matrix product:
//
//   scale = max(max |x| over the block * r, 2^-126), r = 1/448 in float32        q = e4m3(x / scale), to nearest, ties to even
//   y[m, n] = sum over blocks kb of sx[m, kb] sw[n / 128, kb] sum_{k in kb} qx[m, k] qw[n, k]
//
// The inner sums are the matrix cores' (products of two such values are exact in float32, the sum over a block is held in
// float32); the scales are applied to them in float32, and so is the outer sum.  One rounding to y's type at the end.
#pragma once

#include "rs_common.h"

namespace rs {

constexpr int kFpBlock = 128;

typedef int   v8i __attribute__((ext_vector_type(8)));
typedef int   v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

struct QuantParams {
    const void *x;
    int64_t     x_stride;                // elements from a row to the next
    uint8_t    *q;
    int64_t     q_stride;                // bytes; the bytes from K to the stride's end are cleared up to q_cols
    float      *scale;
    uint32_t    R, K, blocks, q_cols;
};

struct LinearParams {
    const uint8_t *x, *w;
    int64_t        x_stride, w_stride, y_stride;
    const float   *x_scale, *w_scale;
    void          *y;
    uint32_t       M, N, K, blocks;
};

template <int DT> __device__ __forceinline__ float widen(const void *p, int64_t i)
{
    if constexpr (DT == RS_DTYPE_F32) return ((const float *)p)[i];
    else if constexpr (DT == RS_DTYPE_BF16) return __uint_as_float((uint32_t)((const uint16_t *)p)[i] << 16);
    else return (float)((const _Float16 *)p)[i];
}
template <int DT> __device__ __forceinline__ void put(void *p, int64_t i, float v)
{
    if constexpr (DT == RS_DTYPE_F32) ((float *)p)[i] = v;
    else if constexpr (DT == RS_DTYPE_BF16) ((__bf16 *)p)[i] = (__bf16)v;
    else ((_Float16 *)p)[i] = (_Float16)v;
}

__device__ __forceinline__ float block_scale(float peak) { return fmaxf(peak * (1.0f / 448.0f), 0x1p-126f); }

// One block of 1 x 128: sixteen lanes, eight values each.
template <int DT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantParams p)
{
    const uint32_t i = blockIdx.x * 16u + threadIdx.x / 16u, part = threadIdx.x % 16u;
    const bool live = i < p.R * (uint64_t)p.blocks;
    const uint32_t r = live ? i / p.blocks : 0, kb = live ? i - r * p.blocks : 0;
    const uint32_t k0 = kb * kFpBlock + part * 8u;
    float x[8], peak = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = live && k0 + j < p.K ? widen<DT>(p.x, (int64_t)r * p.x_stride + k0 + j) : 0.0f;
        peak = fmaxf(peak, fabsf(x[j]));
    }
#pragma unroll
    for (int d = 8; d; d >>= 1) peak = fmaxf(peak, __shfl_xor(peak, d));
    const float scale = block_scale(peak);
    if (!live) return;
    if (part == 0) p.scale[(size_t)r * p.blocks + kb] = scale;
    if (k0 >= p.q_cols) return;
    uint2 q;
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] / scale, x[1] / scale, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] / scale, x[3] / scale, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] / scale, x[5] / scale, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] / scale, x[7] / scale, hi, true);
    q.x = (uint32_t)lo; q.y = (uint32_t)hi;
    *(uint2 *)(p.q + (int64_t)r * p.q_stride + k0) = q;      // q_cols is a multiple of 8
}

// One block of 128 x 128: a workgroup, two threads to a row.
template <int DT>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(QuantParams p)
{
    __shared__ float peaks[4];
    const uint32_t rb = blockIdx.x / p.blocks, kb = blockIdx.x - rb * p.blocks;
    const uint32_t r = rb * kFpBlock + threadIdx.x / 2u, k0 = kb * kFpBlock + threadIdx.x % 2u * 64u;
    const int64_t at = (int64_t)r * p.x_stride + k0;
    float peak = 0.0f;
    for (uint32_t j = 0; j < 64; ++j) if (r < p.R && k0 + j < p.K) peak = fmaxf(peak, fabsf(widen<DT>(p.x, at + j)));
#pragma unroll
    for (int d = 32; d; d >>= 1) peak = fmaxf(peak, __shfl_xor(peak, d));
    if (threadIdx.x % 64 == 0) peaks[threadIdx.x / 64] = peak;
    __syncthreads();
    const float scale = block_scale(fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3])));
    if (threadIdx.x == 0) p.scale[(size_t)rb * p.blocks + kb] = scale;
    if (r >= p.R) return;
    for (uint32_t j = 0; j < 64 && k0 + j < p.q_cols; j += 2) {
        const float a = k0 + j < p.K ? widen<DT>(p.x, at + j) : 0.0f, b = k0 + j + 1 < p.K ? widen<DT>(p.x, at + j + 1) : 0.0f;
        *(uint16_t *)(p.q + (int64_t)r * p.q_stride + k0 + j) = (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(a / scale, b / scale, 0, false);
    }
}

// 16 bytes of a row from column k on; columns from K on read as 0.
__device__ __forceinline__ v4i load16(const uint8_t *row, uint32_t k, uint32_t K)
{
    v4i v = {0, 0, 0, 0};
    if (k + 16u <= K) v = *(const v4i *)(row + k);
    else if (k < K) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) if (k + j < K) w[j / 4] |= (uint32_t)row[k + j] << (8 * (j % 4));
        v = v4i{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    }
    return v;
}

__device__ __forceinline__ v8i join(v4i a, v4i b) { return v8i{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }

// Eight values of 8 bits as bfloat16, which holds every one of them.
__device__ __forceinline__ v8bf widen8(int lo, int hi)
{
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 16 x 16 sums over a block of 128.  Lane l gives 32 bytes of row l % 16 of either side (any 32 of the block's columns, as
// long as both sides agree) and has the sums of w's rows 4 (l / 16) + 0..3 with x's row l % 16.
//
// The matrix instructions that take 8 bits do not hold their sums in 32: of the eight products that are added at once, what lies
// 14 binades and more under the largest is dropped (256 * 256 + 4 is 65536; measured 3.1e-5 of a result's size over
// 4096 random columns).  Those that take bfloat16 keep 24 bits (1.0e-7), at half the rate.
__device__ __forceinline__ v4f block_product(v8i w, v8i x)
{
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(w[2 * i], w[2 * i + 1]), widen8(x[2 * i], x[2 * i + 1]), acc, 0, 0, 0);
    return acc;
}

// The same on the matrix cores' 8-bit instructions: for outputs of 16 bits, whose own rounding is fifty times as large.
__device__ __forceinline__ v4f block_product_8(v8i w, v8i x)
{
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, zero, 0, 0, 0, 0, 0, 0);
}

// Four consecutive float32 values, or eight of 16 bits, in one store.
template <int DT> __device__ __forceinline__ void put_wide(void *p, int64_t i, v4f a, v4f b)
{
    if constexpr (DT == RS_DTYPE_F32) *(v4f *)((float *)p + i) = a;
    else if constexpr (DT == RS_DTYPE_BF16) {
        v8bf v;
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = (__bf16)a[j]; v[j + 4] = (__bf16)b[j]; }
        *(v8bf *)((__bf16 *)p + i) = v;
    } else {
        v8h v;
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = (_Float16)a[j]; v[j + 4] = (_Float16)b[j]; }
        *(v8h *)((_Float16 *)p + i) = v;
    }
}

// A wave per 16 rows of w and 16 MT rows of x.
template <int DT, int MT>
__global__ __launch_bounds__(256) void linear_kernel(LinearParams p)
{
    const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u;
    const uint32_t n0 = (blockIdx.x * 4u + wave) * 16u, m0 = blockIdx.y * (16u * MT);
    if (n0 >= p.N) return;
    const uint32_t i = lane % 16u, part = lane / 16u;
    const uint8_t *wr = p.w + (int64_t)min(n0 + i, p.N - 1u) * p.w_stride;
    v4f acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t kb = 0; kb < p.blocks; ++kb) {
        const uint32_t k = kb * kFpBlock + part * 32u;
        const v8i w = join(load16(wr, k, p.K), load16(wr, k + 16u, p.K));
        const float sw = p.w_scale[(size_t)(n0 / kFpBlock) * p.blocks + kb];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const uint32_t m = min(m0 + t * 16u + i, p.M - 1u);
            const uint8_t *xr = p.x + (int64_t)m * p.x_stride;
            const v4f s = block_product(w, join(load16(xr, k, p.K), load16(xr, k + 16u, p.K)));
            const float f = sw * p.x_scale[(size_t)m * p.blocks + kb];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[t][j] = __builtin_fmaf(s[j], f, acc[t][j]);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const uint32_t m = m0 + t * 16u + i;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t n = n0 + part * 4u + j;
            if (n < p.N) put<DT>(p.y, (int64_t)m * p.y_stride + n, acc[t][j]);
        }
    }
}

// -------------------------------------------------------------- many rows --
// A workgroup of eight waves makes 256 rows of w x 64 MT rows of x, a wave 128 x 16 MT of it: a quarter of w's rows in a lane's
// reach would not do, since every block has to be scaled in the vector unit before it is added (four sums a lane and
// 16 x 16 product), so the sums sit in ordinary registers, 32 MT of them.
//
// A block of 128 columns is one stage: rows of 128 bytes go from memory to LDS without passing through registers, while
// the stage before is multiplied.  The eight 16-byte pieces of a row are stored in an order that depends on the row
// (place = piece ^ f(row)), so that the eight rows read at once lie in different banks.  The first operand's rows are
// dealt so that a lane's sums are 32 consecutive columns of y.
typedef __attribute__((address_space(1))) const void *GlobalPtr;
typedef __attribute__((address_space(3))) void *LdsPtr;

constexpr int kTileN = 256;
constexpr int64_t kTileStride = (1ll << 32) / 256 - kFpBlock;

__device__ __forceinline__ uint32_t w_turn(uint32_t row) { return (row & 3u) | ((row >> 3) & 4u); }
__device__ __forceinline__ uint32_t x_turn(uint32_t row) { return row & 7u; }

template <int DT, int MT, bool EXACT>
struct LinearTile {
    static constexpr uint32_t kTileM = 64 * MT, kRows = kTileN + kTileM, kStage = kRows * kFpBlock;
    static constexpr uint32_t kLoads = kRows / 64;           // 16-byte pieces of a stage per thread

    // A wave fills eight rows of a stage with one load: thread's row and piece of load i, w's rows first.
    static __device__ __forceinline__ uint32_t row_of(uint32_t i) { return (i * 8u + threadIdx.x / 64u) * 8u + threadIdx.x % 64u / 8u; }

    struct Source {
        const uint8_t *w, *x;            // of the tile's first rows
        uint32_t       at[kLoads];       // bytes from there to the thread's pieces of the first block
    };
    static __device__ __forceinline__ Source source(const LinearParams &p, uint32_t n0, uint32_t m0)
    {
        Source s;
        s.w = p.w + (int64_t)n0 * p.w_stride;
        s.x = p.x + (int64_t)m0 * p.x_stride;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const bool is_w = i < kTileN / 64;
            const uint32_t r = row_of(i) - (is_w ? 0u : kTileN);
            const uint32_t piece = (threadIdx.x & 7u) ^ (is_w ? w_turn(r) : x_turn(r));
            s.at[i] = (is_w ? min(r, p.N - 1u - n0) * (uint32_t)p.w_stride : min(r, p.M - 1u - m0) * (uint32_t)p.x_stride) + piece * 16u;
        }
        return s;
    }
    static __device__ __forceinline__ void fill(const LinearParams &p, const Source &s, uint32_t n0, uint32_t m0, uint32_t kb, uint8_t *lds)
    {
        const uint32_t k = kb * kFpBlock;
        if (k + kFpBlock <= p.K) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i)
                __builtin_amdgcn_global_load_lds((GlobalPtr)((i < kTileN / 64 ? s.w : s.x) + k + s.at[i]), (LdsPtr)(lds + (i * 8u + threadIdx.x / 64u) * 1024u), 16, 0, 0);
            return;
        }
        // the last block where K is no whole number of them
#pragma unroll 1
        for (uint32_t i = 0; i < kLoads; ++i) {
            const bool is_w = i < kTileN / 64;
            const uint32_t r = row_of(i) - (is_w ? 0u : kTileN);
            const uint32_t piece = (threadIdx.x & 7u) ^ (is_w ? w_turn(r) : x_turn(r));
            const uint8_t *from = is_w ? s.w + min(r, p.N - 1u - n0) * p.w_stride : s.x + min(r, p.M - 1u - m0) * p.x_stride;
            *(v4i *)(lds + row_of(i) * kFpBlock + (threadIdx.x & 7u) * 16u) = load16(from, k + piece * 16u, p.K);
        }
    }

    static __device__ __forceinline__ v8i fragment(const uint8_t *lds, uint32_t row, uint32_t turn, uint32_t part)
    {
        const uint8_t *r = lds + row * kFpBlock;
        return join(*(const v4i *)(r + ((part ^ turn) * 16u)), *(const v4i *)(r + (((part + 4u) ^ turn) * 16u)));
    }

    static __device__ __forceinline__ void step(const LinearParams &p, const Source &source, uint32_t n0, uint32_t m0, uint32_t next,
                                                const uint8_t *__restrict now_lds, uint8_t *__restrict next_lds, const float (&f)[MT], v4f (&acc)[8][MT])
    {
        if (next < p.blocks) fill(p, source, n0, m0, next, next_lds);
        const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u, i = lane % 16u, part = lane / 16u;
        const uint32_t wn = (wave & 1u) * 128u, wm = (wave >> 1) * (16u * MT);
        v8i x[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const uint32_t r = wm + t * 16u + i;
            x[t] = fragment(now_lds + kTileN * kFpBlock, r, x_turn(r), part);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const uint32_t r = wn + i / 4u * 32u + u * 4u + i % 4u;
            const v8i w = fragment(now_lds, r, w_turn(r), part);
            v4f s[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) s[t] = EXACT ? block_product(w, x[t]) : block_product_8(w, x[t]);
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[u][t][j] = __builtin_fmaf(s[t][j], f[t], acc[u][t][j]);
        }
    }
};

template <int DT, int MT, bool EXACT>
__global__ __launch_bounds__(512, 2) void linear_tile_kernel(LinearParams p)
{
    using L = LinearTile<DT, MT, EXACT>;
    extern __shared__ uint8_t lds[];
    // Workgroup b runs on XCD b % 8: each XCD takes a stretch of the tiles, in panels of eight rows of tiles, so that the 32 tiles
    // it works on at a time share their rows in its L2.
    const uint32_t tm = (p.M + L::kTileM - 1u) / L::kTileM, tn = (p.N + kTileN - 1u) / kTileN, tiles = tm * tn;
    const uint32_t each = tiles / 8u, rest = tiles % 8u, xcd = blockIdx.x % 8u;
    const uint32_t id = xcd * each + min(xcd, rest) + blockIdx.x / 8u;
    const uint32_t panel = id / (8u * tn), high = min(8u, tm - panel * 8u), in = id - panel * 8u * tn;
    const uint32_t m0 = (panel * 8u + in % high) * L::kTileM, n0 = in / high * kTileN;

    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u, i = lane % 16u, part = lane / 16u;
    const uint32_t wn = (wave & 1u) * 128u, wm = (wave >> 1) * (16u * MT);
    const float *sw = p.w_scale + (size_t)min((n0 + wn) / kFpBlock, (p.N - 1u) / kFpBlock) * p.blocks;
    const float *sx[MT];
    v4f acc[8][MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        sx[t] = p.x_scale + (size_t)min(m0 + wm + t * 16u + i, p.M - 1u) * p.blocks;
#pragma unroll
        for (int u = 0; u < 8; ++u) acc[u][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const typename L::Source source = L::source(p, n0, m0);
    L::fill(p, source, n0, m0, 0, lds);
    for (uint32_t kb = 0; kb < p.blocks; ++kb) {
        float f[MT];
        const float s = sw[kb];
#pragma unroll
        for (int t = 0; t < MT; ++t) f[t] = sx[t][kb] * s;
        wait_vmem();
        __syncthreads();
        const bool odd = kb & 1u;
        L::step(p, source, n0, m0, kb + 1u, lds + (odd ? L::kStage : 0u), lds + (odd ? 0u : L::kStage), f, acc);
    }
    // a lane has columns wn + 32 part .. + 31 of its rows of y
    const uint32_t n = n0 + wn + part * 32u;
    constexpr uint32_t kVec = DT == RS_DTYPE_F32 ? 4 : 8;
    const bool wide = n + 32u <= p.N && !(p.y_stride % kVec) && !((uintptr_t)p.y & 15);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const uint32_t m = m0 + wm + t * 16u + i;
        if (m >= p.M) continue;
        const int64_t at = (int64_t)m * p.y_stride + n;
        if (wide) {
#pragma unroll
            for (int u = 0; u < 8; u += kVec / 4) put_wide<DT>(p.y, at + u * 4, acc[u][t], acc[(u + 1) % 8][t]);
        } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) if (n + u * 4u + j < p.N) put<DT>(p.y, at + u * 4 + j, acc[u][t][j]);
        }
    }
}

}  // namespace rs
