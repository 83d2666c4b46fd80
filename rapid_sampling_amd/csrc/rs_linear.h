// Values in 8 bits (e4m3fn) with a float32 scale for each block of 128 along the rows, and their matrix product:
//
//   scale = max(max |x| over the block * r, 2^-126), r = 1/448 in float32        q = e4m3(x / scale), to nearest, ties to even
//   y[m, n] = sum over blocks kb of sx[m, kb] sw[n / 128, kb] sum_{k in kb} qx[m, k] qw[n, k]
//
// The inner sums are the matrix cores', on bfloat16, which holds every value in 8 bits (see block_product); the scales are applied to
// them in float32, and the outer sum is of float32.  One rounding to y's type at the end.
#pragma once

#include "rs_common.h"
#include "rs_tile.h"

namespace rs {

typedef int   v8i __attribute__((ext_vector_type(8)));
typedef int   v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
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
    const uint8_t *x, *w;                // x in 8 bits, or of another type: then x_scale is null and x_stride counts elements
    int64_t        x_stride, w_stride, y_stride;
    const float   *x_scale, *w_scale;
    void          *y;
    uint32_t       M, N, K, blocks;
    uint32_t       split;                // workgroups that share a tile's blocks of columns
    float         *parts;                // ... their sums, and how many have left theirs, per tile; zero between calls
    uint32_t      *arrived;
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

// x / scale, rounded once: the quotient by way of the reciprocal, and what it is off by divided once more.  Of small blocks both
// are taken 2^64 times as large, which is exact: what the quotient is off by, some 2^-24 of x, would be below float32's range.
// (Compared with the division on the CPU, for every significand of the scale and the five numbers about each point halfway between two
// 8-bit values, 6.7e8 pairs: the same.  Without the larger numbers 1.8 % of them are not at a scale of 2^-126, none from 2^-94 on.)
struct Divisor {
    float up, s, r;
    __device__ __forceinline__ explicit Divisor(float scale)
        : up(scale < 0x1p-60f ? 0x1p64f : 1.0f), s(scale < __builtin_inff() ? scale * up : 0.0f), r(1.0f / (scale * up)) {}
    __device__ __forceinline__ float operator()(float x) const
    {
        x *= up;
        const float q = x * r;
        // (-0 stays one; an infinite scale gives 0 for a finite x, NaN for an infinite one)
        return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-q, s, x), r, q), x);
    }
};
__device__ __forceinline__ uint2 quantize8(const float (&x)[8], float scale)
{
    const Divisor d(scale);
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(d(x[0]), d(x[1]), lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(d(x[2]), d(x[3]), lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(d(x[4]), d(x[5]), hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(d(x[6]), d(x[7]), hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// Eight values of a row from column k on, at any address; 0 from column K on.
template <int DT>
__device__ __forceinline__ void load8(const void *base, int64_t at, uint32_t k, uint32_t K, float (&x)[8])
{
    if (k + 8u <= K) {
        if constexpr (DT == RS_DTYPE_F32) {
            v4f a, b;
            __builtin_memcpy(&a, (const float *)base + at + k, 16);
            __builtin_memcpy(&b, (const float *)base + at + k + 4, 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) { x[j] = a[j]; x[j + 4] = b[j]; }
        } else {
            uint16_t v[8];
            __builtin_memcpy(v, (const uint16_t *)base + at + k, 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = DT == RS_DTYPE_BF16 ? __uint_as_float((uint32_t)v[j] << 16) : (float)__builtin_bit_cast(_Float16, v[j]);
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) x[j] = k + j < K ? widen<DT>(base, at + k + j) : 0.0f;
    }
}
__device__ __forceinline__ float largest8(const float (&x)[8])
{
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[j]));
    return m;
}
// Largest over 16 lanes, in all of them.
template <int CTRL> __device__ __forceinline__ float turn_max(float v)
{
    return fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float max16(float v)
{
    return turn_max<0x121>(turn_max<0x122>(turn_max<0x124>(turn_max<0x128>(v))));       // row_ror 8, 4, 2, 1
}

// One block of 1 x 128: sixteen lanes, eight values each.
template <int DT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantParams p)
{
    const uint32_t i = blockIdx.x * 16u + threadIdx.x / 16u, part = threadIdx.x % 16u;
    const bool live = i < (uint64_t)p.R * p.blocks;
    const uint32_t r = live ? i / p.blocks : 0, kb = live ? i - r * p.blocks : 0;
    const uint32_t k0 = kb * kFpBlock + part * 8u;
    float x[8];
    load8<DT>(p.x, (int64_t)r * p.x_stride, k0, p.K, x);
    const float scale = block_scale(max16(largest8(x)));
    if (!live) return;
    if (part == 0) p.scale[(size_t)r * p.blocks + kb] = scale;
    if (k0 < p.q_cols) *(uint2 *)(p.q + (int64_t)r * p.q_stride + k0) = quantize8(x, scale);       // q_cols is a multiple of 8
}

// One block of 128 x 128: a workgroup, sixteen lanes to a row, eight rows to a thread.
template <int DT>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(QuantParams p)
{
    __shared__ float peaks[4];
    const uint32_t rb = blockIdx.x / p.blocks, kb = blockIdx.x - rb * p.blocks;
    const uint32_t r0 = rb * kFpBlock + threadIdx.x / 16u, k0 = kb * kFpBlock + threadIdx.x % 16u * 8u;
    float x[8][8], peak = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t r = r0 + j * 16u;
        load8<DT>(p.x, (int64_t)min(r, p.R - 1u) * p.x_stride, k0, r < p.R ? p.K : 0u, x[j]);
        peak = fmaxf(peak, largest8(x[j]));
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) peak = fmaxf(peak, __shfl_xor(peak, d));
    if (threadIdx.x % 64 == 0) peaks[threadIdx.x / 64] = peak;
    __syncthreads();
    const float scale = block_scale(fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3])));
    if (threadIdx.x == 0) p.scale[(size_t)rb * p.blocks + kb] = scale;
    if (k0 >= p.q_cols) return;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t r = r0 + j * 16u;
        if (r < p.R) *(uint2 *)(p.q + (int64_t)r * p.q_stride + k0) = quantize8(x[j], scale);
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

__device__ __forceinline__ void widen_block(v8i q, v8bf (&b)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = widen8(q[2 * i], q[2 * i + 1]);
}

// 16 x 16 sums over a block of 128.  Lane l gives 32 bytes of row l % 16 of either side (any 32 of the block's columns, as
// long as both sides agree) and has the sums of w's rows 4 (l / 16) + 0..3 with x's row l % 16.
//
// On bfloat16, whatever y's type: the matrix instructions that take 8 bits do not hold their sums in 32.  Of the eight products that
// they add at once, what lies 14 binades and more under the largest is dropped (256 * 256 + 4 is 65536, for both kinds of them),
// always towards the largest, and no rounding of y covers that where large products cancel: 3.1e-5 of a result's size over 4096
// random columns, up to 7 * 2^-13 of the sum of magnitudes.  Those that take bfloat16 keep 24 bits (1.0e-7), at half the rate:
// 8192^3 into bfloat16 1005 us, 560 with the former.
__device__ __forceinline__ v4f block_product(const v8bf (&w)[4], const v8bf (&x)[4])
{
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i], x[i], acc, 0, 0, 0);
    return acc;
}

// Four consecutive values, or eight of 16 bits, in one store.  y's rows begin at any multiple of a value's size (an odd number of
// columns), and the hardware stores at any address: 128 x 50257 x 2048 into bfloat16 41 us, 65 in single values.
template <int DT> __device__ __forceinline__ void put_four(void *p, int64_t i, v4f a)
{
    if constexpr (DT == RS_DTYPE_F32) __builtin_memcpy((float *)p + i, &a, 16);
    else if constexpr (DT == RS_DTYPE_BF16) {
        const v4bf v = {(__bf16)a[0], (__bf16)a[1], (__bf16)a[2], (__bf16)a[3]};
        __builtin_memcpy((__bf16 *)p + i, &v, 8);
    } else {
        const v4h v = {(_Float16)a[0], (_Float16)a[1], (_Float16)a[2], (_Float16)a[3]};
        __builtin_memcpy((_Float16 *)p + i, &v, 8);
    }
}
template <int DT> __device__ __forceinline__ void put_wide(void *p, int64_t i, v4f a, v4f b)
{
    if constexpr (DT == RS_DTYPE_F32) put_four<DT>(p, i, a);
    else if constexpr (DT == RS_DTYPE_BF16) {
        v8bf v;
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = (__bf16)a[j]; v[j + 4] = (__bf16)b[j]; }
        __builtin_memcpy((__bf16 *)p + i, &v, 16);
    } else {
        v8h v;
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = (_Float16)a[j]; v[j + 4] = (_Float16)b[j]; }
        __builtin_memcpy((_Float16 *)p + i, &v, 16);
    }
}

// --------------------------------------------------------------- few rows --
// Bound by reading w once.  A workgroup makes 16 NT rows of w x up to 16 rows of x; its waves take the blocks of 128 columns in
// turn, so that it reads 1 KB of each row at a time and nothing is shared but the sums, which go through LDS once, at
// the end, and are added in the order of the waves.  A wave asks for its next block before it multiplies the one it has.
//
// XT < 0: x is in 8 bits.  Else it is of that type, and every workgroup rounds all of it (a few rows) into LDS while its first
// rows of w are on their way: one launch in the place of two.
template <int XT, int NT>
struct LinearFew {
    struct Block {
        v8i   w[NT], x;
        float f, s;                      // x's scale (of a row that is in memory), w's
    };
    const uint8_t *w[NT], *x;            // the lane's rows, at its columns of the first block; x in memory or in LDS
    const float   *sw, *sx;

    __device__ __forceinline__ LinearFew(const LinearParams &p, uint32_t n0, uint32_t m0, const uint8_t *lds)
    {
        const uint32_t lane = threadIdx.x % 64u, i = lane % 16u, part = lane / 16u;
#pragma unroll
        for (int u = 0; u < NT; ++u) w[u] = p.w + (int64_t)min(n0 + u * 16u + i, p.N - 1u) * p.w_stride + part * 16u;
        const uint32_t m = min(m0 + i, p.M - 1u);
        x = (XT < 0 ? p.x + (int64_t)m * p.x_stride : lds + m * (p.blocks * kFpBlock)) + part * 16u;
        sx = (XT < 0 ? p.x_scale : (const float *)(lds + p.M * p.blocks * kFpBlock)) + (size_t)m * p.blocks;
        sw = p.w_scale + (size_t)(n0 / kFpBlock) * p.blocks;
    }
    // (w is read once and need not stay in the caches; x is read by every workgroup)
    __device__ __forceinline__ void load(const LinearParams &p, uint32_t kb, Block &b) const
    {
        const uint32_t k = kb * kFpBlock;
        if (k + kFpBlock <= p.K) {
#pragma unroll
            for (int u = 0; u < NT; ++u)
                b.w[u] = join(__builtin_nontemporal_load((const v4i *)(w[u] + k)), __builtin_nontemporal_load((const v4i *)(w[u] + k + 64)));
            if constexpr (XT < 0) b.x = join(*(const v4i *)(x + k), *(const v4i *)(x + k + 64));
        } else {
            const uint32_t at = threadIdx.x % 64u / 16u * 16u;
#pragma unroll
            for (int u = 0; u < NT; ++u) b.w[u] = join(load16(w[u] - at, k + at, p.K), load16(w[u] - at, k + at + 64u, p.K));
            if constexpr (XT < 0) b.x = join(load16(x - at, k + at, p.K), load16(x - at, k + at + 64u, p.K));
        }
        b.s = sw[kb];
        if constexpr (XT < 0) b.f = sx[kb];
    }
    __device__ __forceinline__ void multiply(Block b, uint32_t kb, v4f (&acc)[NT]) const
    {
        if constexpr (XT >= 0) {
            b.x = join(*(const v4i *)(x + kb * kFpBlock), *(const v4i *)(x + kb * kFpBlock + 64));
            b.f = sx[kb];
        }
        const float f = b.s * b.f;
        v8bf xb[4];
        widen_block(b.x, xb);
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            v8bf wb[4];
            widen_block(b.w[u], wb);
            const v4f s = block_product(wb, xb);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[u][j] = __builtin_fmaf(s[j], f, acc[u][j]);
        }
    }
};

template <int DT, int XT, int NT>
__global__ __launch_bounds__(512) void linear_few_kernel(LinearParams p)
{
    using L = LinearFew<XT, NT>;
    __shared__ v4f sums[8][NT][64];
    extern __shared__ uint8_t lds[];
    const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u, waves = blockDim.x / 64u, i = lane % 16u, part = lane / 16u;
    const uint32_t n0 = blockIdx.x * (16u * NT), m0 = blockIdx.y * 16u;
    const L rows(p, n0, m0, lds);
    // (every workgroup begins at another block: see the kernel for many rows)
    const uint32_t turn = blockIdx.x % p.blocks;
    auto turned = [&](uint32_t kb) { kb += turn; return kb < p.blocks ? kb : kb - p.blocks; };
    typename L::Block now, next;
    if (wave < p.blocks) rows.load(p, turned(wave), now);
    if constexpr (XT >= 0) {
        for (uint32_t c = threadIdx.x / 16u; c < p.M * p.blocks; c += waves * 4u) {
            const uint32_t r = c / p.blocks, k = (c - r * p.blocks) * kFpBlock + threadIdx.x % 16u * 8u;
            float x[8];
            load8<XT>(p.x, (int64_t)r * p.x_stride, k, p.K, x);
            const float scale = block_scale(max16(largest8(x)));
            *(uint2 *)(lds + r * (p.blocks * kFpBlock) + k) = quantize8(x, scale);
            if (threadIdx.x % 16u == 0) ((float *)(lds + p.M * p.blocks * kFpBlock))[c] = scale;
        }
        __syncthreads();
    }
    v4f acc[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (wave < p.blocks) {
        uint32_t kb = turned(wave);
        for (uint32_t j = wave + waves; j < p.blocks; j += waves) {
            const uint32_t following = turned(j);
            rows.load(p, following, next);
            rows.multiply(now, kb, acc);
            now = next;
            kb = following;
        }
        rows.multiply(now, kb, acc);
    }
#pragma unroll
    for (int u = 0; u < NT; ++u) sums[wave][u][lane] = acc[u];
    __syncthreads();
    for (uint32_t u = wave; u < (uint32_t)NT; u += waves) {
        v4f s = sums[0][u][lane];
        for (uint32_t o = 1; o < waves; ++o) s += sums[o][u][lane];
        const uint32_t m = m0 + i, n = n0 + u * 16u + part * 4u;
        if (m >= p.M) continue;
        const int64_t at = (int64_t)m * p.y_stride + n;
        if (n + 4u <= p.N) put_four<DT>(p.y, at, s);
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) if (n + j < p.N) put<DT>(p.y, at + j, s[j]);
    }
}

// -------------------------------------------------------------- many rows --
// A workgroup of WN x WM waves makes 16 NU WN rows of w x 16 MT WM rows of x, a wave 16 NU x 16 MT of it.  Every block has to be
// scaled in the vector unit before it is added (four sums a lane and 16 x 16 product), so a wave's sums sit in 4 NU MT ordinary
// registers; a product's sums are added while the matrix cores make the next.
//
// A block of 128 columns is one stage: rows of 128 bytes go from memory to LDS without passing through registers, up to
// STAGES - 1 blocks ahead of the one that is multiplied.  The eight 16-byte pieces of a row are stored in an order that depends on
// the row (place = piece ^ turn(row)), so that the eight rows read at once lie in different banks.  The first operand's rows are
// dealt so that a lane's sums are 4 NU consecutive columns of y.
typedef __attribute__((address_space(3))) void *LdsPtr;

template <int NU> __device__ __forceinline__ uint32_t w_turn(uint32_t row) { return (row & 3u) | ((row / NU) & 4u); }
__device__ __forceinline__ uint32_t x_turn(uint32_t row) { return row & 7u; }

__device__ __forceinline__ uint32_t wave_id() { return uniform(threadIdx.x / 64u); }

// All but the newest N loads of this wave are done, and so are every other wave's, and their reads of LDS.
template <int N> __device__ __forceinline__ void stage_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory");
}

template <int WN, int WM, int NU, int MT, int STAGES>
struct LinearTile {
    static constexpr uint32_t kWaves = WN * WM, kThreads = 64 * kWaves, kTileN = 16 * NU * WN, kTileM = 16 * MT * WM;
    static constexpr uint32_t kRows = kTileN + kTileM, kStage = kRows * kFpBlock, kLds = STAGES * kStage;
    static constexpr uint32_t kLoads = kRows * 8 / kThreads, kLoadsW = kTileN * 8 / kThreads;    // 16-byte pieces of a stage per thread
    static_assert(kRows * 8 % kThreads == 0 && kTileN * 8 % kThreads == 0 && kTileN <= 256 && kTileM <= 256, "whole loads; rs_tile.h");
    static_assert(kWaves % 4 == 0, "w_turn is the same for every load of a thread, or for every other one");
    static_assert(NU == 4 || NU == 8, "");
    static constexpr int kBufferFlags = 0x00027000;              // untyped, offsets in bytes

    // A wave fills eight rows of a stage with one load: the thread's row of load i, w's rows first.
    static __device__ __forceinline__ uint32_t row_of(uint32_t i) { return tile_row(i, kWaves, wave_id(), threadIdx.x % 64u); }

    // The tile's rows as two buffers; rows behind the last read as 0.
    struct Source {
        __amdgpu_buffer_rsrc_t w, x;
        uint32_t w_stride, x_stride, w_rows, x_rows;
        uint32_t w_piece[2], x_piece;    // byte of a block of the thread's piece of its row of an even, of an odd load
        uint32_t first[kLoads];          // at(i, 0)

        // The thread's byte of load i, of the block that begins at column k
        __device__ __forceinline__ uint32_t at(uint32_t i, uint32_t k) const
        {
            return i < kLoadsW ? tile_at(row_of(i), w_rows, w_stride, w_piece[kWaves % 8 ? i % 2 : 0] + k)
                               : tile_at(row_of(i) - kTileN, x_rows, x_stride, x_piece + k);
        }
    };
    static __device__ __forceinline__ Source source(const LinearParams &p, uint32_t n0, uint32_t m0)
    {
        Source s;
        s.w_stride = (uint32_t)p.w_stride;
        s.x_stride = (uint32_t)p.x_stride;
        s.w_rows = min(p.N - n0, kTileN);
        s.x_rows = min(p.M - m0, kTileM);
        s.w = __builtin_amdgcn_make_buffer_rsrc((void *)(p.w + (int64_t)n0 * p.w_stride), 0, (int)tile_bytes(s.w_rows, s.w_stride, p.K), kBufferFlags);
        s.x = __builtin_amdgcn_make_buffer_rsrc((void *)(p.x + (int64_t)m0 * p.x_stride), 0, (int)tile_bytes(s.x_rows, s.x_stride, p.K), kBufferFlags);
        for (uint32_t i = 0; i < 2; ++i) s.w_piece[i] = ((threadIdx.x & 7u) ^ w_turn<NU>(row_of(i))) * 16u;
        s.x_piece = ((threadIdx.x & 7u) ^ x_turn(row_of(0))) * 16u;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            s.first[i] = s.at(i, 0);
            asm volatile("" : "+v"(s.first[i]));      // once, and not for every block (2 to 4 % of 256 x 4096 x 4096)
        }
        return s;
    }
    static __device__ __forceinline__ void fill(const LinearParams &p, const Source &s, uint32_t n0, uint32_t m0, uint32_t kb, uint8_t *lds)
    {
        const uint32_t k = kb * kFpBlock;
        if (k + kFpBlock <= p.K) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const LdsPtr to = (LdsPtr)(lds + (i * kWaves + wave_id()) * 1024u);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(i < kLoadsW ? s.w : s.x, to, 16, s.first[i], k, 0, 0);
            }
            return;
        }
        // the last block where K is no whole number of them: through registers, with the bytes from K on cleared
        v4i v[kLoads];
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(i < kLoadsW ? s.w : s.x, s.at(i, k), 0, 0);
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t r = row_of(i) - (i < kLoadsW ? 0u : kTileN);
            const int32_t left = (int32_t)(p.K - k) - (int32_t)(((threadIdx.x & 7u) ^ (i < kLoadsW ? w_turn<NU>(r) : x_turn(r))) * 16u);
#pragma unroll
            for (int d = 0; d < 4; ++d) v[i][d] &= left >= 4 * d + 4 ? -1 : left <= 4 * d ? 0 : (1 << 8 * (left - 4 * d)) - 1;
            *(v4i *)(lds + row_of(i) * kFpBlock + (threadIdx.x & 7u) * 16u) = v[i];
        }
        wait_vmem();
    }

    static __device__ __forceinline__ v8i fragment(const uint8_t *lds, uint32_t row, uint32_t turn, uint32_t part)
    {
        const uint8_t *r = lds + row * kFpBlock;
        return join(*(const v4i *)(r + ((part ^ turn) * 16u)), *(const v4i *)(r + (((part + 4u) ^ turn) * 16u)));
    }

    // Asks for block `next` and multiplies the one in now_lds.
    static __device__ __forceinline__ void step(const LinearParams &p, const Source &source, uint32_t n0, uint32_t m0, uint32_t next, bool more,
                                                const uint8_t *__restrict now_lds, uint8_t *__restrict next_lds, const float (&f)[MT], v4f (&acc)[NU][MT])
    {
        if (more) fill(p, source, n0, m0, next, next_lds);
        const uint32_t wave = wave_id(), lane = threadIdx.x % 64u, i = lane % 16u, part = lane / 16u;
        const uint32_t wn = wave % WN * (16u * NU), wm = wave / WN * (16u * MT);
        v8bf xb[MT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const uint32_t r = wm + t * 16u + i;
            widen_block(fragment(now_lds + kTileN * kFpBlock, r, x_turn(r), part), xb[t]);
        }
        const uint32_t r0 = wn + i / 4u * (4u * NU) + i % 4u;
        v8i w = fragment(now_lds, r0, w_turn<NU>(r0), part);
        v4f s[MT];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            v8i ahead = w;
            if (u < NU - 1) {
                const uint32_t r = r0 + (u + 1) * 4u;
                ahead = fragment(now_lds, r, w_turn<NU>(r), part);
            }
            v8bf wb[4];
            widen_block(w, wb);
            // (the sums of the row of products before, each behind a product of this one)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const v4f made = block_product(wb, xb[t]);
                if (u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[u - 1][t][j] = __builtin_fmaf(s[t][j], f[t], acc[u - 1][t][j]);
                s[t] = made;
            }
            w = ahead;
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[NU - 1][t][j] = __builtin_fmaf(s[t][j], f[t], acc[NU - 1][t][j]);
    }
};

template <int DT, int WN, int WM, int NU, int MT, int STAGES, bool SPLIT>
__global__ __launch_bounds__(64 * WN * WM, 2) void linear_tile_kernel(LinearParams p)
{
    using L = LinearTile<WN, WM, NU, MT, STAGES>;
    extern __shared__ uint8_t lds[];
    const uint32_t tm = (p.M + L::kTileM - 1u) / L::kTileM, tn = (p.N + L::kTileN - 1u) / L::kTileN, tiles = tm * tn;
    // Workgroup b runs on XCD b % 8: each XCD takes a stretch of the tiles, in panels of eight rows of tiles, so that the 32 tiles
    // it works on at a time share their rows in its L2.
    uint32_t id = blockIdx.x, part_of = 0;
    if (SPLIT && p.split > 1u) { part_of = id / tiles; id -= part_of * tiles; }
    else {
        const uint32_t each = tiles / 8u, rest = tiles % 8u, xcd = id % 8u;
        id = xcd * each + min(xcd, rest) + id / 8u;
    }
    const uint32_t panel = id / (8u * tn), high = min(8u, tm - panel * 8u), in = id - panel * 8u * tn;
    const uint32_t tile_n = in / high, m0 = (panel * 8u + in % high) * L::kTileM, n0 = tile_n * L::kTileN;
    const uint32_t kb0 = p.blocks * part_of / p.split, count = p.blocks * (part_of + 1u) / p.split - kb0;

    const uint32_t wave = wave_id(), lane = threadIdx.x % 64u, i = lane % 16u, part = lane / 16u;
    const uint32_t wn = wave % WN * (16u * NU), wm = wave / WN * (16u * MT);
    const float *sw = p.w_scale + (size_t)min((n0 + wn) / kFpBlock, (p.N - 1u) / kFpBlock) * p.blocks;
    // x's scales as a buffer as well: addressed with 32 bits, and 0 for rows that are not there
    const uint32_t sx_rows = min(p.M - m0, L::kTileM);
    const __amdgpu_buffer_rsrc_t sx = __builtin_amdgcn_make_buffer_rsrc((void *)(p.x_scale + (size_t)m0 * p.blocks), 0, (int)(sx_rows * p.blocks * 4u), L::kBufferFlags);
    auto x_scale = [&](int t, uint32_t kb) { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sx, tile_at(wm + t * 16u + i, sx_rows, p.blocks * 4u, 0u), kb * 4u, 0)); };
    v4f acc[NU][MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NU; ++u) acc[u][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // Where w is read once, by one row of tiles, every workgroup begins at another block: rows are usually a power of two of bytes
    // apart, and workgroups in step would ask the same memory channels at a time.
    uint32_t first = tm == 1u ? kb0 + tile_n % count : kb0;
    auto after = [&](uint32_t kb) { return kb + 1u == kb0 + count ? kb0 : kb + 1u; };
    const typename L::Source source = L::source(p, n0, m0);
    // (a block's scales are asked for one block ahead, before that block's rows: waiting for them waits for nothing newer)
    float f[MT], ahead[MT], ahead_w = sw[first];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        ahead[t] = x_scale(t, first);
        asm volatile("" : "+v"(ahead[t]));       // here, and not in the loop, where it would wait for the next block's
    }
    uint32_t kb = first, to_fill = first;
#pragma unroll
    for (int b = 0; b < STAGES - 1; ++b)
        if (b < (int)count) { L::fill(p, source, n0, m0, to_fill, lds + b * L::kStage); to_fill = after(to_fill); }
    uint32_t now = 0, next = (STAGES - 1) * L::kStage;
    for (uint32_t j = 0; j < count; ++j) {
        // (towards the end there are no newer stages to leave under way)
        if (STAGES == 2 || j + STAGES - 1 > count) stage_barrier<0>();
        else stage_barrier<(STAGES - 2) * L::kLoads>();
#pragma unroll
        for (int t = 0; t < MT; ++t) f[t] = ahead[t] * ahead_w;
        kb = after(kb);
        ahead_w = sw[kb];
#pragma unroll
        for (int t = 0; t < MT; ++t) ahead[t] = x_scale(t, kb);
        L::step(p, source, n0, m0, to_fill, j + STAGES - 1u < count, lds + now, lds + next, f, acc);
        to_fill = after(to_fill);
        now = now == (STAGES - 1) * L::kStage ? 0u : now + L::kStage;
        next = next == (STAGES - 1) * L::kStage ? 0u : next + L::kStage;
    }
    if (SPLIT && p.split > 1u) {
        // every workgroup leaves its sums; the last of the tile's adds them up, in the order of the blocks
        constexpr uint32_t kPart = L::kThreads * NU * MT * 2;
        uint64_t *parts = (uint64_t *)p.parts + (size_t)id * p.split * kPart + threadIdx.x;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    a_store(&parts[part_of * kPart + ((u * MT + t) * 2 + h) * L::kThreads],
                            (uint64_t)__float_as_uint(acc[u][t][2 * h + 1]) << 32 | __float_as_uint(acc[u][t][2 * h]));
        uint32_t *last = (uint32_t *)lds;
        wait_vmem();
        __syncthreads();
        if (threadIdx.x == 0) {
            *last = __hip_atomic_fetch_add(&p.arrived[id], 1u, __ATOMIC_RELAXED, RS_AGENT) == p.split - 1u;
            if (*last) a_store(&p.arrived[id], 0u);
        }
        __syncthreads();
        if (!*last) return;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[u][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
        for (uint32_t s = 0; s < p.split; ++s) {
            uint64_t v[2 * NU * MT];
#pragma unroll
            for (int o = 0; o < 2 * NU * MT; ++o) v[o] = a_load(&parts[s * kPart + o * L::kThreads]);
#pragma unroll
            for (int o = 0; o < 2 * NU * MT; ++o) {
                acc[o / 2 / MT][o / 2 % MT][o % 2 * 2] += __uint_as_float((uint32_t)v[o]);
                acc[o / 2 / MT][o / 2 % MT][o % 2 * 2 + 1] += __uint_as_float((uint32_t)(v[o] >> 32));
            }
        }
    }
    // a lane has 4 NU columns of its rows of y
    const uint32_t n = n0 + wn + part * (4u * NU);
    constexpr uint32_t kVec = DT == RS_DTYPE_F32 ? 4 : 8;
    const bool wide = n + 4u * NU <= p.N;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const uint32_t m = m0 + wm + t * 16u + i;
        if (m >= p.M) continue;
        const int64_t at = (int64_t)m * p.y_stride + n;
        if (wide) {
#pragma unroll
            for (int u = 0; u < NU; u += kVec / 4) put_wide<DT>(p.y, at + u * 4, acc[u][t], acc[(u + 1) % NU][t]);
        } else {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) if (n + u * 4u + j < p.N) put<DT>(p.y, at + u * 4 + j, acc[u][t][j]);
        }
    }
}

}  // namespace rs
