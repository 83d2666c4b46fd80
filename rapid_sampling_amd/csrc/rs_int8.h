// Values as 8-bit integers with a float32 scale for each row, and their matrix product:
//
//   scale = max(max |x| * r, 2^-126), r = 1/127 in float32        q = x / scale, to the nearest integer, ties to even
//   y[m, n] = sx[m] sw[n] sum_k qx[m, k] qw[n, k]
//
// The sums are whole numbers of 32 bits, which no K up to 131071 leaves (128^2 K < 2^31): exact, in any order.  They are
// rounded to float32 once, multiplied with the product of the two scales, and rounded to y's type.
#pragma once

#include "rs_product.h"

namespace rs {

struct Int8Rows {                    // of the quantiser
    const void *x;
    int64_t     x_stride;            // elements
    int8_t     *q;
    int64_t     q_stride;            // bytes; those behind column K are cleared
    float      *scale;
    uint32_t    R, K;
};

struct Int8Params {
    Product      a;                  // P: w, Q: x
    const float *x_scale, *w_scale;
    void        *y;
    int64_t      y_stride;
    const void  *x;                  // few rows: x and w with 64-bit strides
    int64_t      x_stride, w_stride; // elements of x, bytes of w
    const int8_t *w;
    uint32_t     M, N, K;
    int         *parts;              // sums of workgroups that share a tile's reduction, and how many have left theirs; zero between calls
    uint32_t    *arrived;
};

// A row's largest magnitude as the bits of a float without its sign: NaN is larger than infinity, infinity than any number.
__device__ __forceinline__ uint32_t largest_bits(const float (&x)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    return m;
}
// A row with an infinity or a NaN has the scale NaN, and so have its results, and integers of 0.
__device__ __forceinline__ float row_scale(uint32_t peak)
{
    return peak < 0x7F800000u ? fmaxf(__uint_as_float(peak) * (1.0f / 127.0f), 0x1p-126f) : __builtin_nanf("");
}
// (with 1.5 2^23 added a number's integer, to the nearest and ties to even, is in the lowest bits of the sum)
__device__ __forceinline__ uint2 quantize8_int8(const float (&x)[8], float scale)
{
    if (!(scale < __builtin_inff())) return make_uint2(0u, 0u);
    const Divisor d(scale);
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float up = x[j] * d.up, q = up * d.r;                              // as Divisor, but for the sign of 0
        v[j] = __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, d.s, up), d.r, q) + 12582912.0f);
    }
    auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t e) {
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(e, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
    };
    return make_uint2(four(v[0], v[1], v[2], v[3]), four(v[4], v[5], v[6], v[7]));
}

// LANES threads to a row (64 or 256), eight values at a time; the first PIECES of a thread's are kept in registers, the others read again.  Bound by memory,
// or the launch: 131072 x 4096 in bfloat16 274 us (5.9 TB/s), 4096 x 4096 14.4 (3.5), 32 x 4096 4.8.
template <int DT, int LANES, int PIECES>
__global__ __launch_bounds__(256) void int8_rows_kernel(Int8Rows p)
{
    __shared__ uint32_t peaks[4];
    const uint32_t r = blockIdx.x * (256u / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const bool live = r < p.R;
    const int64_t at = (int64_t)min(r, p.R - 1u) * p.x_stride;
    float x[PIECES][8];
    uint32_t peak = 0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) load8<DT>(p.x, at, (i * LANES + lane) * 8u, p.K, x[i]);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) peak = max(peak, largest_bits(x[i]));
    for (uint32_t k = (PIECES * LANES + lane) * 8u; k < p.K; k += LANES * 8u) {
        float more[8];
        load8<DT>(p.x, at, k, p.K, more);
        peak = max(peak, largest_bits(more));
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) peak = max(peak, (uint32_t)__shfl_xor((int)peak, d));
    if (LANES > 64) {
        if (threadIdx.x % 64u == 0) peaks[threadIdx.x / 64u] = peak;
        __syncthreads();
        peak = max(max(peaks[0], peaks[1]), max(peaks[2], peaks[3]));
    }
    if (!live) return;
    const float scale = row_scale(peak);
    if (lane == 0) p.scale[r] = scale;
    int8_t *q = p.q + (int64_t)r * p.q_stride;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const uint32_t k = (i * LANES + lane) * 8u;
        if (k < (uint32_t)p.q_stride) *(uint2 *)(q + k) = quantize8_int8(x[i], scale);
    }
    for (uint32_t k = (PIECES * LANES + lane) * 8u; k < (uint32_t)p.q_stride; k += LANES * 8u) {
        float more[8];
        load8<DT>(p.x, at, k, p.K, more);
        *(uint2 *)(q + k) = quantize8_int8(more, scale);
    }
}

// --------------------------------------------------------------- few rows --
// Bound by reading w once (1 row, 65536 x 4096, beyond the caches: 48 us, 5.6 TB/s).  A workgroup makes 16 NT rows of w x up to 16 rows of x; its waves take the blocks of 128 columns in turn, and
// their sums go through LDS once, at the end.  A wave asks for its next block before it multiplies the one it has.
//
// XT < 0: x is in 8 bits.  Else it is of that type, and every workgroup rounds all of it (a few rows) into LDS while its first rows of w
// are on their way: one launch in the place of two.  Such workgroups are no more than the chip holds, and go from one stretch of w
// to another.
template <int DT, int XT, int NT>
__global__ __launch_bounds__(512) void int8_few_kernel(Int8Params p)
{
    __shared__ v4i sums[8][NT][64];
    __shared__ uint32_t peaks[4];
    extern __shared__ char lds[];
    const uint32_t lane = threadIdx.x % 64u, wave = wave_id(), waves = blockDim.x / 64u, i = lane % 16u, part = lane / 16u;
    const uint32_t m0 = blockIdx.y * 16u, blocks = (p.K + 127u) / 128u, stretches = (p.N + 16u * NT - 1u) / (16u * NT);
    const uint32_t m = min(m0 + i, p.M - 1u);
    const uint8_t *w[NT], *x = XT < 0 ? (const uint8_t *)p.x + (int64_t)m * p.x_stride : (const uint8_t *)lds + m * (blocks * 128u);
    struct Block { v4i w[NT][2], x[2]; };
    auto load = [&](uint32_t kb, Block &b) {
        const uint32_t k = kb * 128u + part * 16u;
        const bool whole = kb * 128u + 128u <= p.K;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int u = 0; u < NT; ++u) b.w[u][h] = whole ? *(const v4i *)(w[u] + k + 64 * h) : load16(w[u], k + 64u * h, p.K);
            if constexpr (XT < 0) b.x[h] = whole ? *(const v4i *)(x + k + 64 * h) : load16(x, k + 64u * h, p.K);
        }
    };
    Block now, next;
    uint32_t turn = 0;
    auto turned = [&](uint32_t kb) { kb += turn; return kb < blocks ? kb : kb - blocks; };
    // (every workgroup begins at another block: rows are usually a power of two of bytes apart, and workgroups in step would ask the same
    // memory channels at a time)
    auto begin = [&](uint32_t stretch) {
        turn = stretch % blocks;
#pragma unroll
        for (int u = 0; u < NT; ++u) w[u] = (const uint8_t *)p.w + (int64_t)min((stretch * NT + u) * 16u + i, p.N - 1u) * p.w_stride;
        if (wave < blocks) load(turned(wave), now);
    };
    // (each XCD has a part of w of its own, see Tile::choose: 1 row, 65536 x 2048 29.9 us in plain order, 27.5 so; 65536 x 8192 104 and 100; 65536 x 1024
    // 16.2 and 17.1)
    auto place = [&](uint32_t id) { return id % 8u * (stretches / 8u) + min(id % 8u, stretches % 8u) + id / 8u; };
    begin(place(blockIdx.x));
    if constexpr (XT >= 0) {
        // The waves are shared out among the rows, and of its row a wave takes pieces of 512 values in turn, the first of which it keeps in
        // registers; where there are more rows than waves (of up to 384 columns) it takes a piece, and all, of several.
        constexpr uint32_t kHeld = 4;
        const uint32_t high = p.M <= 2u ? p.M : 4u, each = max(waves / high, 1u), step = waves / each, pieces = (blocks + 3u) / 4u;
        const uint32_t row = wave / each, sub = wave % each;
        const bool several = waves < high;
        const uint32_t count = row >= p.M ? 0u : several ? (p.M - row + step - 1u) / step : sub >= pieces ? 0u : (pieces - sub + each - 1u) / each;
        auto row_of = [&](uint32_t e) { return several ? row + e * step : row; };
        auto first_of = [&](uint32_t e) { return (several ? 0u : (sub + e * each) * 512u) + lane * 8u; };
        float held[kHeld][8];
        auto fetch = [&](uint32_t e, float (&v)[8]) { load8<XT>(p.x, (int64_t)row_of(e) * p.x_stride, first_of(e), p.K, v); };
        uint32_t peak = 0;
        auto note = [&](uint32_t e, const float (&v)[8]) {
            peak = max(peak, largest_bits(v));
            if (!several && e + 1u < count) return;
#pragma unroll
            for (int d = 32; d; d >>= 1) peak = max(peak, (uint32_t)__shfl_xor((int)peak, d));
            if (lane == 0) atomicMax(&peaks[row_of(e)], peak);
            peak = 0;
        };
        auto put_piece = [&](uint32_t e, const float (&v)[8]) {
            const uint32_t k = first_of(e);
            if (k < blocks * 128u) *(uint2 *)(lds + row_of(e) * (blocks * 128u) + k) = quantize8_int8(v, row_scale(peaks[row_of(e)]));
        };
#pragma unroll
        for (uint32_t h = 0; h < kHeld; ++h)
            if (h < count) fetch(h, held[h]);
        if (threadIdx.x < 4u) peaks[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t h = 0; h < kHeld; ++h)
            if (h < count) note(h, held[h]);
        for (uint32_t e = kHeld; e < count; ++e) {
            float v[8];
            fetch(e, v);
            note(e, v);
        }
        __syncthreads();
#pragma unroll
        for (uint32_t h = 0; h < kHeld; ++h)
            if (h < count) put_piece(h, held[h]);
        for (uint32_t e = kHeld; e < count; ++e) {
            float v[8];
            fetch(e, v);
            put_piece(e, v);
        }
        __syncthreads();
    }
    auto take = [&](Block &b, uint32_t kb, v4i (&acc)[NT]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (XT >= 0) b.x[h] = *(const v4i *)(x + kb * 128u + part * 16u + 64 * h);
#pragma unroll
            for (int u = 0; u < NT; ++u) acc[u] = multiply<kInt8>(b.w[u][h], b.x[h], acc[u]);
        }
    };
    for (uint32_t id = blockIdx.x;;) {
        v4i acc[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[u] = v4i{0, 0, 0, 0};
        if (wave < blocks) {
            uint32_t kb = turned(wave);
            for (uint32_t j = wave + waves; j < blocks; j += waves) {
                const uint32_t following = turned(j);
                load(following, next);
                take(now, kb, acc);
                now = next;
                kb = following;
            }
            take(now, kb, acc);
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) sums[wave][u][lane] = acc[u];
        const uint32_t n0 = place(id) * (16u * NT);
        id += gridDim.x;
        const bool more = XT >= 0 && id < stretches;
        if (more) begin(place(id));
        __syncthreads();
        for (uint32_t u = wave; u < (uint32_t)NT; u += waves) {
            v4i s = sums[0][u][lane];
            for (uint32_t o = 1; o < waves; ++o) s += sums[o][u][lane];
            const uint32_t row = m0 + i, n = n0 + u * 16u + part * 4u;
            if (row >= p.M) continue;
            const float f = XT < 0 ? p.x_scale[row] : row_scale(peaks[row]);
            v4f y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = in_float32((float)s[j] * (f * p.w_scale[min(n + j, p.N - 1u)]));
            store_row<DT>(p.y, (int64_t)row * p.y_stride, n, p.N, y);
        }
        if (!more) return;
        __syncthreads();
    }
}

// -------------------------------------------------------------- many rows --
// Results go to memory by way of LDS, by whole rows.  4096 x 131072 x 4096 1.94 ms (2.2 POP/s; the matrix cores alone would make 4.2, see rs_product.h for
// what the tiles wait for), 32 x 131072 x 4096 97 us (5.7 TB/s).
template <int DT, int WN, int WM, int NU, int MT, int STAGES>
using Int8Tile = Tile<kInt8, false, false, DT != RS_DTYPE_F32, WN, WM, NU, MT, STAGES>;

template <int DT, int WN, int WM, int NU, int MT, int STAGES, bool SPLIT>
__global__ __launch_bounds__(64 * WN * WM, 2) void int8_tile_kernel(Int8Params p)
{
    using T = Int8Tile<DT, WN, WM, NU, MT, STAGES>;
    extern __shared__ char lds[];
    T tile;
    const uint32_t part = tile.choose(p.a, blockIdx.x);
    typename T::Acc acc;
    tile.make(p.a, part, lds, acc);
    if (SPLIT && p.a.split > 1u) {
        // every workgroup leaves its sums; the last of the tile's adds them up
        constexpr uint32_t kPart = T::kThreads * T::NU * T::MT * 2;
        const uint32_t tiles = gridDim.x / p.a.split, id = blockIdx.x % tiles;
        uint64_t *parts = (uint64_t *)p.parts + (size_t)id * p.a.split * kPart + threadIdx.x;
#pragma unroll
        for (int u = 0; u < T::NU; ++u)
#pragma unroll
            for (int t = 0; t < T::MT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    a_store(&parts[part * kPart + ((u * T::MT + t) * 2 + h) * T::kThreads], (uint64_t)(uint32_t)acc[u][t][2 * h + 1] << 32 | (uint32_t)acc[u][t][2 * h]);
        uint32_t *last = (uint32_t *)lds;
        wait_vmem();
        __syncthreads();
        if (threadIdx.x == 0) {
            *last = __hip_atomic_fetch_add(&p.arrived[id], 1u, __ATOMIC_RELAXED, RS_AGENT) == p.a.split - 1u;
            if (*last) a_store(&p.arrived[id], 0u);
        }
        __syncthreads();
        if (!*last) return;
#pragma unroll
        for (int u = 0; u < T::NU; ++u)
#pragma unroll
            for (int t = 0; t < T::MT; ++t) acc[u][t] = v4i{0, 0, 0, 0};
#pragma unroll 2
        for (uint32_t s = 0; s < p.a.split; ++s) {
            uint64_t v[2 * T::NU * T::MT];
#pragma unroll
            for (int o = 0; o < 2 * T::NU * T::MT; ++o) v[o] = a_load(&parts[s * kPart + o * T::kThreads]);
#pragma unroll
            for (int o = 0; o < 2 * T::NU * T::MT; ++o) {
                acc[o / 2 / T::MT][o / 2 % T::MT][o % 2 * 2] += (int)(uint32_t)v[o];
                acc[o / 2 / T::MT][o / 2 % T::MT][o % 2 * 2 + 1] += (int)(uint32_t)(v[o] >> 32);
            }
        }
    }
    auto row_of = [&](int t, v4f (&v)[T::NU]) {
        const float f = p.x_scale[min(tile.m(t), p.M - 1u)];
#pragma unroll
        for (int u = 0; u < T::NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][j] = in_float32((float)acc[u][t][j] * (f * p.w_scale[min(tile.n(u) + j, p.N - 1u)]));
    };
    const TileStore<DT, T> out(lds);
#pragma unroll
    for (int t = 0; t < T::MT; ++t) {
        v4f v[T::NU];
        row_of(t, v);
        if constexpr (DT == RS_DTYPE_F32) {
            out.put(v);
            out.flush(tile, t, (float *)p.y, p.y_stride, p.M, p.N);
        } else out.put(t, v);
    }
    if constexpr (DT != RS_DTYPE_F32) out.flush(tile, p.y, p.y_stride, p.M, p.N);
}

}  // namespace rs
