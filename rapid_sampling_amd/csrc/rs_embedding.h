// Rows of a table by token, and the table's gradient.
//
//   y[i] = s w[t_i]          dw[v] = s sum over i with t_i = v of g_i, in the order of i, in float32
//
// The gradient's positions are put in the order of their tokens first (a radix sort that keeps the order of equal ones), so that a row of
// dw is one stretch of them: no floating-point atomics, and the same sums every time.  Rows without a token are written as zeros by
// the same pass.  Bound by memory: y and g once, dw once.
#pragma once

#include "rs_linear.h"

namespace rs {

constexpr int kTableInt8 = 3, kTableFp8 = 4;         // types of a table, next to RS_DTYPE_*

struct TokenList {
    const void *at;
    int64_t     stride;
    int32_t     is_64;
    __device__ __forceinline__ int64_t operator[](int64_t i) const
    {
        return is_64 ? ((const int64_t *)at)[i * stride] : (int64_t)((const int32_t *)at)[i * stride];
    }
};

struct EmbeddingParams {
    TokenList    tokens;
    const void  *w;
    int64_t      w_stride;           // elements
    const float *w_scale;
    void        *y;
    float        scale;
    uint32_t     M, V, K;
    uint32_t     width;              // log2 of the threads of a row
};

// Eight values of a row of the table from column k on.
template <int WT>
__device__ __forceinline__ void table8(const EmbeddingParams &p, int64_t token, uint32_t k, float (&x)[8])
{
    if constexpr (WT == kTableInt8 || WT == kTableFp8) {
        const uint8_t *row = (const uint8_t *)p.w + token * p.w_stride + k;         // (rows begin at multiples of 16 bytes)
        uint2 q = make_uint2(0u, 0u);
        if (k + 8u <= p.K) q = *(const uint2 *)row;
        else
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) if (k + j < p.K) (j < 4 ? q.x : q.y) |= (uint32_t)row[j] << (8 * (j % 4));
        const float f = WT == kTableInt8 ? p.w_scale[token] : p.w_scale[(token / kFpBlock) * ((p.K + kFpBlock - 1) / kFpBlock) + k / kFpBlock];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t b = (j < 4 ? q.x : q.y) >> (8 * (j % 4)) & 0xFFu;
            if constexpr (WT == kTableInt8) x[j] = (float)(int8_t)b * f;
            else x[j] = __builtin_amdgcn_cvt_f32_fp8((int)b, 0) * f;
        }
    } else load8<WT>(p.w, token * p.w_stride, k, p.K, x);
}
// Eight values into columns k and following of a row of K that begins at element `at`.
template <int DT>
__device__ __forceinline__ void store8(void *y, int64_t at, uint32_t k, uint32_t K, const float (&x)[8])
{
    if (k + 8u <= K) {
        const v4f a = {x[0], x[1], x[2], x[3]}, b = {x[4], x[5], x[6], x[7]};
        put_wide<DT>(y, at + k, a, b);
        if constexpr (DT == RS_DTYPE_F32) put_four<DT>(y, at + k + 4, b);
    } else
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) if (k + j < K) put<DT>(y, at + k + j, x[j]);
}

// 2^width threads to a row, eight values at a time.
template <int WT, int DT>
__global__ __launch_bounds__(256) void embedding_kernel(EmbeddingParams p)
{
    const int64_t i = ((int64_t)blockIdx.x << (8 - p.width)) + (threadIdx.x >> p.width);
    if (i >= p.M) return;
    const int64_t token = p.tokens[i];
    for (uint32_t k = (threadIdx.x & ((1u << p.width) - 1u)) * 8u; k < p.K; k += 8u << p.width) {
        float x[8];
        if (token >= 0 && token < (int64_t)p.V) {
            table8<WT>(p, token, k, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = in_float32(x[j] * p.scale);
        } else
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = token < 0 ? 0.0f : __builtin_nanf("");
        store8<DT>(p.y, i * p.K, k, p.K, x);
    }
}

// -------------------------------------------------------------------- order --
// A digit of up to 11 bits at a time.  A workgroup of 16 waves takes a stretch of the list, each wave a part of it, 64 tokens at
// a time; a counter for each digit and wave in LDS.
constexpr uint32_t kSortWaves = 16, kSortThreads = 64 * kSortWaves, kSortBits = 11, kSortTile = 8192, kSortAlone = 16384;

struct SortParams {
    TokenList       tokens;          // of the first digit: what is sorted; a token that is none counts as V
    const uint32_t *keys_in, *at_in;
    uint32_t       *keys, *at;       // sorted by this digit
    uint32_t       *counts;          // [digit][workgroup]
    uint32_t        N, V, shift, bits, first;
    uint32_t       *keys_b, *at_b;   // a workgroup that does it all alone: the other side
    uint32_t        digits;          // ... and how many digits
};

__device__ __forceinline__ uint32_t sort_key(const SortParams &p, uint32_t i)
{
    if (!p.first) return p.keys_in[i];
    const int64_t t = p.tokens[i];
    return t >= 0 && t < (int64_t)p.V ? (uint32_t)t : p.V;
}
// The lanes with the same digit as this one's.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, uint32_t bits, bool live)
{
    uint64_t same = __ballot(live);
    for (uint32_t b = 0; b < bits; ++b) {
        const uint64_t set = __ballot(digit >> b & 1u);
        same &= digit >> b & 1u ? set : ~set;
    }
    return same;
}
// counts[wave][digit] of the tokens from `from` to `to`; then (PLACE) each goes to where its counter points.
template <bool PLACE>
__device__ __forceinline__ void sort_part(const SortParams &p, uint32_t from, uint32_t to, uint32_t *counts)
{
    const uint32_t lane = threadIdx.x % 64u, mask = (1u << p.bits) - 1u;
    for (uint32_t i0 = from; i0 < to; i0 += 64u) {
        const uint32_t i = i0 + lane;
        const bool live = i < to;
        const uint32_t key = live ? sort_key(p, i) : 0u, digit = key >> p.shift & mask;
        const uint64_t same = same_digit(digit, p.bits, live);
        const uint32_t before = __popcll(same & ((1ull << lane) - 1ull));
        const uint32_t have = live ? counts[digit] : 0u;
        if (PLACE && live) {
            p.keys[have + before] = key;
            p.at[have + before] = p.first ? i : p.at_in[i];
        }
        __builtin_amdgcn_wave_barrier();
        if (live && before == 0) counts[digit] = have + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
}
// The stretch of this wave.
__device__ __forceinline__ void sort_stretch(uint32_t first, uint32_t last, uint32_t &from, uint32_t &to)
{
    const uint32_t each = ((last - first + kSortWaves - 1u) / kSortWaves + 63u) & ~63u, wave = threadIdx.x / 64u;
    from = min(first + wave * each, last);
    to = min(from + each, last);
}
__device__ __forceinline__ void sort_count(const SortParams &p, uint32_t first, uint32_t last, uint32_t *counts)
{
    for (uint32_t i = threadIdx.x; i < kSortWaves << p.bits; i += kSortThreads) counts[i] = 0;
    __syncthreads();
    uint32_t from, to;
    sort_stretch(first, last, from, to);
    sort_part<false>(p, from, to, counts + ((threadIdx.x / 64u) << p.bits));
    __syncthreads();
}
// Exclusive sums over the workgroup's threads.
__device__ __forceinline__ uint32_t sums_before(uint32_t v, uint32_t *held, uint32_t &total)
{
    uint32_t s = v;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t o = __shfl_up(s, d);
        if (threadIdx.x % 64u >= d) s += o;
    }
    __syncthreads();
    if (threadIdx.x % 64u == 63u) held[threadIdx.x / 64u] = s;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    for (uint32_t w = 0; w < kSortWaves; ++w) {
        if (w < threadIdx.x / 64u) before += held[w];
        total += held[w];
    }
    return before + s - v;
}

// Up to kSortAlone tokens, by one workgroup, all digits.
__global__ __launch_bounds__(1024) void sort_alone_kernel(SortParams p)
{
    extern __shared__ uint32_t counts[];
    __shared__ uint32_t held[kSortWaves];
    for (uint32_t d = 0; d < p.digits; ++d) {
        sort_count(p, 0, p.N, counts);
        uint32_t from, to, base = 0, total;
        for (uint32_t b0 = 0; b0 < 1u << p.bits; b0 += kSortThreads) {
            const uint32_t b = b0 + threadIdx.x;
            uint32_t n = 0;
            if (b < 1u << p.bits)
                for (uint32_t w = 0; w < kSortWaves; ++w) n += counts[(w << p.bits) + b];
            uint32_t at = base + sums_before(n, held, total);
            base += total;
            if (b < 1u << p.bits)
                for (uint32_t w = 0; w < kSortWaves; ++w) {
                    const uint32_t c = counts[(w << p.bits) + b];
                    counts[(w << p.bits) + b] = at;
                    at += c;
                }
        }
        __syncthreads();
        sort_stretch(0, p.N, from, to);
        sort_part<true>(p, from, to, counts + ((threadIdx.x / 64u) << p.bits));
        // the next digit reads what the other waves have written
        __threadfence();
        __syncthreads();
        p.first = 0;
        p.shift += p.bits;
        p.keys_in = p.keys; p.at_in = p.at;
        p.keys = p.keys_b; p.at = p.at_b;
        p.keys_b = (uint32_t *)p.keys_in; p.at_b = (uint32_t *)p.at_in;
    }
}

// More: one digit in three launches.  Counts of each stretch ...
__global__ __launch_bounds__(1024) void sort_count_kernel(SortParams p)
{
    extern __shared__ uint32_t counts[];
    const uint32_t first = blockIdx.x * kSortTile;
    sort_count(p, first, min(first + kSortTile, p.N), counts);
    for (uint32_t b = threadIdx.x; b < 1u << p.bits; b += kSortThreads) {
        uint32_t n = 0;
        for (uint32_t w = 0; w < kSortWaves; ++w) n += counts[(w << p.bits) + b];
        p.counts[(size_t)b * gridDim.x + blockIdx.x] = n;
    }
}
// ... where each stretch's tokens of a digit begin ...
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t *counts, uint32_t many)
{
    __shared__ uint32_t held[kSortWaves];
    uint32_t base = 0, total;
    for (uint32_t i0 = 0; i0 < many; i0 += 4u * kSortThreads) {
        const uint32_t i = i0 + threadIdx.x * 4u;
        uint32_t v[4], n = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = i + j < many ? counts[i + j] : 0u; n += v[j]; }
        uint32_t at = base + sums_before(n, held, total);
        base += total;
#pragma unroll
        for (int j = 0; j < 4; ++j) { if (i + j < many) counts[i + j] = at; at += v[j]; }
    }
}
// ... and there they go.
__global__ __launch_bounds__(1024) void sort_place_kernel(SortParams p)
{
    extern __shared__ uint32_t counts[];
    const uint32_t first = blockIdx.x * kSortTile, last = min(first + kSortTile, p.N);
    sort_count(p, first, last, counts);
    for (uint32_t b = threadIdx.x; b < 1u << p.bits; b += kSortThreads) {
        uint32_t at = p.counts[(size_t)b * gridDim.x + blockIdx.x];
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            const uint32_t c = counts[(w << p.bits) + b];
            counts[(w << p.bits) + b] = at;
            at += c;
        }
    }
    __syncthreads();
    uint32_t from, to;
    sort_stretch(first, last, from, to);
    sort_part<true>(p, from, to, counts + ((threadIdx.x / 64u) << p.bits));
}

// --------------------------------------------------------------------- sums --
struct TableGradParams {
    const uint32_t *keys, *at;       // sorted by token
    const void     *g;
    int64_t         g_stride;        // elements
    float          *parts;           // sums of whole chunks of one token, [chunk][K]
    void           *dw;
    float           scale;
    uint32_t        N, V, K, chunk;  // log2 of a chunk's tokens
    uint32_t        width;           // log2 of the threads of a row
};

// The sum of g's rows at the sorted places a .. b - 1, eight columns from k on; loads of eight rows under way at a time.
template <int GT>
__device__ __forceinline__ void add_rows(const TableGradParams &p, uint32_t a, uint32_t b, uint32_t k, float (&s)[8])
{
    for (; a < b; a += 8u) {
        float x[8][8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) load8<GT>(p.g, (int64_t)p.at[min(a + e, b - 1u)] * p.g_stride, k, a + e < b ? p.K : 0u, x[e]);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += x[e][j];
    }
}

// A chunk of the sorted places that holds one token only: its sum, for a row that is much longer than the others.
template <int GT>
__global__ __launch_bounds__(256) void table_chunk_kernel(TableGradParams p)
{
    const uint32_t first = blockIdx.x << p.chunk, k = (blockIdx.y * 256u + threadIdx.x) * 8u;
    const uint32_t token = p.keys[first];
    if (token >= p.V || token != p.keys[first + (1u << p.chunk) - 1u] || k >= p.K) return;
    float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    add_rows<GT>(p, first, first + (1u << p.chunk), k, s);
    store8<RS_DTYPE_F32>(p.parts, (int64_t)blockIdx.x * p.K, k, p.K, s);
}

// Fifteen rows of dw: sixteen threads look for where each of them begins in the sorted tokens, and where the last ends.
constexpr uint32_t kTableRows = 15;
template <int GT, int DT>
__global__ __launch_bounds__(256) void table_grad_kernel(TableGradParams p)
{
    __shared__ uint32_t begins[kTableRows + 1];
    const uint32_t v0 = blockIdx.x * kTableRows;
    {
        // the first place whose token is `wanted` or more lies in lo .. hi; sixteen places between them are looked at at a time
        const uint32_t wanted = v0 + threadIdx.x / 16u, lane = threadIdx.x % 16u, group = threadIdx.x % 64u / 16u;
        uint32_t lo = 0, hi = p.N;
        while (lo < hi) {
            const uint32_t step = (hi - lo + 15u) / 16u, at = lo + lane * step;
            const bool less = at < hi && p.keys[at] < wanted;
            const uint32_t n = __popcll(__ballot(less) >> (16u * group) & 0xFFFFull);
            // the first n of them are less: it lies behind the n-th, and not behind the one after it
            if (n == 0) hi = lo;
            else {
                hi = min(hi, lo + n * step);
                lo = lo + (n - 1u) * step + 1u;
            }
        }
        if (lane == 0) begins[threadIdx.x / 16u] = lo;
    }
    __syncthreads();
    const uint32_t C = 1u << p.chunk;
    for (uint32_t r = threadIdx.x >> p.width; r < kTableRows && v0 + r < p.V; r += 256u >> p.width) {
        const uint32_t a = begins[r], b = begins[r + 1u];
        for (uint32_t k = (threadIdx.x & ((1u << p.width) - 1u)) * 8u; k < p.K; k += 8u << p.width) {
            float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            const uint32_t c0 = (a + C - 1u) >> p.chunk, c1 = b >> p.chunk;        // the whole chunks in between
            if (c0 < c1) {
                add_rows<GT>(p, a, c0 << p.chunk, k, s);
                for (uint32_t c = c0; c < c1; ++c) {
                    float x[8];
                    load8<RS_DTYPE_F32>(p.parts, (int64_t)c * p.K, k, p.K, x);
#pragma unroll
                    for (int j = 0; j < 8; ++j) s[j] += x[j];
                }
                add_rows<GT>(p, c1 << p.chunk, b, k, s);
            } else add_rows<GT>(p, a, b, k, s);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] *= p.scale;
            store8<DT>(p.dw, (int64_t)(v0 + r) * p.K, k, p.K, s);
        }
    }
}

}  // namespace rs
