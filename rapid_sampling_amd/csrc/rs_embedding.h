// Rows of a table by token, and the table's gradient.
//
//   y[i] = s w[t_i]          dw[v] = s sum over i with t_i = v of g_i, in the order of i, in float32
//
// The gradient's positions are put in the order of their tokens first (a radix sort that keeps the order of equal ones), so that a row of
// dw is one stretch of them: no floating-point atomics, and the same sums every time.  Bound by memory: y and g once, dw once.
#pragma once

#include "rs_linear.h"
#include "rs_sort.h"

namespace rs {

constexpr int kTableInt8 = 3, kTableFp8 = 4;         // types of a table, next to RS_DTYPE_*

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

// Eight values of a row as they lie in memory, and widened.  Reading and widening are apart so that several reads are under way at a
// time.  A thread has the columns from k on, the last of a row the last eight of it: what two threads have both is the same in both.
template <int DT> struct Eight { v4i v[DT == RS_DTYPE_F32 ? 2 : 1]; };
__device__ __forceinline__ uint32_t eight_from(uint32_t k, uint32_t K) { return K >= 8u ? min(k, K - 8u) : 0u; }
template <int DT> __device__ __forceinline__ Eight<DT> read8(const void *base, int64_t at, uint32_t k, uint32_t K)
{
    Eight<DT> r;
    const char *p = (const char *)base + (at + k) * (DT == RS_DTYPE_F32 ? 4 : 2);
    if (K >= 8u) __builtin_memcpy(&r, p, sizeof(r));
    else {
        uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (uint32_t j = 0; j < 7; ++j)
            if (j < K) {
                if constexpr (DT == RS_DTYPE_F32) w[j] = ((const uint32_t *)p)[j];
                else w[j / 2] |= (uint32_t)((const uint16_t *)p)[j] << (16 * (j % 2));
            }
        __builtin_memcpy(&r, w, sizeof(r));
    }
    return r;
}
template <int DT> __device__ __forceinline__ void widen8(const Eight<DT> &r, float (&x)[8])
{
    if constexpr (DT == RS_DTYPE_F32) __builtin_memcpy(x, &r, 32);
    else {
        uint16_t v[8];
        __builtin_memcpy(v, &r, 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = DT == RS_DTYPE_BF16 ? __uint_as_float((uint32_t)v[j] << 16) : (float)__builtin_bit_cast(_Float16, v[j]);
    }
}

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

// 2^width threads to a row, eight values at a time.  Bound by the launch or by memory: 64 rows of 4096 in int8 2.6 us, 8192 in bfloat16 31 (4.3 TB/s,
// read and written), in int8 or e4m3 into bfloat16 16.5 (6.1).
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
// Pairs of a token and its place, a digit of up to 11 bits at a time.  A workgroup of 16 waves takes a stretch of the list, each wave a part of it, 64 tokens at
// a time; a counter for each digit and wave in LDS.
constexpr uint32_t kSortBatch = 8, kSortWaves = 16, kSortThreads = 64 * kSortWaves, kSortBits = 11, kSortTile = 4096, kSortAlone = 16384;

struct SortParams {
    TokenList       tokens;          // of the first digit: what is sorted; a token that is none counts as V
    const uint2    *in;              // (token, place)
    uint2          *out;             // sorted by this digit
    uint32_t       *counts;          // [digit][workgroup]
    uint32_t        N, V, shift, bits, first;
    uint2          *out_b;           // a workgroup that does it all alone: the other side
    uint32_t        digits;          // ... and how many digits
};

__device__ __forceinline__ uint2 sort_pair(const SortParams &p, uint32_t i)
{
    if (!p.first) return p.in[i];
    const int64_t t = p.tokens[i];
    return make_uint2(t >= 0 && t < (int64_t)p.V ? (uint32_t)t : p.V, i);
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
    for (uint32_t i0 = from; i0 < to; i0 += 64u * kSortBatch) {
        // (a batch's tokens are asked for at once: each would cost a trip to memory by itself)
        uint2 pairs[kSortBatch];
#pragma unroll
        for (uint32_t e = 0; e < kSortBatch; ++e) {
            const uint32_t i = i0 + e * 64u + lane;
            pairs[e] = i < to ? sort_pair(p, i) : make_uint2(0u, 0u);
        }
#pragma unroll
        for (uint32_t e = 0; e < kSortBatch; ++e) {
            if (i0 + e * 64u >= to) continue;
            const bool live = i0 + e * 64u + lane < to;
            const uint32_t digit = pairs[e].x >> p.shift & mask;
            const uint64_t same = same_digit(digit, p.bits, live);
            const uint32_t before = __popcll(same & ((1ull << lane) - 1ull));
            const uint32_t have = live ? counts[digit] : 0u;
            if (PLACE && live) p.out[have + before] = pairs[e];
            __builtin_amdgcn_wave_barrier();
            if (live && before == 0) counts[digit] = have + (uint32_t)__popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
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

// dw is cleared first, all of it, and the rows that have a token written once more: they are few next to a vocabulary.
struct ClearParams {
    char    *at;
    uint64_t bytes;
};
__device__ __forceinline__ void clear_part(const ClearParams &c, uint32_t group, uint32_t groups)
{
    const uint32_t head = (uint32_t)min((uint64_t)(-(uintptr_t)c.at & 15u), c.bytes);
    const uint64_t pieces = (c.bytes - head) / 16u;
    for (uint64_t i = (uint64_t)group * kSortThreads + threadIdx.x; i < pieces; i += (uint64_t)groups * kSortThreads)
        *(uint4 *)(c.at + head + i * 16u) = make_uint4(0u, 0u, 0u, 0u);
    if (group == 0 && threadIdx.x < 32u) {
        const uint64_t at = threadIdx.x < 16u ? threadIdx.x : head + pieces * 16u + threadIdx.x - 16u;
        if (threadIdx.x < 16u ? at < head : at < c.bytes) c.at[at] = 0;
    }
}
__global__ __launch_bounds__(1024) void clear_kernel(ClearParams c) { clear_part(c, blockIdx.x, gridDim.x); }

// One workgroup, all digits; the others of the launch clear dw meanwhile.  It takes some 5 ns for a token of 17 bits.
__global__ __launch_bounds__(1024) void sort_alone_kernel(SortParams p, ClearParams c)
{
    extern __shared__ uint32_t counts[];
    __shared__ uint32_t held[kSortWaves];
    if (blockIdx.x) {
        clear_part(c, blockIdx.x - 1u, gridDim.x - 1u);
        return;
    }
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
        // the next digit reads what the other waves of this workgroup have written
        __threadfence_block();
        __syncthreads();
        p.first = 0;
        p.shift += p.bits;
        p.in = p.out;
        p.out = p.out_b;
        p.out_b = (uint2 *)p.in;
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
// The sorted places are cut into chunks of one size, whatever their tokens; a workgroup sums those of one chunk, for 2048 columns.  A
// token whose places lie within a chunk is written at once.  One that goes on into the next leaves a part, and so does every
// chunk that it comes from another into; a second launch joins these in their order.  Bound by memory: 8192 rows of 4096 in bfloat16 36 us
// and 8 (g is read once, at random, and as much of dw is written).
struct TableGradParams {
    const uint2    *pairs;           // (token, place), sorted by token
    const void     *g;
    int64_t         g_stride;        // elements
    float          *parts;           // [chunk][2][K]: of the token that comes from the chunk before; of the one that goes on
    void           *dw;
    float           scale;
    uint32_t        N, V, K, chunk;  // chunk: log2 of a chunk's places
};

template <int DT>
__device__ __forceinline__ void table_row(const TableGradParams &p, uint32_t token, uint32_t k, const float (&s)[8])
{
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = s[j] * p.scale;
    store8<DT>(p.dw, (int64_t)token * p.K, k, p.K, y);
}

template <int GT, int DT>
__global__ __launch_bounds__(256) void table_chunk_kernel(TableGradParams p)
{
    const uint32_t first = blockIdx.x << p.chunk, last = min(first + (1u << p.chunk), p.N), own = (blockIdx.y * 256u + threadIdx.x) * 8u;
    if (own >= p.K) return;
    const uint32_t k = eight_from(own, p.K);
    const bool goes_on = last < p.N && p.pairs[last].x == p.pairs[last - 1u].x;
    uint32_t token = p.pairs[first].x;
    bool from_before = first > 0u && p.pairs[first - 1u].x == token;
    float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    auto leave = [&](bool to_next) {
        if (token >= p.V) return;
        if (from_before || to_next) store8<RS_DTYPE_F32>(p.parts, ((int64_t)blockIdx.x * 2 + (from_before ? 0 : 1)) * p.K, k, p.K, s);
        else table_row<DT>(p, token, k, s);
    };
    // (the keys and places are the same for the whole workgroup; behind the last place: its token once more, not added)
    constexpr uint32_t kBatch = 16;
    for (uint32_t i = first; i < last; i += kBatch) {
        Eight<GT> x[kBatch];
        uint2 pairs[kBatch];
#pragma unroll
        for (uint32_t e = 0; e < kBatch; ++e) pairs[e] = p.pairs[min(i + e, last - 1u)];
#pragma unroll
        for (uint32_t e = 0; e < kBatch; ++e) x[e] = read8<GT>(p.g, (int64_t)pairs[e].y * p.g_stride, k, p.K);
#pragma unroll
        for (uint32_t e = 0; e < kBatch; ++e) {
            if (pairs[e].x != token) {
                leave(false);
                token = pairs[e].x;
                from_before = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] = 0.0f;
            }
            float v[8];
            widen8<GT>(x[e], v);
            if (i + e < last)
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] += v[j];
        }
    }
    leave(goes_on);
}

// The chunk in which a token begins that goes on into the next joins its parts.
template <int DT>
__global__ __launch_bounds__(256) void table_join_kernel(TableGradParams p)
{
    const uint32_t C = 1u << p.chunk, c0 = blockIdx.x, first = c0 << p.chunk, last = first + C, own = (blockIdx.y * 256u + threadIdx.x) * 8u;
    if (last >= p.N) return;
    const uint32_t token = p.pairs[last - 1u].x;
    if (token >= p.V || p.pairs[last].x != token || (first > 0u && p.pairs[first - 1u].x == token) || own >= p.K) return;
    const uint32_t k = eight_from(own, p.K);
    float s[8];
    widen8<RS_DTYPE_F32>(read8<RS_DTYPE_F32>(p.parts, ((int64_t)c0 * 2 + 1) * p.K, k, p.K), s);
    for (uint32_t c = c0 + 1u; ; c += 8u) {
        Eight<RS_DTYPE_F32> x[8];
        bool there[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const uint64_t at = (uint64_t)(c + e) << p.chunk;
            there[e] = at < p.N && p.pairs[min(at, (uint64_t)p.N - 1u)].x == token;
        }
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) x[e] = read8<RS_DTYPE_F32>(p.parts, (int64_t)(there[e] ? c + e : c0) * 2 * p.K, k, p.K);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            float v[8];
            widen8<RS_DTYPE_F32>(x[e], v);
            if (there[e])
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] += v[j];
        }
        if (!there[7]) break;
    }
    table_row<DT>(p, token, k, s);
}

}  // namespace rs
