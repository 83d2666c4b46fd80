// Log probabilities of given tokens, with the row's entropy, the token's rank and the likeliest alternatives, and the
// gradient of the logits.  z = x / T, m = max z, S = sum e^(z - m):
//
//   logprob = (z_t - m) - ln S            entropy H = ln S - sum e^(z - m) (z - m) / S
//   rank    = 1 + #{x > x_t} + #{x = x_t, i < t}
//   top     = the largest logits, equal ones by the lower index
//   dx_i    = ([i = t] g + sum_j [i = id_j] a_j - p_i (g + sum_j a_j + h (ln p_i + H))) / T,   p_i = e^(z_i - m) / S
//
// NaN counts as less than -inf in the orders; a row that holds NaN or +inf has NaN for its sums.  A row of nothing but
// -inf has no distribution: its log probabilities are -inf, its entropy 0, its gradient 0.
#pragma once

#include "rs_common.h"

namespace rs {

constexpr int kLpThreads = 256;          // of a workgroup; NT below is this or, for short rows, a single wave
constexpr int kLpTopMax  = RS_LOGPROBS_TOP_MAX;
template <int NT> constexpr int kLpCap = NT == kLpThreads ? 512 : 384;      // candidates that are put in order
constexpr int kLpSegs    = 8;            // stretches that a thread's windows of a slice are divided into, at most
constexpr int kLpStretches = 32;         // ... and a row's, where it is split
template <int NT> constexpr int kLpUnits = NT == kLpThreads ? 1024 : 512;   // stretches that are read again
constexpr float kLn2 = 0.693147180559945309f;

// What a workgroup of a split row leaves for the last of the row's workgroups.
struct alignas(16) LpSlice {
    float    m, s, t;                    // see LpSums
    uint32_t above;                      // tokens of the slice that come before the given one
    float    seg[kLpSegs][kLpThreads];   // largest logit of each stretch of each thread's windows
};
static_assert(sizeof(LpSlice) == 16 + 4 * kLpSegs * kLpThreads, "rs_logprobs_workspace_bytes");

struct LpParams {
    const void *logits;
    int64_t     stride_b, stride_t;      // elements from a batch, from a position to the next
    const void *tokens;
    int64_t     token_b, token_t;
    int32_t     tokens_64;               // int64 token ids, else int32
    int32_t     T, V;
    int32_t     top;
    float       c, inv_t;                // log2(e) / T, 1 / T
    float      *logprobs, *entropy;
    int32_t    *rank;
    float      *top_logprobs;
    int32_t    *top_tokens;
    float4     *stats;                   // for the gradient: max, log2 of the sum, entropy; or null
    uint32_t    row0;                    // the launch's first row
    uint32_t    S, J;                    // workgroups per row (at most kLpStretches); windows per thread and slice
    uint32_t    seg_log;                 // a stretch is 2^seg_log windows, four at least
    LpSlice    *slices;                  // split rows: what the workgroups of a row leave for the last of them
    uint32_t   *arrived;                 // ... and how many have, per row; zero between calls
};

struct LpGradParams {
    const void   *logits;
    int64_t       stride_b, stride_t;
    const void   *tokens;
    int64_t       token_b, token_t;
    int32_t       tokens_64;
    int32_t       T, V;
    int32_t       top;
    float         c, inv_t;
    const float4 *stats;
    const int32_t *top_tokens;
    const float  *g, *h, *a;             // gradients of logprob, entropy, alternatives; any may be null
    int32_t       g_stride, h_stride, a_stride;
    void         *grad;                  // contiguous rows of the logits' type
    uint32_t      row0;                  // the launch's first row
    uint32_t      chunks;                // workgroups per row
};

// ------------------------------------------------------------- element types --
// A window is 16 bytes of a row: 4 or 8 logits.  Rows begin at any multiple of the element's size, so windows are read
// and written without a claim on alignment: the hardware takes 16 bytes at any address.
template <int DT> struct Elem;
template <> struct Elem<RS_DTYPE_F32> {
    using T = float;
    static constexpr int kVec = 4, kBits = 32;     // bits of an order key that tell values apart
    static __device__ __forceinline__ void wide(const uint4 r, float (&x)[4])
    {
        x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint4 narrow(const float (&x)[4])
    {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    static __device__ __forceinline__ float one(T v) { return v; }
    static __device__ __forceinline__ T round(float x) { return x; }
};
template <> struct Elem<RS_DTYPE_BF16> {
    using T = uint16_t;
    static constexpr int kVec = 8, kBits = 16;
    static __device__ __forceinline__ void wide(const uint4 r, float (&x)[8])
    {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    }
    static __device__ __forceinline__ T round(float x)       // to nearest, ties to even; NaN stays one
    {
        const __bf16 b = (__bf16)x;
        return __builtin_bit_cast(uint16_t, b);
    }
    static __device__ __forceinline__ uint4 narrow(const float (&x)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)round(x[2 * i]) | (uint32_t)round(x[2 * i + 1]) << 16;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float one(T v) { return __uint_as_float((uint32_t)v << 16); }
};
template <> struct Elem<RS_DTYPE_F16> {
    using T = uint16_t;
    static constexpr int kVec = 8, kBits = 19;     // sign, 5 + 3 bits of exponent once widened, 10 of significand
    static __device__ __forceinline__ float one(T v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ T round(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
    static __device__ __forceinline__ void wide(const uint4 r, float (&x)[8])
    {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = one((T)w[i]); x[2 * i + 1] = one((T)(w[i] >> 16)); }
    }
    static __device__ __forceinline__ uint4 narrow(const float (&x)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)round(x[2 * i]) | (uint32_t)round(x[2 * i + 1]) << 16;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <int DT>
__device__ __forceinline__ uint4 load_window(const typename Elem<DT>::T *row, uint32_t n)
{
    uint4 r;
    __builtin_memcpy(&r, row + (size_t)n * Elem<DT>::kVec, 16);
    return r;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Order of the logits as whole numbers: 0 nothing, 1 NaN, then the numbers; -0 is 0.
__device__ __forceinline__ uint32_t lp_key(float x) { return x != x ? 1u : fkey(x + 0.0f); }
// ... and of the tokens: by the logit, equal ones by the lower index.  All are distinct.
__device__ __forceinline__ uint64_t lp_token(float x, uint32_t i) { return (uint64_t)lp_key(x) << 32 | (0xFFFFFFFFu - i); }

// ------------------------------------------------------------- running sums --
struct LpSums {
    float m, s, t;      // largest logit x; sum of e = 2^((x - m) c); sum of e (x - m) c
};

// The sums as they are for a maximum of `m` (at least a.m).  Where nothing but -inf was seen a.s and a.t are 0, and stay so.
__device__ __forceinline__ void lp_rebase(LpSums &a, float m, float c)
{
    const float d = fmaxf((a.m - m) * c, -1e30f);       // -inf - (-inf) and the like: NaN -> -1e30
    const float f = exp2_hw(d);
    a.t = f * __builtin_fmaf(a.s, d, a.t);
    a.s = f * a.s;
    a.m = m;
}

// N more logits; returns the largest.  Two exponents of a lane's window share the sums' chains; the terms of (x - m) c below -200
// have e = 0 and must not make 0 * inf.  (One operation less for z, with m c taken off in one step, and one less for t, with the
// rare NaN looked for afterwards, did not make a call faster: it is bound by what it reads, 5.2 to 5.5 TB/s.)
template <int N>
__device__ __forceinline__ float lp_take(LpSums &a, const float (&x)[N], float c)
{
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    lp_rebase(a, fmaxf(a.m, top), c);
    const float base = a.m == -__builtin_inff() ? 0.0f : a.m;
    float s[2] = {0.0f, 0.0f}, t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float z = (x[i] - base) * c;
        const float e = exp2_hw(z);
        s[i & 1] += e;
        t[i & 1] = __builtin_fmaf(e, fmaxf(z, -200.0f), t[i & 1]);
    }
    a.s += s[0] + s[1];
    a.t += t[0] + t[1];
    return top;
}

// Reductions over the 64 lanes, the result in all of them: within rows of 16 lanes, then across the rows; a lane without a
// source keeps its own maximum, adds nothing.
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_max(float v)
{
    return fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(v), (int)__float_as_uint(v), CTRL, ROWS, 0xf, false)));
}
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_sum(float v) { return v + __uint_as_float(dpp0_u32<CTRL, ROWS>(__float_as_uint(v))); }
__device__ __forceinline__ float wave_max_f(float v)
{
    v = dpp_max<0x111, 0xf>(v); v = dpp_max<0x112, 0xf>(v); v = dpp_max<0x114, 0xf>(v); v = dpp_max<0x118, 0xf>(v);
    v = dpp_max<0x142, 0xa>(v); v = dpp_max<0x143, 0xc>(v);
    return __uint_as_float(lane63_u32(__float_as_uint(v)));
}
__device__ __forceinline__ float wave_sum_f(float v)
{
    v = dpp_sum<0x111, 0xf>(v); v = dpp_sum<0x112, 0xf>(v); v = dpp_sum<0x114, 0xf>(v); v = dpp_sum<0x118, 0xf>(v);
    v = dpp_sum<0x142, 0xa>(v); v = dpp_sum<0x143, 0xc>(v);
    return __uint_as_float(lane63_u32(__float_as_uint(v)));
}

// The sums of a wave, in every lane.
__device__ __forceinline__ void lp_wave(LpSums &a, float c)
{
    lp_rebase(a, wave_max_f(a.m), c);
    a.s = wave_sum_f(a.s);
    a.t = wave_sum_f(a.t);
}

template <int NT>
struct LpShared {
    float    m[NT / kWave], s[NT / kWave], t[NT / kWave];
    uint32_t above[NT / kWave];
    uint32_t key[NT];            // order key of each thread's largest logit
    union {
        float    seg[kLpSegs][NT];      // largest logit of each stretch (rows that are not split)
        uint64_t lane_top[NT];
    };
    uint64_t cand[kLpCap<NT>];
    uint32_t unit[kLpUnits<NT>];             // stretches to read again: stretch << 8 | thread
    uint32_t n, n_units;
    uint32_t last;
};

// The sums of the workgroup, in every thread.
template <int NT>
__device__ __forceinline__ void lp_block(LpSums &a, uint32_t &above, float c, LpShared<NT> &sh)
{
    const uint32_t w = threadIdx.x / kWave;
    lp_wave(a, c);
    if (threadIdx.x % kWave == 0) { sh.m[w] = a.m; sh.s[w] = a.s; sh.t[w] = a.t; sh.above[w] = above; }
    __syncthreads();
    float m = sh.m[0];
#pragma unroll
    for (int i = 1; i < (NT / kWave); ++i) m = fmaxf(m, sh.m[i]);
    LpSums all{m, 0.0f, 0.0f};
    above = 0;
#pragma unroll
    for (int i = 0; i < (NT / kWave); ++i) {
        LpSums one{sh.m[i], sh.s[i], sh.t[i]};
        lp_rebase(one, m, c);
        all.s += one.s; all.t += one.t;
        above += sh.above[i];
    }
    a = all;
}

// --------------------------------------------------------- the alternatives --
// The `top` largest tokens of the row.  Each thread's largest logit is known from the pass, and that of each stretch of its
// windows.  The top-th largest of the threads', tau, is no larger than the top-th largest logit (that many threads hold one as
// large), so every token wanted is at least tau, and only stretches whose own largest is at least tau hold such tokens: about as
// many stretches as tokens are wanted.  Their windows alone are read again, spread over the workgroup.  What is at least tau goes
// to a list, a few tokens more than are wanted, and a token's place is the number of tokens in the list before it.
//
// A list that does not fit (rows of hundreds of equal logits, or of large ones that all fall to a few threads) is cut by the same
// bound over the threads of the second reading, with the index as part of the order, and, if it still does not fit, by halving
// the range of the bound until it does.  That ends: the orders are distinct.  (Cutting lists of more than 128 as well made rows of
// 131072 uniform bfloat16 logits slower, 26 us in the place of 18.)  Where there are more such stretches than can be noted, the
// whole row is read in their place: one of 131072 equal logits takes 69 us, 64 of them 84.
template <int DT, int NT>
struct LpRow {
    using E = Elem<DT>;
    const typename E::T *row;
    uint32_t V, full, J, seg_log, segs;  // logits; whole windows; windows of a thread in a slice, stretches in a slice

    // A list that has outgrown its room is made again: the rest of the row need not be looked at for it.
    static __device__ __forceinline__ bool full_list(const LpShared<NT> &sh) { return *(const volatile uint32_t *)&sh.n > (uint32_t)kLpCap<NT>; }
    template <typename F> __device__ __forceinline__ void tail(F f) const
    {
        const uint32_t i = full * E::kVec + threadIdx.x;
        if (i < V) f(E::one(row[i]), i);
    }
    // f(logit, index) for the windows of the stretches in sh.unit and the row's last few logits
    template <typename F> __device__ __forceinline__ void units(const LpShared<NT> &sh, uint32_t n_units, float least, bool listing, F f) const
    {
        constexpr int U = 4;
        const uint32_t items = n_units << seg_log, mask = (1u << seg_log) - 1u;
        for (uint32_t i = threadIdx.x; i < items; i += U * NT) {
            if (listing && full_list(sh)) break;
            uint4 raw[U];
            uint32_t n[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t at = i + u * NT;
                n[u] = full;
                if (at < items) {
                    const uint32_t unit = sh.unit[at >> seg_log], slice = (unit >> 8) / segs, j = (((unit >> 8) - slice * segs) << seg_log) + (at & mask);
                    if (j < J) n[u] = (slice * J + j) * NT + (unit & 255u);
                }
                if (n[u] < full) raw[u] = load_window<DT>(row, n[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (n[u] >= full) continue;
                float x[E::kVec];
                E::wide(raw[u], x);
                float most = x[0];
#pragma unroll
                for (int k = 1; k < E::kVec; ++k) most = fmaxf(most, x[k]);
                if (most >= least)
#pragma unroll
                    for (int k = 0; k < E::kVec; ++k) if (x[k] >= least) f(x[k], n[u] * E::kVec + k);
            }
        }
        tail(f);
    }
    // ... for the whole row
    template <typename F> __device__ __forceinline__ void all(const LpShared<NT> &sh, bool listing, F f) const
    {
        constexpr int U = 4;
        for (uint32_t n0 = threadIdx.x; n0 < full; n0 += U * NT) {
            if (listing && full_list(sh)) break;
            uint4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) if (n0 + u * NT < full) raw[u] = load_window<DT>(row, n0 + u * NT);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t n = n0 + u * NT;
                if (n >= full) continue;
                float x[E::kVec];
                E::wide(raw[u], x);
#pragma unroll
                for (int k = 0; k < E::kVec; ++k) f(x[k], n * E::kVec + k);
            }
        }
        tail(f);
    }
};

// A t with at least `k` and, unless keys are equal, at most k + spare of the workgroup's keys >= t; only the upper BITS bits matter.
// No key is larger than `most`.
template <int BITS, int NT, typename K>
__device__ __forceinline__ K lp_kth(const K *key, uint32_t k, uint32_t spare, K most)
{
    constexpr int kAll = (int)sizeof(K) * 8;
    K mine[NT / kWave];
#pragma unroll
    for (int i = 0; i < (NT / kWave); ++i) mine[i] = key[i * kWave + threadIdx.x % kWave];
    K t = 0;
    for (int bit = kAll - 1; bit >= kAll - BITS; --bit) {
        const K c = t | (K)1 << bit;
        if (c > most) continue;
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < (NT / kWave); ++i) n += (uint32_t)__popcll(__ballot(mine[i] >= c));
        if (n >= k) t = c;
        if (n >= k && n <= k + spare) break;
    }
    return t;
}

// The k-th largest of the workgroup's keys, found by taking the largest away again and again: for a few of them faster than by
// the bits (1 x 65536 float32 logits with 5 alternatives 8.7 us in the place of 9.4; as fast with 8 to 12).
template <int NT>
__device__ __forceinline__ uint32_t lp_kth_of_few(const uint32_t *key, uint32_t k)
{
    uint32_t mine[NT / kWave], n = 0, t;
#pragma unroll
    for (int i = 0; i < NT / kWave; ++i) mine[i] = key[i * kWave + threadIdx.x % kWave];
    do {
        uint32_t most = mine[0];
#pragma unroll
        for (int i = 1; i < NT / kWave; ++i) most = max(most, mine[i]);
        t = wave_max_u32(most);
#pragma unroll
        for (int i = 0; i < NT / kWave; ++i) {
            n += (uint32_t)__popcll(__ballot(mine[i] == t));
            mine[i] = mine[i] == t ? 0u : mine[i];
        }
    } while (n < k);
    return t;
}

// seg[s] is the thread's largest logit of stretch s of the row, `largest` the largest of those.
template <int DT, int NT, int N>
__device__ __forceinline__ void lp_alternatives(const LpRow<DT, NT> &row, float largest, const float (&seg)[N], const LpSums &a, float log_s, float inv_t,
                                                uint32_t top, float *out_logprobs, int32_t *out_tokens, LpShared<NT> &sh)
{
    const uint32_t tid = threadIdx.x, lane = tid % kWave;
    sh.key[tid] = lp_key(largest);
    if (tid == 0) sh.n = sh.n_units = 0;
    __syncthreads();
    // (one alternative is the largest logit itself)
    uint32_t tau = top == 1u ? uniform(lp_key(a.m)) : top <= 8u ? lp_kth_of_few<NT>(sh.key, top)
                                                    : lp_kth<Elem<DT>::kBits, NT>(sh.key, top, top / 4u, uniform(lp_key(a.m)));
    if (tau <= fkey(-__builtin_inff())) tau = 1u;        // fewer numbers than are wanted, perhaps: NaN too
    const float least = fkey_inv(tau);
    if (tau != 1u) {
        // one place in the list for each stretch; one addition to its length for each wave
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) mine |= seg[i] >= least ? 1u << i : 0u;
        const uint32_t count = (uint32_t)__popc(mine), upto = wave_inclusive_scan(count), all = lane63(upto);
        uint32_t at = 0;
        if (all) {
            if (lane == 0) at = atomicAdd(&sh.n_units, all);
            at = uniform(at) + upto - count;
            for (; mine; mine &= mine - 1u, ++at)
                if (at < (uint32_t)kLpUnits<NT>) sh.unit[at] = (uint32_t)__builtin_ctz(mine) << 8 | tid;
        }
        __syncthreads();
    }
    auto list = [&](uint64_t from) {
        return [&sh, from](float x, uint32_t i) {
            const uint64_t k = lp_token(x, i);
            if (k >= from) {
                const uint32_t at = atomicAdd(&sh.n, 1u);
                if (at < kLpCap<NT>) sh.cand[at] = k;
            }
        };
    };
    const uint64_t from = (uint64_t)tau << 32;
    const uint32_t n_units = sh.n_units;
    auto walk = [&](bool listing, auto f) {
        if (tau != 1u && n_units <= (uint32_t)kLpUnits<NT>) row.units(sh, n_units, least, listing, f);
        else row.all(sh, listing, f);
    };
    walk(true, list(from));
    __syncthreads();
    if (sh.n > (uint32_t)kLpCap<NT>) {
        uint64_t best = 0;
        walk(false, [&](float x, uint32_t i) { best = max(best, lp_token(x, i)); });
        __syncthreads();                                 // (the stretches' room is used again)
        sh.lane_top[tid] = best;
        __syncthreads();
        uint64_t lo = max(lp_kth<64, NT>(sh.lane_top, top, 0u, (uint64_t)~0ull), from), hi = ~0ull;
        for (uint64_t t = lo;; t = lo + (hi - lo) / 2) {
            __syncthreads();
            if (tid == 0) sh.n = 0;
            __syncthreads();
            walk(true, list(t));
            __syncthreads();
            if (sh.n > (uint32_t)kLpCap<NT>) lo = t;
            else if (sh.n < top) hi = t;
            else break;
        }
    }
    const uint32_t n = sh.n;
    auto put = [&](uint64_t k, uint32_t place) {
        if (place >= top) return;
        const float x = (uint32_t)(k >> 32) == 1u ? __builtin_nanf("") : fkey_inv((uint32_t)(k >> 32));
        out_tokens[place] = (int32_t)(0xFFFFFFFFu - (uint32_t)k);
        out_logprobs[place] = x == -__builtin_inff() && a.s == a.s ? x : (x - a.m) * inv_t - log_s;
    };
    for (uint32_t i = tid; i < n; i += NT) {
        const uint64_t k = sh.cand[i];
        uint32_t place = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < n; ++j) place += sh.cand[j] > k;
        put(k, place);
    }
}

// ------------------------------------------------------------------- forward --
// U windows of each thread, whole ones below `full` only.  A batch is asked for before the one before it is worked on.
template <int DT, int NT, int U>
__device__ __forceinline__ void lp_ask(const typename Elem<DT>::T *row, uint32_t n0, uint32_t full, uint4 (&raw)[U])
{
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t n = n0 + u * NT;
        if (n < full) raw[u] = load_window<DT>(row, n);
    }
}

// Returns the largest logit of the batch.  GUARD: lanes whose window is not below `full` have none.
template <int DT, int NT, int U, bool GUARD>
__device__ __forceinline__ float lp_batch(const uint4 *raw, uint32_t n0, uint32_t full, uint32_t token_window, float before, float after,
                                          float c, LpSums &a, uint32_t &above)
{
    using E = Elem<DT>;
    float x[U * E::kVec], edge[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t n = n0 + u * NT;
        float v[E::kVec];
        E::wide(raw[u], v);
        edge[u] = n < token_window ? before : after;
        if (GUARD && n >= full) edge[u] = __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) x[u * E::kVec + i] = GUARD && n >= full ? -__builtin_inff() : v[i];
    }
    const float top = lp_take(a, x, c);
#pragma unroll
    for (int i = 0; i < U * E::kVec; ++i) above += (uint32_t)__popcll(__ballot(x[i] >= edge[i / E::kVec]));
    return top;
}

__device__ __forceinline__ float lp_stretch(const LpSlice *slices, uint32_t segs, uint32_t s, uint32_t tid)
{
    const uint32_t slice = s / segs;
    return a_load(&slices[slice].seg[s - slice * segs][tid]);
}

// One workgroup of NT threads per row, or S of them (SPLIT), each on a stretch of the row, of which the last to arrive finishes the
// row.  Nothing waits.  One pass over the logits with each thread's running maximum and sums, two batches of 64 bytes a thread
// under way.  Bound by the memory where there are rows enough: 8192 x 131072 bfloat16 logits with 20 alternatives 382 us,
// 5.6 TB/s; a call of one row by its chain of loads: the token, its logit, the slices' sums, the stretches, their windows
// (1 x 65536 float32 with 5 alternatives 8.7 us, without any 4.8).
template <int DT, int NT, bool SPLIT>
__global__ __launch_bounds__(NT) void logprobs_kernel(LpParams p)
{
    using E = Elem<DT>;
    constexpr int U = 4;
    static_assert(!SPLIT || NT == kLpThreads, "what the slices leave is of that many threads");
    __shared__ LpShared<NT> sh;
    const uint32_t r = SPLIT ? blockIdx.x / p.S : p.row0 + blockIdx.x, slice = SPLIT ? blockIdx.x - r * p.S : 0;
    const uint32_t b = r / (uint32_t)p.T, pos = r - b * (uint32_t)p.T;
    const uint32_t V = (uint32_t)p.V, full = V / E::kVec, tid = threadIdx.x;
    const typename E::T *row = (const typename E::T *)p.logits + (int64_t)b * p.stride_b + (int64_t)pos * p.stride_t;
    const uint32_t first = slice * p.J * NT, end = min(full, first + p.J * NT);
    uint4 raw[U];
    lp_ask<DT, NT, U>(row, first + tid, end, raw);
    const uint32_t last = full * E::kVec + tid;          // the row's last few logits
    const bool has_last = (!SPLIT || slice == p.S - 1u) && last < V;
    const float x_last = has_last ? E::one(row[last]) : -__builtin_inff();
    const int64_t at = (int64_t)b * p.token_b + (int64_t)pos * p.token_t;
    const int64_t token = p.tokens_64 ? ((const int64_t *)p.tokens)[at] : (int64_t)((const int32_t *)p.tokens)[at];
    const bool given = token >= 0 && token < (int64_t)V;
    const uint32_t tok = given ? (uint32_t)token : 0u;
    const float x_t = E::one(row[tok]);
    const uint32_t token_window = tok / E::kVec, beside = token_window * E::kVec + tid;
    const bool is_beside = tid < (uint32_t)E::kVec && beside < tok && token_window >= first && token_window < end;
    const float x_beside = is_beside ? E::one(row[beside]) : __builtin_nanf("");
    // a window before the token's counts x >= x_t, one behind it x > x_t, that is x >= the next number up; the token's own
    // window counts the latter, and the equal ones before the token are added.  Below -inf there is nothing but NaN.
    float before = x_t, after;
    {
        const uint32_t bits = __float_as_uint(x_t + 0.0f);
        after = __uint_as_float(bits & 0x80000000u ? bits - 1u : bits + 1u);
        if (x_t != x_t) before = after = -__builtin_inff();
    }

    LpSums a{-__builtin_inff(), 0.0f, 0.0f};
    uint32_t above = 0, n = first;
    float seg = -__builtin_inff();
    for (; n + U * NT <= end; ) {
        uint4 now[U];
#pragma unroll
        for (int u = 0; u < U; ++u) now[u] = raw[u];
        lp_ask<DT, NT, U>(row, n + U * NT + tid, end, raw);
        seg = fmaxf(seg, lp_batch<DT, NT, U, false>(now, n + tid, end, token_window, before, after, p.c, a, above));
        n += U * NT;
        const uint32_t j = (n - first) / NT;
        if (!(j & ((1u << p.seg_log) - 1u))) {
            if (p.top) sh.seg[(j >> p.seg_log) - 1u][tid] = seg;
            seg = -__builtin_inff();
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (n + u * NT < end) seg = fmaxf(seg, lp_batch<DT, NT, 1, true>(raw + u, n + u * NT + tid, end, token_window, before, after, p.c, a, above));
    const uint32_t segs = (p.J + (1u << p.seg_log) - 1u) >> p.seg_log;
    if (p.top) {
        // the stretch that the slice ends in, and those behind it
        for (uint32_t g = end > first ? (end - first) / NT >> p.seg_log : 0u; g < segs; ++g) {
            sh.seg[g][tid] = seg;
            seg = -__builtin_inff();
        }
    }
    const float largest = a.m;
    if (!SPLIT || slice == p.S - 1u) {
        const float x[1] = {x_last};
        lp_take(a, x, p.c);
        above += (uint32_t)__popcll(__ballot(x_last >= (has_last ? (last < tok ? before : after) : __builtin_nanf(""))));
    }
    above += (uint32_t)__popcll(__ballot(x_beside == x_t));
    lp_block(a, above, p.c, sh);

    float mine = largest;
    float seg_of[SPLIT ? kLpStretches : kLpSegs];
    if constexpr (SPLIT) {
        LpSlice *slices = p.slices + (size_t)r * p.S;
        if (p.top) for (uint32_t g = 0; g < segs; ++g) a_store(&slices[slice].seg[g][tid], sh.seg[g][tid]);
        if (tid == 0) {
            a_store(&slices[slice].m, a.m); a_store(&slices[slice].s, a.s); a_store(&slices[slice].t, a.t);
            a_store(&slices[slice].above, above);
        }
        wait_vmem();
        __syncthreads();
        if (tid == 0) {
            sh.last = __hip_atomic_fetch_add(&p.arrived[r], 1u, __ATOMIC_RELAXED, RS_AGENT) == p.S - 1u;
            if (sh.last) a_store(&p.arrived[r], 0u);
        }
        __syncthreads();
        if (!sh.last) return;
        // the row's sums, from the slices' in every wave; the largest logit of each thread over the slices
        a = LpSums{-__builtin_inff(), 0.0f, 0.0f};
        above = 0;
        const uint32_t lane = tid % kWave;
        if (lane < p.S) {
            a = LpSums{a_load(&slices[lane].m), a_load(&slices[lane].s), a_load(&slices[lane].t)};
            above = a_load(&slices[lane].above);
        }
        // (all under way at once: what other workgroups have written comes from far)
        if (p.top) {
#pragma unroll
            for (int s = 0; s < kLpStretches; ++s) seg_of[s] = s < (int)(p.S * segs) ? lp_stretch(slices, segs, s, tid) : -__builtin_inff();
#pragma unroll
            for (int s = 0; s < kLpStretches; ++s) mine = fmaxf(mine, seg_of[s]);
        }
        lp_wave(a, p.c);
        above = wave_sum(above);
    }

    const float log_s = logf(a.s);
    const bool empty = a.s == 0.0f;                     // nothing but -inf
    if (tid < kWave) {
        if (x_t != x_t)                                 // NaN: behind every number, among its like by the index
            for (uint32_t j = tid; j < ((tok + kWave - 1u) & ~(kWave - 1u)); j += kWave) {
                const float x = j < tok ? E::one(row[j]) : 0.0f;
                above += (uint32_t)__popcll(__ballot(x != x));
            }
        if (tid == 0) {
            const float h = log_s - a.t * kLn2 / a.s;
            const float lp = x_t == -__builtin_inff() && a.s == a.s ? x_t : (x_t - a.m) * p.inv_t - log_s;
            const float entropy = empty ? 0.0f : h;
            if (p.logprobs) p.logprobs[r] = given ? lp : token < 0 ? 0.0f : __builtin_nanf("");
            if (p.entropy) p.entropy[r] = entropy;
            if (p.rank) p.rank[r] = given ? (int32_t)above + 1 : 0;
            if (p.stats) p.stats[r] = empty ? make_float4(0.0f, __builtin_inff(), 0.0f, 0.0f) : make_float4(a.m, log2f(a.s), entropy, 0.0f);
        }
    }
    if (p.top) {
        const LpRow<DT, NT> whole{row, V, full, p.J, p.seg_log, segs};
        float *const lps = p.top_logprobs + (size_t)r * p.top;
        int32_t *const ids = p.top_tokens + (size_t)r * p.top;
        if constexpr (!SPLIT)
#pragma unroll
            for (int s = 0; s < kLpSegs; ++s) seg_of[s] = s < (int)segs ? sh.seg[s][tid] : -__builtin_inff();
        lp_alternatives<DT, NT>(whole, mine, seg_of, a, log_s, p.inv_t, (uint32_t)p.top, lps, ids, sh);
    }
}

// ------------------------------------------------------------------ gradient --
// dx_i = p_i (alpha + beta log2 p_i), with alpha = -(g + sum a + h H) / T and beta = -h ln2 / T: one exponential and a few products
// per logit, read once and written once, a wave for 256 windows.  The few tokens that were named are then written once more,
// whole, by the wave that wrote them first.  Bound by the memory: 8192 x 131072 bfloat16 logits 724 us, 5.9 TB/s.  (Workgroups of
// four waves were up to 4 % slower on long rows, and 275 us in the place of 93 on 262144 x 256.)
constexpr uint32_t kLpGradWindows = 4 * kWave;

template <int DT>
__global__ __launch_bounds__(kWave) void logprobs_grad_kernel(LpGradParams p)
{
    using E = Elem<DT>;
    constexpr int U = 4;
    const uint32_t in = blockIdx.x / p.chunks, chunk = blockIdx.x - in * p.chunks, r = p.row0 + in;
    const uint32_t b = r / (uint32_t)p.T, pos = r - b * (uint32_t)p.T;
    const uint32_t V = (uint32_t)p.V, full = V / E::kVec, lane = threadIdx.x;
    const typename E::T *row = (const typename E::T *)p.logits + (int64_t)b * p.stride_b + (int64_t)pos * p.stride_t;
    typename E::T *out = (typename E::T *)p.grad + (size_t)r * V;
    const uint32_t n0 = chunk * (U * kWave) + lane;
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) if (n0 + u * kWave < full) raw[u] = load_window<DT>(row, n0 + u * kWave);

    const float4 st = p.stats[r];
    const int64_t at = (int64_t)b * p.token_b + (int64_t)pos * p.token_t;
    const int64_t token = p.tokens_64 ? ((const int64_t *)p.tokens)[at] : (int64_t)((const int32_t *)p.tokens)[at];
    float g = p.g && token >= 0 ? p.g[(int64_t)r * p.g_stride] : 0.0f;
    if (p.g && token >= (int64_t)V) g = __builtin_nanf("");      // (the entropy and the alternatives do not know the token)
    const float h = p.h ? p.h[(int64_t)r * p.h_stride] : 0.0f;
    float a = 0.0f;
    int64_t id = -1;
    if (p.a && lane < (uint32_t)p.top) {
        id = p.top_tokens[(size_t)r * p.top + lane];
        a = p.a[((int64_t)r * p.top + lane) * p.a_stride];
    }
    float a_sum = p.a ? wave_sum_f(a) : 0.0f;
    const float alpha = -(g + a_sum + h * st.z) * p.inv_t, beta = -h * kLn2 * p.inv_t;
    const float m = st.x, log2_s = st.y;
    auto grad = [&](float x) {
        const float z = (x - m) * p.c - log2_s;
        return exp2_hw(z) * __builtin_fmaf(beta, fmaxf(z, -200.0f), alpha);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t n = n0 + u * kWave;
        if (n < full) {
            float x[E::kVec];
            E::wide(raw[u], x);
#pragma unroll
            for (int i = 0; i < E::kVec; ++i) x[i] = grad(x[i]);
            const uint4 v = E::narrow(x);
            __builtin_memcpy(out + (size_t)n * E::kVec, &v, 16);
        }
    }
    const bool last = chunk == p.chunks - 1u;
    if (last) {
        const uint32_t i = full * E::kVec + lane;
        if (i < V) out[i] = E::round(grad(E::one(row[i])));
    }
    // the named tokens of this chunk
    const int64_t begin = (int64_t)chunk * (U * kWave * E::kVec);
    const int64_t end = last ? (int64_t)V : begin + U * kWave * E::kVec;
    const bool token_here = token >= begin && token < end;
    const bool id_here = id >= begin && id < end;
    const uint64_t any = __ballot(id_here || token_here);
    if (any == 0 || log2_s == __builtin_inff()) return;
    wait_vmem();
    const uint64_t both = __ballot(id_here && id == token);
    if (id_here) out[id] = E::round(grad(E::one(row[id])) + (a + (id == token ? g : 0.0f)) * p.inv_t);
    if (token_here && !both && lane == 0) out[token] = E::round(grad(E::one(row[token])) + g * p.inv_t);
}

}  // namespace rs
