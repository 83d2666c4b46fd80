// Instantiations, launchers and C entry points of the log probabilities and their gradient.
#include "rs_logprobs.h"

#include <algorithm>
#include <cmath>

namespace rs {

constexpr uint32_t kLpSplitMost = 512;   // workgroups of a call whose rows are split

// Workgroups per row: one, or enough for about two to a compute unit, each with at least four windows per thread.  (With four to a
// compute unit 64 rows of 152064 bfloat16 logits and 20 alternatives took 18.5 us in the place of 17.0, 385 of 50257 23.1 in the
// place of 19.6, with one 16.8 and 19.6; 48 of 32768 float32 are as fast either way.)
static uint32_t lp_split(uint32_t rows, uint32_t windows)
{
    const uint32_t most = kLpSplitMost / rows, per = (windows + 4u * kLpThreads - 1u) / (4u * kLpThreads);
    return std::max(1u, std::min(std::min(most, per), (uint32_t)kLpStretches));
}

static int lp_check(const void *logits, int32_t dtype, const void *tokens, int32_t tokens_64, int64_t B, int64_t T, int64_t V, double temperature, int32_t top)
{
    if (!(V > 0 && V <= 1048576)) return RS_ERR_VOCAB;
    if (B <= 0 || T <= 0 || B > 0x7FFFFFFF || T > 0x7FFFFFFF || B * T > 0x7FFFFFFF) return RS_ERR_BATCH;
    if (!(temperature >= 0.001 && temperature <= 1000.0)) return RS_ERR_TEMPERATURE;
    if (!logits || !tokens) return RS_ERR_NULL;
    if (dtype != RS_DTYPE_F32 && dtype != RS_DTYPE_BF16 && dtype != RS_DTYPE_F16) return RS_ERR_ARG;
    if (tokens_64 != 0 && tokens_64 != 1) return RS_ERR_ARG;
    if (top < 0 || top > kLpTopMax || top > V) return RS_ERR_ARG;
    if (((uintptr_t)logits & (dtype == RS_DTYPE_F32 ? 3 : 1)) || ((uintptr_t)tokens & (tokens_64 ? 7 : 3))) return RS_ERR_ALIGN;
    return RS_OK;
}

// f(first row, rows) for as many rows at a time as a launch of `threads` to a row holds.
template <typename F>
static void lp_rows(uint32_t rows, uint32_t threads, F f)
{
    const uint32_t most = kGridThreads / threads;
    for (uint32_t done = 0; done < rows; done += std::min(most, rows - done)) f(done, std::min(most, rows - done));
}

template <int DT>
static void lp_launch(LpParams p, uint32_t rows, bool one_wave, hipStream_t st)
{
    p.row0 = 0;
    if (p.S > 1) hipLaunchKernelGGL((logprobs_kernel<DT, kLpThreads, true>), dim3(rows * p.S), dim3(kLpThreads), 0, st, p);
    else lp_rows(rows, one_wave ? kWave : kLpThreads, [&](uint32_t first, uint32_t n) {
        p.row0 = first;
        if (one_wave) hipLaunchKernelGGL((logprobs_kernel<DT, kWave, false>), dim3(n), dim3(kWave), 0, st, p);
        else hipLaunchKernelGGL((logprobs_kernel<DT, kLpThreads, false>), dim3(n), dim3(kLpThreads), 0, st, p);
    });
}

// Many short rows: a wave each, without a barrier.  When this was chosen 262144 x 256 bfloat16 logits and 20 alternatives took 426 us
// in the place of 1098 by workgroups (now 383), 30000 x 8192 127 in the place of 190, 8192 x 16384 67 in the place of 75; but
// 8192 x 32768 131 in the place of 115, and 1024 x 8192 14.9 in the place of 13.8.  Up to 32 alternatives: the bound of as many as there
// are lanes is a low one (30000 x 8192 with 32 138 in the place of 196, with 48 226 in the place of 204, with 64 1147 in the place of
// 230).
static bool lp_one_wave(uint32_t rows, uint32_t windows, int32_t top) { return windows <= 2048u && rows >= 2048u && top <= 32; }

}  // namespace rs

using namespace rs;

extern "C" {

size_t rs_logprobs_workspace_bytes(void) { return (size_t)kLpSplitMost * (sizeof(LpSlice) + 16); }

int rs_token_logprobs(const void *logits, int32_t dtype, int64_t stride_b, int64_t stride_t,
                      const void *tokens, int32_t tokens_64, int64_t token_stride_b, int64_t token_stride_t,
                      int32_t B, int32_t T, int32_t V, double temperature, int32_t top,
                      float *logprobs, float *entropy, int32_t *rank, float *top_logprobs, int32_t *top_tokens,
                      float *stats, void *workspace, size_t workspace_bytes, void *stream)
{
    const int bad = lp_check(logits, dtype, tokens, tokens_64, B, T, V, temperature, top);
    if (bad != RS_OK) return bad;
    if (!workspace || (top && (!top_logprobs || !top_tokens))) return RS_ERR_NULL;
    if (workspace_bytes < rs_logprobs_workspace_bytes() || ((uintptr_t)workspace & 255)) return RS_ERR_WORKSPACE;
    if ((uintptr_t)stats & 15) return RS_ERR_ALIGN;
    const uint32_t rows = (uint32_t)B * (uint32_t)T;
    const uint32_t vec = dtype == RS_DTYPE_F32 ? 4 : 8, windows = (uint32_t)V / vec;
    LpParams p;
    p.logits = logits; p.stride_b = stride_b; p.stride_t = stride_t;
    p.tokens = tokens; p.tokens_64 = tokens_64; p.token_b = token_stride_b; p.token_t = token_stride_t;
    p.T = T; p.V = V; p.top = top;
    p.c = (float)(1.4426950408889634 / temperature); p.inv_t = (float)(1.0 / temperature);
    p.logprobs = logprobs; p.entropy = entropy; p.rank = rank; p.top_logprobs = top_logprobs; p.top_tokens = top_tokens;
    p.stats = (float4 *)stats;
    // (a thread's windows are worked on four at a time)
    const bool one_wave = lp_one_wave(rows, windows, top);
    const uint32_t threads = one_wave ? kWave : kLpThreads;
    const uint32_t per_row = (windows + threads - 1) / threads, split = one_wave ? 1 : lp_split(rows, windows);
    p.J = split > 1 ? ((per_row + split - 1) / split + 3) / 4 * 4 : per_row;
    p.S = split > 1 ? (per_row + p.J - 1) / p.J : 1;
    // stretches of four windows and more, at most kLpSegs of them in a slice and kLpStretches in a row
    const uint32_t most = p.S > 1 ? std::min((uint32_t)kLpSegs, (uint32_t)kLpStretches / p.S) : (uint32_t)kLpSegs;
    for (p.seg_log = 2; p.J > most << p.seg_log; ) ++p.seg_log;
    p.arrived = (uint32_t *)workspace;
    p.slices = (LpSlice *)((char *)workspace + 16 * (size_t)kLpSplitMost);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == RS_DTYPE_F32) lp_launch<RS_DTYPE_F32>(p, rows, one_wave, st);
    else if (dtype == RS_DTYPE_BF16) lp_launch<RS_DTYPE_BF16>(p, rows, one_wave, st);
    else lp_launch<RS_DTYPE_F16>(p, rows, one_wave, st);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

int rs_token_logprobs_backward(const void *logits, int32_t dtype, int64_t stride_b, int64_t stride_t,
                               const void *tokens, int32_t tokens_64, int64_t token_stride_b, int64_t token_stride_t,
                               int32_t B, int32_t T, int32_t V, double temperature, int32_t top,
                               const float *stats, const int32_t *top_tokens,
                               const float *grad_logprobs, int32_t grad_logprobs_stride,
                               const float *grad_entropy, int32_t grad_entropy_stride,
                               const float *grad_top, int32_t grad_top_stride,
                               void *grad_logits, void *stream)
{
    const int bad = lp_check(logits, dtype, tokens, tokens_64, B, T, V, temperature, top);
    if (bad != RS_OK) return bad;
    if (!stats || !grad_logits || (grad_top && top && !top_tokens)) return RS_ERR_NULL;
    if (((uintptr_t)stats & 15) || ((uintptr_t)grad_logits & (dtype == RS_DTYPE_F32 ? 3 : 1))) return RS_ERR_ALIGN;
    for (const int32_t s : {grad_logprobs_stride, grad_entropy_stride, grad_top_stride}) if (s != 0 && s != 1) return RS_ERR_ARG;
    const uint32_t rows = (uint32_t)B * (uint32_t)T;
    const uint32_t vec = dtype == RS_DTYPE_F32 ? 4 : 8, windows = (uint32_t)V / vec;
    LpGradParams p;
    p.logits = logits; p.stride_b = stride_b; p.stride_t = stride_t;
    p.tokens = tokens; p.tokens_64 = tokens_64; p.token_b = token_stride_b; p.token_t = token_stride_t;
    p.T = T; p.V = V; p.top = top;
    p.c = (float)(1.4426950408889634 / temperature); p.inv_t = (float)(1.0 / temperature);
    p.stats = (const float4 *)stats; p.top_tokens = top_tokens;
    p.g = grad_logprobs; p.h = grad_entropy; p.a = top ? grad_top : nullptr;
    p.g_stride = grad_logprobs_stride; p.h_stride = grad_entropy_stride; p.a_stride = grad_top_stride;
    p.grad = grad_logits;
    p.chunks = std::max(1u, (windows + kLpGradWindows - 1) / kLpGradWindows);
    const hipStream_t st = (hipStream_t)stream;
    lp_rows(rows, p.chunks * kWave, [&](uint32_t first, uint32_t n) {
        const dim3 grid(n * p.chunks), block(kWave);
        p.row0 = first;
        if (dtype == RS_DTYPE_F32) hipLaunchKernelGGL(logprobs_grad_kernel<RS_DTYPE_F32>, grid, block, 0, st, p);
        else if (dtype == RS_DTYPE_BF16) hipLaunchKernelGGL(logprobs_grad_kernel<RS_DTYPE_BF16>, grid, block, 0, st, p);
        else hipLaunchKernelGGL(logprobs_grad_kernel<RS_DTYPE_F16>, grid, block, 0, st, p);
    });
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

}  // extern "C"
