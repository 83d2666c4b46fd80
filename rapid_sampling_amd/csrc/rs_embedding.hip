// Instantiations, launchers and C entry points of the embedding and its gradient.
#include "rs_embedding.h"

#include <algorithm>

namespace rs {

static uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// Threads of a row: one for each eight columns, in powers of two up to a workgroup.
static uint32_t row_width(uint32_t K)
{
    uint32_t w = 0;
    while (w < 8 && (8u << w) < K) ++w;
    return w;
}

template <int WT, int DT> static void launch_embedding(const EmbeddingParams &p, hipStream_t st)
{
    const uint32_t rows = 256u >> p.width;
    hipLaunchKernelGGL((embedding_kernel<WT, DT>), dim3((p.M + rows - 1) / rows), dim3(256), 0, st, p);
}
template <int WT> static void launch_embedding(const EmbeddingParams &p, int32_t dtype, hipStream_t st)
{
    if (dtype == RS_DTYPE_F32) launch_embedding<WT, RS_DTYPE_F32>(p, st);
    else if (dtype == RS_DTYPE_BF16) launch_embedding<WT, RS_DTYPE_BF16>(p, st);
    else launch_embedding<WT, RS_DTYPE_F16>(p, st);
}

// Who sorts: one workgroup, while others clear dw, or stretches of the list in three launches for a digit, behind the clearing.  (Gradient of a table of
// 131072 x 4096, 131072 x 8 and 2000 x 512 in bfloat16, us, one and stretches: 1024 tokens 205, 19, 20 and 227, 31, 27; 8192 230, 47, 35 and 267,
// 53, 40; 16384 270, 80, 55 and 305, 63, 46; 32768 445, 157, 104 and 361, 68, 54.)
static bool sorts_alone(uint32_t N, uint64_t clear) { return N <= kSortAlone / 2 || (N <= kSortAlone && clear >= 1ull << 28); }

static uint64_t take(uint64_t &bytes, uint64_t n)
{
    const uint64_t at = bytes;
    bytes += up(n, 256);
    return at;
}
SortSpace sort_space(uint32_t N, uint32_t V, uint64_t &bytes)
{
    SortSpace s;
    uint32_t bits = 1;
    while (bits < 32 && (V >> bits)) ++bits;             // of a token, or of V itself
    s.digits = (bits + kSortBits - 1) / kSortBits;
    s.bits = (bits + s.digits - 1) / s.digits;
    s.groups = (N + kSortTile - 1) / kSortTile;
    for (int i = 0; i < 2; ++i) s.pairs[i] = take(bytes, 8ull * N);
    s.counts = take(bytes, N <= kSortAlone / 2 ? 0 : 4ull * s.groups << s.bits);
    return s;
}

const uint2 *launch_sort(const TokenList &tokens, uint32_t N, uint32_t V, const SortSpace &s, char *ws, void *clear_at, uint64_t clear_bytes, hipStream_t st)
{
    auto pairs = [&](uint32_t i) { return (uint2 *)(ws + s.pairs[i]); };
    SortParams p = {};
    p.tokens = tokens;
    p.N = N; p.V = V; p.bits = s.bits; p.first = 1; p.digits = s.digits;
    p.counts = (uint32_t *)(ws + s.counts);
    const uint32_t lds = (kSortWaves << s.bits) * 4;
    const ClearParams clear{(char *)clear_at, clear_bytes};
    // (64 KB to a workgroup, one behind the other: 1 GiB in 168 us; in 1023 workgroups 189)
    const uint32_t clears = clear.bytes ? (uint32_t)std::min<uint64_t>(32767, clear.bytes / 65536 + 1) : 0;
    if (sorts_alone(N, clear.bytes)) {
        p.out = pairs(0); p.out_b = pairs(1);
        hipLaunchKernelGGL(sort_alone_kernel, dim3(1 + clears), dim3(kSortThreads), lds, st, p, clear);
    } else {
        if (clears) hipLaunchKernelGGL(clear_kernel, dim3(clears), dim3(kSortThreads), 0, st, clear);
        for (uint32_t d = 0; d < s.digits; ++d) {
            p.out = pairs(d & 1);
            hipLaunchKernelGGL(sort_count_kernel, dim3(s.groups), dim3(kSortThreads), lds, st, p);
            hipLaunchKernelGGL(sort_scan_kernel, dim3(1), dim3(kSortThreads), 0, st, p.counts, s.groups << s.bits);
            hipLaunchKernelGGL(sort_place_kernel, dim3(s.groups), dim3(kSortThreads), lds, st, p);
            p.first = 0; p.shift += s.bits; p.in = p.out;
        }
    }
    return pairs((s.digits - 1) & 1);
}

// Where a gradient's scratch lies.
struct TableSpace {
    SortSpace sort;
    uint64_t parts, bytes = 0;
    uint32_t chunk, chunks;
};
static TableSpace table_space(uint32_t N, uint32_t V, uint32_t K)
{
    TableSpace s;
    s.sort = sort_space(N, V, s.bytes);
    // Chunks of a quarter to half of the tokens' square root, 16 places at least: enough of them for the chip, and 4 to 16 times as many as each has places to
    // join, eight at a time by one workgroup for 2048 columns, for a token that makes up all.  (8192 tokens over 131072 x 4096 in bfloat16 229 us, 264 with
    // one token in half of the places, 301 in all; over 2000 x 4096 49, 94 and 140; 32768 over 2000 x 4096 98, 189 and 279.)
    s.chunk = 4;
    while (s.chunk < 12 && (1ull << (2 * s.chunk + 4)) <= N) ++s.chunk;
    s.chunks = (N + (1u << s.chunk) - 1) >> s.chunk;
    s.parts = take(s.bytes, (uint64_t)s.chunks * 2 * K * 4);
    return s;
}

template <int GT, int DT> static void launch_sums(const TableGradParams &p, uint32_t chunks, hipStream_t st)
{
    const dim3 groups(chunks, (p.K + 2047) / 2048);
    hipLaunchKernelGGL((table_chunk_kernel<GT, DT>), groups, dim3(256), 0, st, p);
    if (chunks > 1) hipLaunchKernelGGL(table_join_kernel<DT>, groups, dim3(256), 0, st, p);
}
template <int GT> static void launch_sums(const TableGradParams &p, uint32_t chunks, int32_t dtype, hipStream_t st)
{
    if (dtype == RS_DTYPE_F32) launch_sums<GT, RS_DTYPE_F32>(p, chunks, st);
    else if (dtype == RS_DTYPE_BF16) launch_sums<GT, RS_DTYPE_BF16>(p, chunks, st);
    else launch_sums<GT, RS_DTYPE_F16>(p, chunks, st);
}

static bool known(int32_t dtype) { return dtype == RS_DTYPE_F32 || dtype == RS_DTYPE_BF16 || dtype == RS_DTYPE_F16; }
static uint32_t size_of(int32_t dtype) { return dtype == RS_DTYPE_F32 ? 4 : 2; }

}  // namespace rs

using namespace rs;

extern "C" {

int rs_embedding(const void *tokens, int32_t tokens_64, int64_t token_stride, const void *w, int32_t w_dtype, int64_t w_stride, const float *w_scale,
                 double scale, int32_t M, int32_t V, int32_t K, void *y, int32_t y_dtype, void *stream)
{
    const bool eight = w_dtype == RS_TABLE_INT8 || w_dtype == RS_TABLE_FP8;
    if (!tokens || !w || !y || (eight && !w_scale)) return RS_ERR_NULL;
    if ((!known(w_dtype) && !eight) || !known(y_dtype) || (tokens_64 != 0 && tokens_64 != 1)) return RS_ERR_ARG;
    if (M <= 0 || V <= 0 || K <= 0 || M >= RS_LINEAR_MAX || V > RS_LINEAR_MAX || K > RS_LINEAR_MAX || (V > 1 && w_stride < (eight ? K : 0))) return RS_ERR_SHAPE;
    if (((uintptr_t)tokens & (tokens_64 ? 7 : 3)) || ((uintptr_t)y & (size_of(y_dtype) - 1))) return RS_ERR_ALIGN;
    if (eight ? ((uintptr_t)w & 15) || (V > 1 && (w_stride & 15)) || ((uintptr_t)w_scale & 3) : ((uintptr_t)w & (size_of(w_dtype) - 1)) != 0) return RS_ERR_ALIGN;
    EmbeddingParams p;
    p.tokens = TokenList{tokens, token_stride, tokens_64};
    p.w = w; p.w_stride = w_stride; p.w_scale = w_scale; p.y = y; p.scale = (float)scale;
    p.M = (uint32_t)M; p.V = (uint32_t)V; p.K = (uint32_t)K; p.width = row_width(p.K);
    const hipStream_t st = (hipStream_t)stream;
    if (w_dtype == RS_DTYPE_F32) launch_embedding<RS_DTYPE_F32>(p, y_dtype, st);
    else if (w_dtype == RS_DTYPE_BF16) launch_embedding<RS_DTYPE_BF16>(p, y_dtype, st);
    else if (w_dtype == RS_DTYPE_F16) launch_embedding<RS_DTYPE_F16>(p, y_dtype, st);
    else if (w_dtype == RS_TABLE_INT8) launch_embedding<kTableInt8>(p, y_dtype, st);
    else launch_embedding<kTableFp8>(p, y_dtype, st);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

size_t rs_embedding_workspace_bytes(int32_t M, int32_t V, int32_t K)
{
    return M > 0 && V > 0 && K > 0 ? table_space((uint32_t)M, (uint32_t)V, (uint32_t)K).bytes : 0;
}

int rs_embedding_backward(const void *tokens, int32_t tokens_64, int64_t token_stride, const void *g, int32_t g_dtype, int64_t g_stride, double scale,
                          int32_t M, int32_t V, int32_t K, void *dw, int32_t dw_dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!tokens || !g || !dw || !workspace) return RS_ERR_NULL;
    if (!known(g_dtype) || !known(dw_dtype) || (tokens_64 != 0 && tokens_64 != 1)) return RS_ERR_ARG;
    if (M <= 0 || V <= 0 || K <= 0 || M >= RS_LINEAR_MAX || V > RS_LINEAR_MAX || K > RS_LINEAR_MAX || (M > 1 && g_stride < 0)) return RS_ERR_SHAPE;
    if (((uintptr_t)tokens & (tokens_64 ? 7 : 3)) || ((uintptr_t)g & (size_of(g_dtype) - 1)) || ((uintptr_t)dw & (size_of(dw_dtype) - 1))) return RS_ERR_ALIGN;
    const TableSpace s = table_space((uint32_t)M, (uint32_t)V, (uint32_t)K);
    if (workspace_bytes < s.bytes || ((uintptr_t)workspace & 255)) return RS_ERR_WORKSPACE;
    char *ws = (char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    TableGradParams t;
    t.pairs = launch_sort(TokenList{tokens, token_stride, tokens_64}, (uint32_t)M, (uint32_t)V, s.sort, ws, dw, (uint64_t)V * K * size_of(dw_dtype), st);
    t.g = g; t.g_stride = M > 1 ? g_stride : 0; t.parts = (float *)(ws + s.parts); t.dw = dw; t.scale = (float)scale;
    t.N = (uint32_t)M; t.V = (uint32_t)V; t.K = (uint32_t)K; t.chunk = s.chunk;
    if (g_dtype == RS_DTYPE_F32) launch_sums<RS_DTYPE_F32>(t, s.chunks, dw_dtype, st);
    else if (g_dtype == RS_DTYPE_BF16) launch_sums<RS_DTYPE_BF16>(t, s.chunks, dw_dtype, st);
    else launch_sums<RS_DTYPE_F16>(t, s.chunks, dw_dtype, st);
    return hipGetLastError() == hipSuccess ? RS_OK : RS_ERR_LAUNCH;
}

}  // extern "C"
