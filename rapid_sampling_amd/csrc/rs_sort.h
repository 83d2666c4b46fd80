// Tokens put in order with their places, for what works by token: rs_embedding.hip has the kernels.
#pragma once

#include "rs_common.h"

namespace rs {

struct TokenList {
    const void *at;
    int64_t     stride;
    int32_t     is_64;
    __device__ __forceinline__ int64_t operator[](int64_t i) const
    {
        return is_64 ? ((const int64_t *)at)[i * stride] : (int64_t)((const int32_t *)at)[i * stride];
    }
};

// Where a sort's scratch lies, from `bytes` on, which moves behind it.
struct SortSpace {
    uint64_t pairs[2], counts;
    uint32_t digits, bits, groups;
};
SortSpace sort_space(uint32_t N, uint32_t V, uint64_t &bytes);

// (token, place) by token and place; a token that is none, or outside the vocabulary, counts as V.  `clear_bytes` from `clear` on are set to 0 meanwhile.
const uint2 *launch_sort(const TokenList &tokens, uint32_t N, uint32_t V, const SortSpace &s, char *workspace, void *clear, uint64_t clear_bytes, hipStream_t st);

}  // namespace rs
