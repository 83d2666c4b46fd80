// Where the loads of a tile's rows go, as plain arithmetic: the kernels use it, and a program without a GPU can walk it.
//
// A buffer load's address has a vector and a scalar part.  The vector part is held against the buffer's size (what lies behind it reads
// as 0); whether the scalar part is added first, taken off the size or left out of the comparison is nothing to build on.  So the row is in
// the vector part, which for rows behind the tile's last lies behind every buffer by itself, and the scalar part is the first column of a
// block that lies within the row: with a row that is there, every byte asked for is there too.  A last block that the row
// does not fill has its column in the vector part as well.  (The last row read once more in the place of those behind it: 32 x 131072
// x 4096 113 us in the place of 105.)
#pragma once

#include <stdint.h>

namespace rs {

constexpr int     kFpBlock    = 128;
constexpr int64_t kTileStride = (1ll << 32) / 256 - kFpBlock;   // a tile's rows, 256 at most, are reached with 32 bits

// Row of the tile that a thread's load fills: eight rows a wave and load, eight threads a row.
constexpr uint32_t tile_row(uint32_t load, uint32_t waves, uint32_t wave, uint32_t lane) { return (load * waves + wave) * 8u + lane / 8u; }

// Byte of `row` (at most 255) at which it is read, for rows `stride` bytes apart, of which there are `rows`; behind every tile's
// bytes where it is not there.  Both factors fit 24 bits.
constexpr uint32_t kTileNone = 0xFFFF9000u;
constexpr uint32_t tile_at(uint32_t row, uint32_t rows, uint32_t stride, uint32_t byte)
{
    return row < rows ? (row & 0xFFu) * (stride & 0xFFFFFFu) + byte : kTileNone;
}

// Bytes from a tile's first row to the last that is looked at, in whole words: a word is read or it is not.  At most 2^32 - 2^15.
constexpr uint32_t tile_bytes(uint32_t rows, uint32_t stride, uint32_t K) { return (rows - 1u) * stride + ((K + 3u) & ~3u); }

}  // namespace rs
