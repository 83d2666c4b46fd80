"""Where the tiles' loads go, walked on the CPU with the kernels' own arithmetic (csrc/rs_tile.h): for a row that is there, every byte that a
load of a whole block asks for is there too, whatever the hardware does with the scalar part of a buffer load's address; for one
that is not, the vector part lies behind the buffer by itself; and a last block that the row does not fill has no scalar part at all."""
import os
import re
import subprocess

from tests.conftest import ROOT

CSRC = os.path.join(ROOT, "rapid_sampling_amd", "csrc")

WALK = r"""
#include "rs_tile.h"
#include <cstdio>
#include <set>
using namespace rs;

static int fail(const char *what, uint32_t rows, uint32_t row, uint64_t stride, uint64_t K) {
    std::printf("%s: rows %u row %u stride %llu K %llu\n", what, rows, row, (unsigned long long)stride, (unsigned long long)K);
    return 1;
}

int main() {
    const uint64_t widths[][2] = {{1, 16}, {16, 16}, {100, 112}, {128, 128}, {130, 144}, {200, 208}, {384, 384}, {4096, 4096}, {4000, 8192},
                                  {(uint64_t)kTileStride, (uint64_t)kTileStride}, {1999, (uint64_t)kTileStride}};
    for (uint32_t waves : {4u, 8u})
        for (uint32_t high : {64u, 128u, 256u})
            for (uint32_t rows = 1; rows <= high; ++rows)
                for (auto &width : widths) {
                    const uint64_t K = width[0], stride = width[1], end = (rows - 1) * stride + K;
                    if (tile_bytes(rows, (uint32_t)stride, (uint32_t)K) != (rows - 1) * stride + (K + 3) / 4 * 4) return fail("size", rows, 0, stride, K);
                    std::set<uint32_t> seen;
                    for (uint32_t load = 0; load < high / (8 * waves); ++load)
                        for (uint32_t wave = 0; wave < waves; ++wave)
                            for (uint32_t lane = 0; lane < 64; lane += 8) {
                                const uint32_t row = tile_row(load, waves, wave, lane);
                                seen.insert(row);
                                if (row >= high || tile_row(load, waves, wave, lane + 7) != row) return fail("row", rows, row, stride, K);
                                for (uint32_t byte = 0; byte < 128; byte += 16) {
                                    const uint64_t at = tile_at(row, rows, (uint32_t)stride, byte);
                                    if (row >= rows) {      // behind the buffer, and no address that begins again at 0
                                        if (at < tile_bytes(rows, (uint32_t)stride, (uint32_t)K) || at + 16 > 0xFFFFFFFFull) return fail("none", rows, row, stride, K);
                                        continue;
                                    }
                                    if (at != row * stride + byte) return fail("place", rows, row, stride, K);
                                    if (K >= 128 && at + (K / 128 - 1) * 128 + 16 > end) return fail("past the end", rows, row, stride, K);
                                    if (K % 128 && tile_at(row, rows, (uint32_t)stride, byte + (uint32_t)K / 128 * 128) != at + K / 128 * 128) return fail("last block", rows, row, stride, K);
                                    if (K % 128 && at + K / 128 * 128 + 16 > 0xFFFFFFFFull) return fail("32 bits", rows, row, stride, K);
                                }
                            }
                    if (seen.size() != high) return fail("rows left out", rows, 0, stride, K);
                }
    // x's scales: rows of 4 bytes a block, no further than the last row's
    for (uint32_t rows = 1; rows <= 256; ++rows)
        for (uint64_t blocks : {1ull, 2ull, 33ull, 131072ull})
            for (uint32_t row = 0; row < 256; ++row)
                if (row < rows ? tile_at(row, rows, (uint32_t)blocks * 4, 0) + (blocks - 1) * 4 + 4 > rows * blocks * 4
                               : tile_at(row, rows, (uint32_t)blocks * 4, 0) < rows * blocks * 4) return fail("scale", rows, row, blocks, 0);
    return 0;
}
"""


def test_every_load_of_a_tile_lies_within_its_rows(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(WALK)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I" + CSRC, "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout


def test_scalar_parts_of_buffer_loads_are_columns():
    """The scalar argument of every buffer load of the product: the block's first column, or nothing."""
    text = open(os.path.join(CSRC, "rs_linear.h")).read()
    found = []
    for m in re.finditer(r"__builtin_amdgcn_raw(?:_ptr)?_buffer_load_(lds|b\d+)\(", text):
        depth, at, args, begin = 1, m.end(), [], m.end()
        while depth:
            c = text[at]
            depth += (c == "(") - (c == ")")
            if (c == "," and depth == 1) or not depth:
                args.append(text[begin:at].strip())
                begin = at + 1
            at += 1
        found.append(args[4] if m.group(1) == "lds" else args[2])
    assert found and set(found) <= {"k", "kb * 4u", "0"}, found
