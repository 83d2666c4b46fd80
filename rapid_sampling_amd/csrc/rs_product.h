// Tiles of a matrix product on the matrix cores, for the operators that make one and do something with its sums:
//
//   sum[m, n] = sum over r of P[n, r] Q[m, r]
//
// of bfloat16, float16 or float32 values with float32 sums, or of 8-bit integers with whole sums.  Either operand lies in memory with
// the values of one row n (or m) side by side, as activations and weights do in y = x w^T, or (transposed) with those of one r
// side by side, as both do in the products that make gradients.
#pragma once

#include "rs_linear.h"

#include <algorithm>

namespace rs {

typedef short v4s __attribute__((ext_vector_type(4)));

constexpr int kInt8 = 100;                       // next to RS_DTYPE_*
constexpr uint32_t kRowBytes = 128;              // of the reduction that a stage holds
template <int DT> constexpr uint32_t kSize = DT == kInt8 ? 1 : DT == RS_DTYPE_F32 ? 4 : 2;
template <int DT> struct SumOf { typedef v4f type; };
template <> struct SumOf<kInt8> { typedef v4i type; };
template <int DT> using Sum = typename SumOf<DT>::type;


// 16 x 16 sums of 64 bytes of each row.  Lane l gives 16 bytes of row l % 16 of either side, the same part of the reduction on both, and has
// the sums of the first side's rows 4 (l / 16) + 0..3 with the second side's row l % 16.  (float32: of what is left of its values in bfloat16)
template <int DT> __device__ __forceinline__ Sum<DT> multiply(v4i p, v4i q, Sum<DT> s)
{
    if constexpr (DT == kInt8) return __builtin_amdgcn_mfma_i32_16x16x64_i8(p, q, s, 0, 0, 0);
    else if constexpr (DT == RS_DTYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, p), __builtin_bit_cast(v8h, q), s, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, p), __builtin_bit_cast(v8bf, q), s, 0, 0, 0);
}
// The products of all fragments of one half of a stage.
template <int DT, int NU, int MT> __device__ __forceinline__ void multiply_all(const v4i (&p)[NU], const v4i (&q)[MT], Sum<DT> (&acc)[NU][MT])
{
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[u][t] = multiply<DT>(p[u], q[t], acc[u][t]);
}

// Eight float32 values as three times eight of bfloat16, x = x0 + x1 + x2 exactly: eight bits of the significand each, cut off, not rounded, so that they have x's
// sign, and products that overflow the same infinity.  Of the nine products of two such sums the five with a first part are made, and of (x1 + x2)(y1 + y2) one, of
// both rounded to bfloat16 (the fourth of a value's parts).  That is off by at most 2^-22 of x y, by 2^-26 on average and in either direction: half of what
// the product's own rounding is.  (x1 y1 in its place, one of nine, is too small by up to 2^-21 and by 0.67 2^-24 on average; x0 and x1 rounded are off by 2^-24 at
// most, but have parts of both signs, whose overflows make NaN.  Products that are left out as well, eight in all, take 19 % longer where M is large.)  Six
// matrix instructions of 16 cycles in the place of eight of 32.
struct Thirds { v4i x[4]; };
__device__ __forceinline__ Thirds thirds(v4i lo, v4i hi)
{
    Thirds r;
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = (uint32_t)lo[j]; v[j + 4] = (uint32_t)hi[j]; }
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            r.x[i][j / 2] = (int)__builtin_amdgcn_perm(v[j + 1], v[j], 0x07060302u);          // the upper halves of both
            if (i == 1) {                                             // v: x1 + x2
                const v2bf two = {(__bf16)__uint_as_float(v[j]), (__bf16)__uint_as_float(v[j + 1])};
                r.x[3][j / 2] = __builtin_bit_cast(int, two);
            }
            if (i < 2)
#pragma unroll
                for (int h = 0; h < 2; ++h) v[j + h] = __float_as_uint(__uint_as_float(v[j + h]) - __uint_as_float(v[j + h] & 0xFFFF0000u));
        }
    return r;
}

// One operand of a product: `rows` rows (n or m) of `red` values, `stride` bytes from a row (transposed: from one r) to the next.  16-byte
// aligned, as is the stride; at most kTileStride.
struct Operand {
    const char *at;
    uint32_t    stride, rows;
};

struct Product {
    Operand  p, q;
    uint32_t red;                    // values of the reduction
    uint32_t split;                  // workgroups that share a tile's reduction
};

// COUNT rows of one operand in LDS, STAGE after stage of the reduction, and how they get there.
//
// Rows from memory go to LDS without passing through registers.  As they are: a stage is 128 bytes of every row, its eight 16-byte
// pieces in an order that depends on the row (place = piece ^ turn), so that the eight rows read at once lie in different banks.
// Transposed: a stage is 128 / size values of r, the COUNT values of each side by side; those of 16 bits are turned by the reads from
// LDS (ds_read_b64_tr_b16: four r of a row to a lane), whose 32-byte pieces are stored in such an order too; those of 32 bits, 64-byte
// pieces in an order of their own, are read one by one.
//
// PAIRS (untransposed): the rows are dealt to the matrix instructions so that a lane's sums of two fragments (of 16 rows; F to a wave) belong
// to eight consecutive rows: 16 bytes of a result in 16 bits.
template <int DT, bool TR, bool PAIRS, int COUNT, int F, int WAVES>
struct Side {
    static constexpr uint32_t kBytes = COUNT * kRowBytes, kLoads = kBytes / (1024 * WAVES), kRed = kRowBytes / kSize<DT>;
    static constexpr uint32_t kWide = COUNT * kSize<DT>;                     // bytes of one r, transposed
    static_assert(kBytes % (1024 * WAVES) == 0, "whole loads");
    static_assert(!TR || (kWide <= 1024 && 1024 % kWide == 0 && DT != kInt8), "a wave's load is whole values of r");
    static constexpr int kBufferFlags = 0x00027000;                          // untyped, offsets in bytes

    const char *base;
    uint32_t    stride, rows, bytes;       // transposed: bytes of one r from the tile's first row on
    uint32_t    byte;                      // as they are: of the row, of the thread's pieces, the same for all its loads
    uint32_t    off[kLoads];
    static_assert(TR || WAVES % 2 == 0, "a thread's loads have one turn");

    // the order of pieces: depends on the row and is the same for all the fragments of a lane
    static __device__ __forceinline__ uint32_t turn(uint32_t row)
    {
        if (!TR) return PAIRS ? (row & 3u) | ((row >> 1) & 4u) : row & 7u;
        return kWide == 128 ? ((row >> 1) & 1u) | ((row >> 2) & 2u) : (row & 3u) | ((row >> 1) & 4u);
    }
    // byte of the source's row (or r) that a byte of the stage holds
    static __device__ __forceinline__ void source_of(uint32_t at, uint32_t &row, uint32_t &byte)
    {
        if (!TR) { row = at / kRowBytes; byte = ((at / 16u % 8u) ^ turn(row)) * 16u; return; }
        row = at / kWide;
        byte = at % kWide;
        if (kSize<DT> == 2) byte = ((byte / 32u) ^ turn(row)) * 32u + byte % 32u;
        else byte ^= (row / 8u & 3u) * 64u;
    }
    // and where a byte of an r is held, of a transposed stage of 16 bits
    static __device__ __forceinline__ uint32_t place_of(uint32_t row, uint32_t byte) { return row * kWide + ((byte / 32u) ^ turn(row)) * 32u + byte % 32u; }
    static __device__ __forceinline__ uint32_t place(uint32_t i) { return (i * WAVES + wave_id()) * 1024u + threadIdx.x % 64u * 16u; }

    __device__ __forceinline__ Side(const Operand &o, uint32_t first)
    {
        stride = o.stride;
        rows = min(o.rows - first, (uint32_t)COUNT);
        base = o.at + (TR ? (int64_t)first * kSize<DT> : (int64_t)first * o.stride);
        bytes = (o.rows - first) * kSize<DT>;
        byte = 0;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            uint32_t row;
            source_of(place(i), row, byte);
            off[i] = TR ? row * stride + byte : tile_at(row, rows, stride, byte);
            asm volatile("" : "+v"(off[i]));               // once, and not for every stage
        }
    }
    // Asks for the stage that begins at r.  What lies behind the reduction's end reads as 0: as they are, pieces from there on by an address
    // behind every buffer, and the bytes of the one that it cuts by clear(); transposed, by the buffer's size.  (What a transposed
    // load reads behind a row's end belongs to sums that nobody asks for.)
    __device__ __forceinline__ void fill(uint32_t r, uint32_t red, char *lds) const
    {
        const uint32_t left = red - r;
        const uint32_t size = TR ? (min(left, kRed) - 1u) * stride + ((bytes + 3u) & ~3u) : tile_bytes(rows, stride, left * kSize<DT>);
        const int64_t at = TR ? (int64_t)r * stride : (int64_t)r * kSize<DT>;
        const __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc((void *)(base + at), 0, (int)size, kBufferFlags);
        const bool there = TR || byte < left * kSize<DT>;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (LdsPtr)(lds + (i * WAVES + wave_id()) * 1024u), 16, there ? off[i] : kTileNone, 0, 0, 0);
    }
    // The bytes behind the reduction's end of the piece that it cuts, of the stage that begins `left` values before it.
    static __device__ __forceinline__ void clear(uint32_t left, char *lds)
    {
        for (uint32_t row = threadIdx.x; !TR && row < (uint32_t)COUNT; row += 64u * WAVES) {
            const uint32_t end = left * kSize<DT>;
            v4i *piece = (v4i *)(lds + row * kRowBytes + ((end / 16u) ^ turn(row)) * 16u);
            v4i v = *piece;
            const int32_t keep = (int32_t)(end % 16u);
#pragma unroll
            for (int d = 0; d < 4; ++d) v[d] &= keep >= 4 * d + 4 ? -1 : keep <= 4 * d ? 0 : (1 << 8 * (keep - 4 * d)) - 1;
            *piece = v;
        }
    }

    // The lane's 16 bytes of fragment f (16 rows from `first` + 16 f on; dealt, if they are) of half `sub` of the stage: its quarter of 64
    // bytes of the row, or (float32) of 128 bytes the half `sub` of its quarter.
    struct Reader {
        static constexpr int kReads = !TR ? 1 : kSize<DT> == 2 ? 2 : 4;
        uint32_t at[TR ? F : 1];
        __device__ __forceinline__ explicit Reader(uint32_t first)
        {
            const uint32_t lane = threadIdx.x % 64u, i = lane % 16u, part = lane / 16u;
            if constexpr (!TR) {
                const uint32_t row = first + (PAIRS ? i / 4u * 8u + i % 4u : i);
                at[0] = row * kRowBytes + ((kSize<DT> == 4 ? 2u * part : part) ^ turn(row)) * 16u;
            } else if constexpr (kSize<DT> == 2) {
                const uint32_t row = 8u * part + i / 4u;
#pragma unroll
                for (int f = 0; f < F; ++f) at[f] = row * kWide + ((first / 16u + f) ^ turn(row)) * 32u + i % 4u * 8u;
            } else
#pragma unroll
                for (int f = 0; f < F; ++f) at[f] = 8u * part * kWide + ((first / 16u + f) ^ part) * 64u + i * 4u;
        }
        __device__ __forceinline__ v4i operator()(const char *lds, int f, int sub) const
        {
            if constexpr (!TR) return *(const v4i *)(lds + (at[0] ^ (sub ? (kSize<DT> == 4 ? 16u : 64u) : 0u)) + (PAIRS ? f / 2 * 32 + f % 2 * 4 : f * 16) * kRowBytes);
            else if constexpr (kSize<DT> == 2) {
                typedef __attribute__((address_space(3))) v4s *P;
                const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(lds + at[f] + sub * 32 * kWide));
                const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(lds + at[f] + (sub * 32 + 4) * kWide));
                return __builtin_bit_cast(v4i, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
            } else {
                v4i v;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = *(const int *)(lds + at[f] + (sub * 4 + j) * kWide);
                return v;
            }
        }
    };
};

// Which tiles (columns x rows): 256 x 256, 128 x 128 or 128 x 64, by how many rounds of them the chip makes.  Of the large ones a compute
// unit makes one at a time, of the others two, and those take 0.6 and 0.45 of the time, not half and a quarter: they read more for a
// product.  (Forward pass over 50257 x 2048 in bfloat16, large and middle: 300 rows 109 and 90 us, 385 rows 108 and 120, 256 rows 63 and
// 67, 1024 rows 217 and 215, with gradients 944 and 998.  int8, middle and small: 77 x 50257 x 2000 24.1 and 31.1 us, 128 x 32768 x 4096
// 29.7 and 25.3.)
enum TileSize { kSmall, kMiddle, kLarge };
inline uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }
inline uint64_t tiles_of(uint64_t rows, uint64_t columns, uint64_t high, uint64_t wide) { return up(rows, high) / high * (up(columns, wide) / wide); }
inline TileSize tile_size(uint64_t rows, uint64_t columns)
{
    const uint64_t large = 20 * (up(tiles_of(rows, columns, 256, 256), 256) / 256), middle = 12 * (up(tiles_of(rows, columns, 128, 128), 512) / 512),
                   small = 9 * (up(tiles_of(rows, columns, 64, 128), 512) / 512);
    return large <= std::min(middle, small) ? kLarge : middle <= small ? kMiddle : kSmall;
}

// A workgroup of WN x WM waves makes 16 NU WN rows of P x 16 MT WM rows of Q, a wave 16 NU x 16 MT of it.
template <int DT_, bool TP_, bool TQ_, bool PAIRS_, int WN_, int WM_, int NU_, int MT_, int STAGES_>
struct Tile {
    static constexpr int DT = DT_, WN = WN_, WM = WM_, NU = NU_, MT = MT_, STAGES = STAGES_;
    static constexpr bool TP = TP_, TQ = TQ_, PAIRS = PAIRS_;
    static constexpr uint32_t kWaves = WN * WM, kThreads = 64 * kWaves, kTileN = 16 * NU * WN, kTileM = 16 * MT * WM;
    typedef Side<DT, TP, PAIRS, kTileN, NU, kWaves> P;
    typedef Side<DT, TQ, false, kTileM, MT, kWaves> Q;
    static constexpr uint32_t kStage = P::kBytes + Q::kBytes, kLds = STAGES * kStage, kLoads = P::kLoads + Q::kLoads, kRed = P::kRed;
    typedef Sum<DT> Acc[NU][MT];

    // Sums of the lane: row m of Q and, for fragment u, the rows n(u) + 0..3 of P.
    uint32_t n0, m0;
    __device__ __forceinline__ uint32_t n(int u) const
    {
        const uint32_t part = threadIdx.x % 64u / 16u;
        return n0 + wave_id() % WN * (16u * NU) + (PAIRS ? u / 2 * 32u + part * 8u + u % 2 * 4u : u * 16u + part * 4u);
    }
    __device__ __forceinline__ uint32_t m(int t) const { return m0 + wave_id() / WN * (16u * MT) + t * 16u + threadIdx.x % 16u; }

    // Which tile.  Groups of 32 columns of tiles one after the other: their rows of P (64 MB of 8192 x 4096 in 16 bits) stay in the last cache for
    // all rows of tiles.  Of a group each XCD (workgroup b runs on XCD b % 8) takes a stretch, in panels of eight rows of tiles, so that
    // the 32 tiles it works on at a time share their rows in its L2.  (A single row of tiles is one group: eight stretches far apart are read faster than
    // one, 32 x 131072 x 4096 in int8 117 us and 100.)
    __device__ __forceinline__ uint32_t choose(const Product &a, uint32_t id)
    {
        const uint32_t tm = (a.q.rows + kTileM - 1u) / kTileM, tn = (a.p.rows + kTileN - 1u) / kTileN, tiles = tm * tn;
        uint32_t part = 0;
        if (a.split > 1u) { part = id / tiles; id -= part * tiles; }
        const uint32_t most = tm == 1u ? tn : 32u, group = id / (tm * most), wide = min(most, tn - group * most);
        id -= group * (tm * most);
        const uint32_t each = tm * wide / 8u, rest = tm * wide % 8u, xcd = id % 8u;
        id = xcd * each + min(xcd, rest) + id / 8u;
        const uint32_t panel = id / (8u * wide), high = min(8u, tm - panel * 8u), in = id - panel * 8u * wide;
        n0 = (group * most + in / high) * kTileN;
        m0 = (panel * 8u + in % high) * kTileM;
        return part;
    }

    __device__ __forceinline__ void make(const Product &a, uint32_t part, char *lds, Acc &acc) const
    {
        const P p(a.p, n0);
        const Q q(a.q, m0);
        const typename P::Reader rp(wave_id() % WN * (16u * NU));
        const typename Q::Reader rq(wave_id() / WN * (16u * MT));
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[u][t] = Sum<DT>{0, 0, 0, 0};
        const uint32_t stages = (a.red + kRed - 1u) / kRed;
        const uint32_t s0 = (uint32_t)((uint64_t)stages * part / a.split), count = (uint32_t)((uint64_t)stages * (part + 1u) / a.split) - s0;
        // Where P is read once, by one row of tiles, every workgroup begins at another stage: rows are usually a power of two of bytes
        // apart, and workgroups in step would ask the same memory channels at a time.
        const uint32_t first = !TP && a.q.rows <= kTileM && count ? s0 + n0 / kTileN % count : s0;
        uint32_t to_fill = first;
        auto fill = [&](char *to) {
            p.fill(to_fill * kRed, a.red, to);
            q.fill(to_fill * kRed, a.red, to + P::kBytes);
            to_fill = to_fill + 1u == s0 + count ? s0 : to_fill + 1u;
        };
#pragma unroll
        for (int b = 0; b < STAGES - 1; ++b)
            if (b < (int)count) fill(lds + b * kStage);
        uint32_t now = 0, next = (STAGES - 1) * kStage, at = first, j = 0;
        // The next stage is there, and the one after the last that is under way is asked for.
        auto arrive = [&]() {
            // (towards the end there are no newer stages to leave under way)
            if (STAGES == 2 || j + STAGES - 1 > count) stage_barrier<0>();
            else stage_barrier<(STAGES - 2) * kLoads>();
            if (a.red - at * kRed < kRed && (a.red * kSize<DT>) % 16u) {
                P::clear(a.red - at * kRed, lds + now);
                Q::clear(a.red - at * kRed, lds + now + P::kBytes);
                stage_barrier<0>();
            }
            at = at + 1u == s0 + count ? s0 : at + 1u;
            if (j + STAGES - 1u < count) fill(lds + next);
        };
        auto advance = [&]() {
            ++j;
            now = now == (STAGES - 1) * kStage ? 0u : now + kStage;
            next = next == (STAGES - 1) * kStage ? 0u : next + kStage;
        };
        if constexpr (kAhead) {
            Raw even, odd;
            auto step = [&](Raw &fresh, const Raw &held) {
                arrive();
                read(lds + now, rp, rq, fresh);
                multiply_raw(held, acc);
                advance();
            };
            if (count) {
                arrive();
                read(lds + now, rp, rq, even);
                advance();
            }
            while (j < count) {
                step(odd, even);
                if (j == count) {
                    multiply_raw(odd, acc);
                    return;
                }
                step(even, odd);
            }
            if (count) multiply_raw(even, acc);
        } else if constexpr (DT == RS_DTYPE_F32) {
            while (j < count) {
                arrive();
                whole(lds + now, rp, rq, acc);
                advance();
            }
        } else {
            // Both halves of a stage in registers: while one is multiplied the other is read, and the second half of a stage is multiplied behind
            // the barrier that the next stage is waited for at (8192 x 8192 x 4096 in bfloat16 476 us without, 413 with).
            v4i p0[NU], q0[MT], p1[NU], q1[MT];
#pragma unroll
            for (int u = 0; u < NU; ++u) p1[u] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < MT; ++t) q1[t] = v4i{0, 0, 0, 0};
            while (j < count) {
                arrive();
                half(lds + now, rp, rq, 0, p0, q0, p1, q1, acc);
                half(lds + now, rp, rq, 1, p1, q1, p0, q0, acc);
                advance();
            }
            multiply_all<DT>(p1, q1, acc);
        }
    }

    // float32: a stage at a time, the first operand's fragments one by one.  Of the smallest tiles, which few waves share a compute unit
    // with, a stage is read while the one before is multiplied.
    static constexpr bool kAhead = DT == RS_DTYPE_F32 && NU * MT <= 8;
    struct Raw { v4i p[NU][2], q[MT][2]; };
    static __device__ __forceinline__ void read(const char *lds, const typename P::Reader &rp, const typename Q::Reader &rq, Raw &r)
    {
#pragma unroll
        for (int t = 0; t < MT; ++t) { r.q[t][0] = rq(lds + P::kBytes, t, 0); r.q[t][1] = rq(lds + P::kBytes, t, 1); }
#pragma unroll
        for (int u = 0; u < NU; ++u) { r.p[u][0] = rp(lds, u, 0); r.p[u][1] = rp(lds, u, 1); }
    }
    static __device__ __forceinline__ void products(const Thirds &p, const Thirds (&q)[MT], Sum<DT> (&acc)[MT])
    {
        constexpr int kFirst[6] = {0, 3, 2, 0, 1, 0}, kSecond[6] = {2, 3, 0, 1, 0, 0};           // the smallest first; 3: see thirds
#pragma unroll
        for (int i = 0; i < 6; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = multiply<DT>(p.x[kFirst[i]], q[t].x[kSecond[i]], acc[t]);
    }
    static __device__ __forceinline__ void multiply_raw(const Raw &r, Acc &acc)
    {
        Thirds q[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) q[t] = thirds(r.q[t][0], r.q[t][1]);
#pragma unroll
        for (int u = 0; u < NU; ++u) products(thirds(r.p[u][0], r.p[u][1]), q, acc[u]);
    }
    static __device__ __forceinline__ void whole(const char *lds, const typename P::Reader &rp, const typename Q::Reader &rq, Acc &acc)
    {
        Thirds q[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) q[t] = thirds(rq(lds + P::kBytes, t, 0), rq(lds + P::kBytes, t, 1));
#pragma unroll
        for (int u = 0; u < NU; ++u) products(thirds(rp(lds, u, 0), rp(lds, u, 1)), q, acc[u]);
    }

    // Reads half `sub` of a stage into p and q and multiplies what was read before, one behind the other.
    static __device__ __forceinline__ void half(const char *lds, const typename P::Reader &rp, const typename Q::Reader &rq, int sub, v4i (&p)[NU], v4i (&q)[MT],
                                                const v4i (&before_p)[NU], const v4i (&before_q)[MT], Acc &acc)
    {
#pragma unroll
        for (int t = 0; t < MT; ++t) q[t] = rq(lds + P::kBytes, t, sub);
#pragma unroll
        for (int u = 0; u < NU; ++u) p[u] = rp(lds, u, sub);
        multiply_all<DT>(before_p, before_q, acc);
        constexpr int kReads = NU * P::Reader::kReads + MT * Q::Reader::kReads, kProducts = NU * MT;
        constexpr int kGroups = NU + MT;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            __builtin_amdgcn_sched_group_barrier(0x100, kReads / kGroups, 0);           // reads of LDS
            __builtin_amdgcn_sched_group_barrier(0x008, kProducts / kGroups, 0);        // products
        }
    }
};

// The columns n + 0..3 of a row that begins at element `at`, as far as there are any.
template <int DT> __device__ __forceinline__ void store_row(void *y, int64_t at, uint32_t n, uint32_t N, v4f a)
{
    if (n + 4u <= N) put_four<DT>(y, at + n, a);
    else
#pragma unroll
        for (int j = 0; j < 4; ++j) if (n + j < N) put<DT>(y, at + n + j, a[j]);
}

// A tile of results of 16 bits on its way to memory, by way of LDS, where a wave's lanes trade pieces: a wave's 16 MT rows of 16 NU columns, 16
// bytes of a row to a lane in the end, and whole rows of the wave's to a store.  The pieces of a row lie in an order of its own, for
// the banks.  put() for every row t of the lane, flush() once; a barrier first, since the tile's stages lay there.
template <int DT, class T> struct TileStore {
    static_assert(DT != RS_DTYPE_F32 && 16u * T::MT * 32u * T::NU * T::kWaves <= T::kLds, "16 bits; the tile fits where its stages were");
    static constexpr uint32_t kPieces = 2u * T::NU, kRow = 16u * kPieces;
    char *at;
    __device__ __forceinline__ explicit TileStore(char *lds) : at(lds + wave_id() * (16u * T::MT * kRow)) { __syncthreads(); }
    static __device__ __forceinline__ uint32_t two(float a, float b)
    {
        if constexpr (DT == RS_DTYPE_BF16) { const __bf16 v[2] = {(__bf16)a, (__bf16)b}; return __builtin_bit_cast(uint32_t, v); }
        else { const _Float16 v[2] = {(_Float16)a, (_Float16)b}; return __builtin_bit_cast(uint32_t, v); }
    }
    __device__ __forceinline__ void put(int t, const v4f (&v)[T::NU]) const
    {
        const uint32_t i = threadIdx.x % 16u, part = threadIdx.x % 64u / 16u;
        char *row = at + (t * 16u + i) * kRow;
        if constexpr (T::PAIRS) {
#pragma unroll
            for (int u = 0; u < T::NU; u += 2)
                *(uint4 *)(row + (((uint32_t)u * 2u + part) ^ (i % kPieces)) * 16u) =
                    make_uint4(two(v[u][0], v[u][1]), two(v[u][2], v[u][3]), two(v[u + 1][0], v[u + 1][1]), two(v[u + 1][2], v[u + 1][3]));
        } else {
#pragma unroll
            for (int u = 0; u < T::NU; ++u)
                *(uint2 *)(row + (((uint32_t)u * 2u + part / 2u) ^ (i % kPieces)) * 16u + part % 2u * 8u) = make_uint2(two(v[u][0], v[u][1]), two(v[u][2], v[u][3]));
        }
    }
    __device__ __forceinline__ void flush(const T &tile, void *y, int64_t y_stride, uint32_t M, uint32_t N) const
    {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const uint32_t lane = threadIdx.x % 64u, piece = lane % kPieces, n = tile.n0 + wave_id() % T::WN * (16u * T::NU) + piece * 8u;
        const uint32_t first = tile.m0 + wave_id() / T::WN * (16u * T::MT);
#pragma unroll
        for (uint32_t r = lane / kPieces; r < 16u * T::MT; r += 64u / kPieces) {
            const uint4 v = *(const uint4 *)(at + r * kRow + (piece ^ (r % 16u % kPieces)) * 16u);
            const uint32_t m = first + r;
            if (m >= M || n >= N) continue;
            uint16_t *to = (uint16_t *)y + (int64_t)m * y_stride + n;
            if (n + 8u <= N) __builtin_memcpy(to, &v, 16);
            else {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (uint32_t j = 0; j < 7; ++j) if (n + j < N) to[j] = (uint16_t)(w[j / 2] >> (16 * (j % 2)));
            }
        }
    }
};

// The same for results of 32 bits, sixteen rows of a wave at a time: put() and flush() for every row t of the lane.
template <class T> struct TileStore<RS_DTYPE_F32, T> {
    static constexpr uint32_t kPieces = 4u * T::NU, kRow = 16u * kPieces;
    static_assert(16u * kRow * T::kWaves <= T::kLds && !T::PAIRS, "sixteen rows of every wave fit where the tile's stages were");
    char *at;
    __device__ __forceinline__ explicit TileStore(char *lds) : at(lds + wave_id() * (16u * kRow)) { __syncthreads(); }
    __device__ __forceinline__ void put(const v4f (&v)[T::NU]) const
    {
        const uint32_t i = threadIdx.x % 16u, part = threadIdx.x % 64u / 16u;
#pragma unroll
        for (int u = 0; u < T::NU; ++u) *(v4f *)(at + i * kRow + (((uint32_t)u * 4u + part) ^ i) * 16u) = v[u];
    }
    __device__ __forceinline__ void flush(const T &tile, int t, float *y, int64_t y_stride, uint32_t M, uint32_t N) const
    {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const uint32_t lane = threadIdx.x % 64u, piece = lane % kPieces, n = tile.n0 + wave_id() % T::WN * (16u * T::NU) + piece * 4u;
        const uint32_t first = tile.m0 + wave_id() / T::WN * (16u * T::MT) + t * 16u;
#pragma unroll
        for (uint32_t r = lane / kPieces; r < 16u; r += 64u / kPieces) {
            const v4f v = *(const v4f *)(at + r * kRow + (piece ^ r) * 16u);
            if (first + r < M) store_row<RS_DTYPE_F32>(y, (int64_t)(first + r) * y_stride, n, N, v);
        }
    }
};

}  // namespace rs
