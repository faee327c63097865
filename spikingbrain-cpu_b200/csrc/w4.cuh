// 4-bit weights with group scales: the packed layout and the register conversions of its kernels.
#pragma once

#include "common.cuh"

namespace sbq {

// ---------------------------------------------------------------------------------------------
// Packed 4-bit weight.
//
// w[n, k] = q[n, k] * s[n, k / group], q an integer in [-8, 7], s a bf16.  Codes u = q + 8 are stored in
// 16-row x 128-column tiles of 1 KiB; tile (nt, kt) starts at byte (nt * KT + kt) * 1024, KT =
// ceil(k / 128).  A tile row is 64 bytes: 16-byte piece t (0..3), 32-bit word w (0..3) of it holds the
// eight columns 32 w + 8 t + {0..7}, column 2 p in bits 4 p .. 4 p + 3 and column 2 p + 1 sixteen bits
// above.  Rows past n and columns past k hold q = 0 (u = 8).
//
// Why this order: lane (g, t) of a warp reads one 16-byte piece of row g and one of row g + 8, the row
// pair of an m16n8k16 A fragment; each word is then 8 consecutive columns, whose 16-bit activations are
// one 16-byte load, and word w covers columns 32 w .. 32 w + 31 over the four lanes of a row, so a group
// of 32, 64 or 128 columns ends on a word.  Masking bits 4 p .. 4 p + 3 of both halves gives two
// neighbouring columns as one 16-bit pair.
//
// Scales: bf16, tile by tile as the codes, [nt][kt][row & 7][group in tile][row >> 3], so that a lane's
// rows g and g + 8 are one 32-bit word per group.  Groups past the end hold 0.
//
// rowmul[n]: the power of two that brings the largest |s| of row n into [2^10, 2^11) (1 for a row of
// zeros).  q has at most 3 significant bits besides its sign and s has 8, so q * s * rowmul is exact in
// fp16 for every scale down to 2^-27 of the row's largest.
// ---------------------------------------------------------------------------------------------
constexpr int kW4TileCols = 128;
constexpr int kW4TileBytes = 1024;

__host__ __device__ inline int64_t w4_tiles_k(int64_t k) { return ceil_div(k, kW4TileCols); }

// Byte offset of the word that holds columns 8 c8 .. 8 c8 + 7 of row r.
__device__ __forceinline__ int64_t w4_word_offset(int64_t r, int64_t c8, int64_t kt_total) {
    const int64_t tile = (r >> 4) * kt_total + (c8 >> 4);
    const int i = (int)(c8 & 15);  // word of the tile row: w = i / 4, t = i % 4
    return tile * kW4TileBytes + (r & 15) * 64 + (i & 3) * 16 + (i >> 2) * 4;
}

// Index (bf16 elements) of the scale of row r, group gi.
__device__ __forceinline__ int64_t w4_scale_index(int64_t r, int64_t gi, int64_t kt_total, int gpt) {
    const int64_t tile = (r >> 4) * kt_total + gi / gpt;
    return ((tile * 8 + (r & 7)) * gpt + gi % gpt) * 2 + ((r >> 3) & 1);
}

// Groups per 128-column tile; 0 for an unsupported group size.
__host__ __device__ inline int w4_groups_per_tile(int group) {
    return group == 128 ? 1 : group == 64 ? 2 : group == 32 ? 4 : 0;
}

__device__ __forceinline__ uint32_t lop3_and_or(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));  // (a & b) | c
    return d;
}

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// The published way from small integers to floats without a conversion instruction: the integer goes into the mantissa
// under an exponent that makes its last place one, and the implied leading one is subtracted with the offset.
//
// Eight codes -> four fp16 pairs of q (exact).  0x6400 | u is 1024 + u; with the code four bits higher
// it is 1024 + 16 u, so two of the four pairs need no shift: (1024 + 16 u) / 16 - 72 = u - 8.
__device__ __forceinline__ void w4_to_half(uint32_t w, uint32_t (&h)[4]) {
    const uint32_t w8 = w >> 8;
    h[0] = lop3_and_or(w, 0x000F000Fu, 0x64006400u);
    h[1] = lop3_and_or(w, 0x00F000F0u, 0x64006400u);
    h[2] = lop3_and_or(w8, 0x000F000Fu, 0x64006400u);
    h[3] = lop3_and_or(w8, 0x00F000F0u, 0x64006400u);
    const uint32_t off = 0x64086408u;    // 1032
    const uint32_t inv16 = 0x2C002C00u;  // 1/16
    const uint32_t m72 = 0xD480D480u;    // -72
    asm("sub.f16x2 %0, %0, %1;" : "+r"(h[0]) : "r"(off));
    asm("sub.f16x2 %0, %0, %1;" : "+r"(h[2]) : "r"(off));
    h[1] = hfma2(h[1], inv16, m72);
    h[3] = hfma2(h[3], inv16, m72);
}

// The same in bf16: 0x4300 | u is 128 + u (bf16 has 7 mantissa bits: every pair is shifted down).
__device__ __forceinline__ void w4_to_bf16(uint32_t w, uint32_t (&h)[4]) {
    const uint32_t one = 0x3F803F80u, m136 = 0xC308C308u;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const uint32_t v = lop3_and_or(w >> (4 * p), 0x000F000Fu, 0x43004300u);
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(h[p]) : "r"(v), "r"(one), "r"(m136));
    }
}

// ---- host: a checked 4-bit weight ------------------------------------------------------------------
struct W4Weight {
    const uint8_t* packed;
    const __nv_bfloat16* scales;
    const float* rowmul;
};

}  // namespace sbq
