// The microscaled four-bit format (OCP Microscaling Formats specification: MXFP4) as this package lays it out.
//
// 32 consecutive entries of a row share a scale 2^(s - 127), one byte s, 255 standing for "not a number"; an entry is a sign,
// two bits of exponent and one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6.
//
//   codes   [matrices, rows, pitch] bytes, two entries to a byte, the even one in the low half; pitch = 64 bytes for every 128
//           entries begun, so that rows start on 16-byte borders and the tensor cores' steps never leave a row; entries behind
//           the row's last are zero.
//   scales  [matrices, row tiles, column tiles, 512] bytes, a tile being 128 rows x 128 entries: byte (r % 32) * 16 + (r / 32) * 4 + b
//           for row r and block b of the tile.  That is how the block-scaled products want 128 rows' scales in tensor memory (lane
//           r % 32, column r / 32, a byte per block), so a tile goes there in one copy.  Rows and blocks that pad a tile have s = 127.
#pragma once
#include <stdint.h>

#define MX4_TILE_BYTES 512       // scales of 128 rows x 128 entries

__host__ __device__ __forceinline__ int mx4_tiles(int n) { return (n + 127) / 128; }
// 64 bytes per 128 entries begun
__host__ __device__ __forceinline__ size_t mx4_pitch(int width) { return (size_t)mx4_tiles(width) * 64; }
// the word with the four scales of a row's entries 128 * kt .. + 127
__host__ __device__ __forceinline__ size_t mx4_scale_word(int row, int kt, int k_tiles) {
  return (((size_t)(row >> 7) * k_tiles + kt) * MX4_TILE_BYTES) + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// 2^(s - 127), exactly: 2^-127 is a subnormal float; s = 255 is not a number
__device__ __forceinline__ float mx4_scale_value(unsigned s) {
  return s == 255u ? __uint_as_float(0x7fc00000u) : s == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23);
}
__device__ __forceinline__ void mx4_unpack_bf16(const uint4& raw, float (&v)[8]) {
  const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// ---- a float as two parts of eight bits -----------------------------------------------------------------------------
// The block-scaled products multiply four-bit entries with eight-bit ones (e4m3: four significant bits), so a row of more bits goes in as
// two parts: the entries of a block over 2^(E - 7), E = floor(log2(largest magnitude)), rounded to e4m3, and what is left over a scale 2^5
// less, rounded once more.  Four and four significant bits and the second part's sign hold the eight of a bfloat16: exactly, where an
// entry is at least 2^-14 of its block's largest (below, e4m3 runs out of exponents); every entry to 2^-22 of the largest.
__device__ __forceinline__ unsigned mx8_scale_high(unsigned largest_bits) {
  return largest_bits >= 0x7f800000u ? 255u : (unsigned)max((int)(largest_bits >> 23) - 7, 0);
}
__device__ __forceinline__ unsigned mx8_scale_low(unsigned high) { return high == 255u ? 255u : (unsigned)max((int)high - 5, 0); }
// Two entries: each part's bytes, the first entry's in the low half.  `high` and `low` are the parts' scales.
__device__ __forceinline__ void mx8_split(float a, float b, unsigned high, unsigned low, unsigned& high_bytes, unsigned& low_bytes) {
  if (high == 255u) { high_bytes = low_bytes = 0u; return; }
  const float inverse = __uint_as_float((254u - high) << 23), onward = __uint_as_float((127u + high - low) << 23);
  a *= inverse;
  b *= inverse;
  unsigned short h, l;
  unsigned back;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(h) : "f"(a), "f"(b));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(h));
  float back_a, back_b;
  asm("{\n.reg .b16 x, y;\nmov.b32 {x, y}, %2;\ncvt.f32.f16 %0, x;\ncvt.f32.f16 %1, y;\n}\n" : "=f"(back_a), "=f"(back_b) : "r"(back));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(l) : "f"((a - back_a) * onward), "f"((b - back_b) * onward));
  high_bytes = h;
  low_bytes = l;
}

// ---- a float as eight parts of four bits ------------------------------------------------------------------------------
// Few rows go in as eight rows of four-bit entries each: the entries of a block over 2^(E - 1), E = floor(log2(largest magnitude)), are below 4
// and rounded to the format's values, at most 0.5 off; what is left goes in over a scale 2^3 less, below 4 again, and so on.  The first
// scale is 2^-106 at least, so that the last is the format's least.  An entry is held to 2^-23 of its block's largest or to 2^-129.
#define MX4_PARTS 8
__device__ __forceinline__ unsigned mx4_first_scale(unsigned largest_bits) {
  return largest_bits >= 0x7f800000u ? 255u : max((largest_bits >> 23), 22u) - 1u;
}
__device__ __forceinline__ unsigned mx4_part_scale(unsigned first, int part) { return first == 255u ? 255u : first - 3u * part; }
__device__ __forceinline__ float mx4_over_first_scale(float v, unsigned first) {
  return first == 255u ? 0.f : v * __uint_as_float((254u - first) << 23);
}
// Eight entries to four bits each, nearest with ties to even, magnitudes above 6 to 6; the first entry in the low bits.
__device__ __forceinline__ unsigned mx4_pack_eight(const float (&v)[8]) {
  unsigned out;
  asm("{\n.reg .b8 a, b, c, d;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      "mov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(out) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return out;
}
// Two codes (a byte) to their values.
__device__ __forceinline__ void mx4_two_values(unsigned byte, float& a, float& b) {
  asm("{\n.reg .b8 c, d, e, f;\n.reg .b32 h;\n.reg .b16 x, y;\nmov.b32 {c, d, e, f}, %2;\ncvt.rn.f16x2.e2m1x2 h, c;\n"
      "mov.b32 {x, y}, h;\ncvt.f32.f16 %0, x;\ncvt.f32.f16 %1, y;\n}\n" : "=f"(a), "=f"(b) : "r"(byte));
}
// The next part of eight entries: their codes; the entries become what is left, over the next part's scale.
__device__ __forceinline__ unsigned mx4_next_part(float (&v)[8]) {
  const unsigned codes = mx4_pack_eight(v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    mx4_two_values((codes >> (8 * i)) & 255u, a, b);
    v[2 * i] = (v[2 * i] - a) * 8.f;
    v[2 * i + 1] = (v[2 * i + 1] - b) * 8.f;
  }
  return codes;
}
// One entry: the codes of all its parts, the first in the low bits.
__device__ __forceinline__ unsigned mx4_all_parts(float v) {
  unsigned all = 0u;
#pragma unroll
  for (int part = 0; part < MX4_PARTS; ++part) {
    unsigned code;
    asm("{\n.reg .b8 a;\ncvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\nmov.b32 %0, {a, a, a, a};\n}\n" : "=r"(code) : "f"(v), "f"(0.f));
    float a, b;
    mx4_two_values(code, a, b);
    all |= (code & 15u) << (4 * part);
    v = (v - a) * 8.f;
  }
  return all;
}
