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
#define MX4_BLOCK 32

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
// the value of a code: below 1 the half is the only one
__device__ __forceinline__ float mx4_code_value(unsigned code) {
  const unsigned magnitude = code & 7u;
  const float v = magnitude < 2u ? 0.5f * (float)magnitude : __uint_as_float(((126u + (magnitude >> 1)) << 23) | ((magnitude & 1u) << 22));
  return code & 8u ? -v : v;
}
