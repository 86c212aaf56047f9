// What the products on the matrix cores (mm_tile.h) share besides the tile: float32
// operands as fp16 planes, the K slices of products of few tiles, and stores of a tile's
// quads.
#pragma once

#include "mm_tile.h"

// float32 as two fp16 planes (mm_tile.h): the shift that brings magnitude `top` (the
// float's bits) to [2^14, 2^15), and plane p of an x that is already shifted.
DPC_DEVICE int half_shift(uint32_t top) {
  const int e = (int)(top >> 23) & 255;
  return top == 0 ? 0 : 14 + 127 - (e ? e : 1);
}

DPC_DEVICE uint16_t half_plane(float x, int p) {
  const _Float16 x0 = (_Float16)x;
  if (p == 0) return __builtin_bit_cast(uint16_t, x0);
  const float rest = x - (float)x0;  // not finite: plane 0 carries it
  return __builtin_bit_cast(uint16_t, (_Float16)(fabsf(x) < INFINITY ? rest : 0.f));
}

DPC_DEVICE uint32_t finite_bits(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

DPC_DEVICE uint32_t wave_max_bits(uint32_t x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, d));
  return x;
}

DPC_DEVICE int tiles_of(int rows) { return (rows + kMmTile - 1) / kMmTile; }

constexpr int kUnits = 256;  // compute units of an MI355X

// K slices of a product of `tiles` tiles, none under 8 steps: one, or as many as fill one
// or two rounds, whichever makes least of the rounds (1.4 us a step, 10 a round) and of
// the results' way to memory and back (0.11 us each).  In integers: several kernels have
// to agree on it.  (dH of 2790 rows, 1000 wide, vocabulary 50001, 44 tiles: 288 us in 5
// slices, 335 in 4.  Of 4900 rows, 2048 wide, vocabulary 32000, 160 tiles: 597 us in 3
// slices, 756 in one.)
constexpr int kMostSliced = 512;  // tiles times slices, if more than one

DPC_HOST_DEVICE int slices(int64_t tiles, int64_t steps) {
  if (tiles < 1 || 2 * tiles > kMostSliced || steps < 16) return 1;
  const int n = (int)tiles, k = steps < 1 << 20 ? (int)steps : 1 << 20;
  int best = 1, least = 140 * k + 1000;  // (one round: more than 256 tiles do not get here)
  for (int r = 1; r <= kMostSliced / kUnits; ++r) {
    int s = r * kUnits / n;
    if (s > k / 8) s = k / 8;
    if (s > 32) s = 32;
    const int t = r * (140 * (k / s) + 1000) + 11 * n * s;
    if (s > 1 && t < least) {
      best = s;
      least = t;
    }
  }
  return best;
}

DPC_DEVICE f32x4_t shifted(f32x4_t x, int n) {
  return n ? f32x4_t{ldexpf(x[0], n), ldexpf(x[1], n), ldexpf(x[2], n), ldexpf(x[3], n)} : x;
}

DPC_DEVICE void store_row4(void* out, int64_t at, int left, bool whole, int bf16, f32x4_t x) {
  if (whole) {  // rows of whole quads
    if (bf16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) =
          make_uint2(f32x2_to_bf16x2_bits(x[0], x[1]), f32x2_to_bf16x2_bits(x[2], x[3]));
    else
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(out) + at) = x;
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r < left) {
      if (bf16)
        static_cast<uint16_t*>(out)[at + r] = f32_to_bf16_bits(x[r]);
      else
        static_cast<float*>(out)[at + r] = x[r];
    }
}

inline int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
