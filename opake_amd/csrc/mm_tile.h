// One 256 x 256 tile of a product of two bf16 matrices on the matrix cores
// (gfx950), for operands of either orientation:
//   K-contiguous: element (i, k) at p[i * ld + k]  (a row holds one index's K values)
//   K-slow:       element (i, k) at p[k * ld + i]  (a row holds one k of every index)
//
// acc[i][j] of a wave holds 16 x 16 blocks: lane l has rows 4 (l / 16) + r
// (r < 4) of operand A's index and column l % 16 of operand B's, so four
// consecutive A indices sit in a lane's four registers.  A is therefore always
// the operand whose index is contiguous in the output.
//
// float32 operands come as three bf16 planes, x = x0 + x1 + x2 exactly, each the
// rounding of what the ones before leave (|x1| <= 2^-9 |x|, |x2| <= 2^-18 |x|).
// The K loop runs over six plane pairs, smallest first: (0,2) (1,1) (2,0) (0,1)
// (1,0) (0,0); the three left out are below 2^-26 of the product.  The products
// are exact and the sums are the MFMA's float32 ones.  At 6 of the bf16 rate's
// 2500 TFLOP/s this is 2.6 times the float32 matrix instructions' 157.
#pragma once

#include "lds_stage.h"

struct MmOperand {
  const uint16_t* p;  // 16-byte aligned
  int64_t ld;         // elements, a multiple of 8
  int64_t plane;      // elements between planes
  int rows;           // valid indices
};

struct MmArgs {
  MmOperand a, b;
  int kl;      // valid K, K-contiguous operands: a multiple of 8 (zero-padded)
  int planes;  // 1 (bf16) or 3 (float32)
  int tiles_a, tiles_b;
  int splits;  // the K steps go out in this many slices
};

constexpr int kMmTile = 256, kMmStep = 64, kMmThreads = 512, kMmWaves = 8;
constexpr int kMmOperandBytes = kMmTile * kMmStep * 2;  // 32 KiB
constexpr int kMmOutOfRange = 0x7ff00000;

// Plane pairs, nibble i of each word: pair i's plane of A and of B.
constexpr uint32_t kMmPairsA = 0x010210u, kMmPairsB = 0x001012u;

// K-contiguous tile: rows of 64 k = 128 bytes, eight 16-byte chunks
// XOR-swizzled by bits 1-3 of the row.  The 64 banks span two rows, so 16
// consecutive rows of one chunk (a fragment read) land on 16 distinct 16-byte
// bank groups.
DPC_DEVICE int mm_kc_off(int row, int chunk) {
  return row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4);
}

DPC_DEVICE int mm_steps(const MmArgs& g) {
  return (g.planes == 1 ? 1 : 6) * ((g.kl + kMmStep - 1) / kMmStep);
}

// Linear workgroup id -> (split, tile of A, tile of B); false past the last.
// Dispatch is round-robin over the 8 XCDs: each XCD takes a contiguous range of
// ids, walked in groups of four B tiles, so it re-reads operand tiles from its own
// L2.
DPC_DEVICE bool mm_tile_of(const MmArgs& g, int* split, int* ta, int* tb) {
  const int tiles = g.tiles_a * g.tiles_b, n = tiles * g.splits, blk = blockIdx.x;
  if (blk >= n) return false;
  const int xcd = blk & 7;
  int lin = xcd * (n >> 3) + min(xcd, n & 7) + (blk >> 3);
  const int sp = lin / tiles;
  lin -= sp * tiles;
  const int per = 4 * g.tiles_a, grp = lin / per, first = grp * 4;
  const int size = min(g.tiles_b - first, 4), in = lin - grp * per;
  *tb = __builtin_amdgcn_readfirstlane(first + in % size);
  *ta = __builtin_amdgcn_readfirstlane(in / size);
  *split = __builtin_amdgcn_readfirstlane(sp);
  return true;
}

// The wave's 128 x 64 accumulators: rows (wave & 1) * 128 of A, columns
// (wave >> 1) * 64 of B.
struct MmAcc {
  f32x4_t v[8][4];
};

template <bool kKc>
struct MmStage {
  int voff[4];  // byte offsets of this lane's four 16-byte chunks of a step
  int kchunk;   // K-contiguous: first k of the lane's chunk
  DPC_DEVICE void init(const MmOperand& o, int w, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (kKc) {
        const int row = 8 * (w + 8 * j) + (lane >> 3);
        kchunk = ((lane & 7) ^ ((row >> 1) & 7)) * 8;
        voff[j] = (int)((row * o.ld + kchunk) * 2);
      } else {
        const int row = 2 * (w + 8 * j) + (lane >> 5);
        voff[j] = (int)((row * o.ld + tile_slot_col(row, lane & 31)) * 2);
      }
    }
  }
  // Step at k0 of plane `pl` of the tile from index i0, into LDS address `lds`.
  // Rows past the operand's and k past kl are out of the buffer's range (zeros).
  DPC_DEVICE void issue(const MmOperand& o, int pl, int i0, int k0, int kl, uint32_t lds,
                        int w) const {
    const uint16_t* base = o.p + (int64_t)pl * o.plane;
    uint32_t bytes;
    int bad = 0;
    if (kKc) {
      base += (int64_t)i0 * o.ld + k0;
      bytes = (uint32_t)((min(o.rows - i0, kMmTile) * o.ld - k0) * 2);
      bad = k0 + kchunk >= kl ? kMmOutOfRange : 0;
    } else {
      base += (int64_t)k0 * o.ld + i0;
      bytes = (uint32_t)((min(kl - k0, kMmStep) * o.ld - i0) * 2);
    }
    const u32x4_t rs = rsrc_words(base, bytes);
#pragma unroll
    for (int j = 0; j < 4; ++j) dma16(rs, lds + (w + 8 * j) * 1024, voff[j] | bad, 0);
  }
};

// Fragment of 16 indices from c0, 32-deep sub-step kk.  kMixed: the other
// operand is K-slow, whose transposing reads fix the order of the k-slots
// (frag16_off: slot 8 q + 4 h + e is k = 16 h + 4 q + e).
template <bool kKc, bool kMixed>
DPC_DEVICE bf16x8_t mm_frag(const uint8_t* tile, int c0, int kk, int lane) {
  if (!kKc) {
    const int o = frag16_off(c0, 0, lane) + kk * 32 * kTileRowBytes;
    return join_frag(read_tr(tile, o), read_tr(tile, o + 16 * kTileRowBytes));
  }
  const int row = c0 + (lane & 15), q = lane >> 4;
  if (!kMixed)
    return *reinterpret_cast<const bf16x8_t*>(tile + mm_kc_off(row, 4 * kk + q));
  const i16x4_t lo = *reinterpret_cast<const i16x4_t*>(
      tile + mm_kc_off(row, 4 * kk + (q >> 1)) + 8 * (q & 1));
  const i16x4_t hi = *reinterpret_cast<const i16x4_t*>(
      tile + mm_kc_off(row, 4 * kk + 2 + (q >> 1)) + 8 * (q & 1));
  return join_frag(lo, hi);
}

// The K loop of one tile: steps [s0, s1) into acc.  One LDS stage (64 KiB of
// `lds`).  Ends with a barrier, after which `lds` is free.
template <bool kAKc, bool kBKc>
DPC_DEVICE void mm_loop(const MmArgs& g, int ta, int tb, int split, uint8_t* lds, MmAcc& acc) {
  const int tid = threadIdx.x, lane = tid & 63,
            w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w & 1, wn = w >> 1;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc.v[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int ks = max(1, (g.kl + kMmStep - 1) / kMmStep);
  const long long n = mm_steps(g);
  const int s0 = (int)(n * split / g.splits), s1 = (int)(n * (split + 1) / g.splits);
  int pair = s0 / ks, k0 = (s0 - pair * ks) * kMmStep;
  pair = __builtin_amdgcn_readfirstlane(g.planes == 1 ? 5 : pair);
  k0 = __builtin_amdgcn_readfirstlane(k0);
  uint8_t* la = lds;
  uint8_t* lb = lds + kMmOperandBytes;
  MmStage<kAKc> sa;
  MmStage<kBKc> sb;
  sa.init(g.a, w, lane);
  sb.init(g.b, w, lane);
  constexpr bool kMixed = kAKc != kBKc;
  for (int s = s0; s < s1; ++s) {
    sa.issue(g.a, (kMmPairsA >> (4 * pair)) & 15, ta * kMmTile, k0, g.kl, lds_addr(la), w);
    sb.issue(g.b, (kMmPairsB >> (4 * pair)) & 15, tb * kMmTile, k0, g.kl, lds_addr(lb), w);
    k0 += kMmStep;
    if (k0 >= g.kl) {
      k0 = 0;
      ++pair;
    }
    DPC_WAIT_VMCNT(0);
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8_t fb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) fb[j] = mm_frag<kBKc, kMixed>(lb, wn * 64 + j * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bf16x8_t fa = mm_frag<kAKc, kMixed>(la, wm * 128 + i * 16, kk, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc.v[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa, fb[j], acc.v[i][j], 0, 0, 0);
      }
    }
    __syncthreads();
  }
}
