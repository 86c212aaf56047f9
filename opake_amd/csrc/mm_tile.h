// One 256 x 256 tile of a product of two 16-bit matrices on the matrix cores
// (gfx950), for operands of either orientation:
//   K-contiguous: element (i, k) at p[i * ld + k]  (a row holds one index's K values)
//   K-slow:       element (i, k) at p[k * ld + i]  (a row holds one k of every index)
// or native: a [rows, columns] matrix as the matrix cores hold it, in blocks of 256
// rows x 64 columns (32 KiB each, `ld` of them side by side for every 256 rows), each
// of 1 KiB pieces of 16 rows x 32 columns: lane l's 16 bytes are row l % 16 at columns
// 4 (l / 16) + r and 16 + 4 (l / 16) + r (r < 4).  That is what a lane has in the
// accumulators of a tile whose A index is the column, so a product's result is stored
// as it is, and read back as the K-contiguous operand (index: row) of the next product
// as it is, or through the transposing reads as a K-slow one (index: column).
//
// acc[i][j] of a wave holds 16 x 16 blocks: lane l has rows 4 (l / 16) + r
// (r < 4) of operand A's index and column l % 16 of operand B's, so four
// consecutive A indices sit in a lane's four registers.  A is therefore always
// the operand whose index is contiguous in the output.
//
// float32 operands (kHalf) come as two fp16 planes, x = (x0 + x1) 2^-shift with the
// shift that brings the tensor's largest magnitude to [2^14, 2^15): x0 is x's rounding to
// 11 bits, x1 that of what it leaves.  So at most 2^-23 |x| is lost (2^-24.5 in the mean
// square), or 2^-39 of the largest where x1 is subnormal (the matrix cores keep fp16's
// subnormals).  A step of 64 k goes over the plane pairs (1, 0), (0, 1), (0, 0), one after
// the other while the caches hold them; the pair left out is at most 2^-22 of the product
// (2^-24.6), so a term is at most 2^-21 of itself away (2^-23.7).  The products are exact
// and the sums are the MFMA's float32 ones: float32 accuracy (gradients 6e-7 from 64 bits
// where products in float32 are 1.2e-6 off) at three bf16-rate products, 2500 / 3
// TFLOP/s against the float32 matrix instructions' 157.
#pragma once

#include "lds_stage.h"

struct MmOperand {
  const uint16_t* p;  // 16-byte aligned
  int64_t ld;         // elements, a multiple of 8; native: blocks
  int64_t plane;      // elements between planes
  int rows;           // valid indices
};

struct MmArgs {
  MmOperand a, b;
  int kl;      // valid K, K-contiguous operands: a multiple of 8 (zero-padded)
  int tiles_a, tiles_b;
  int splits;  // the K steps go out in this many slices
};

constexpr int kMmTile = 256, kMmStep = 64, kMmThreads = 512, kMmWaves = 8;
constexpr int kMmOperandBytes = kMmTile * kMmStep * 2;  // 32 KiB
constexpr int kMmOutOfRange = 0x7ff00000;

// A step's plane pairs, nibble i of each word: pair i's plane of A and of B.
constexpr uint32_t kMmPairsA = 0x001u, kMmPairsB = 0x010u;
constexpr int kMmPairs = 3;

// K-contiguous tile: rows of 64 k = 128 bytes, eight 16-byte chunks
// XOR-swizzled by bits 1-3 of the row.  The 64 banks span two rows, so 16
// consecutive rows of one chunk (a fragment read) land on 16 distinct 16-byte
// bank groups.
DPC_DEVICE int mm_kc_off(int row, int chunk) {
  return row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4);
}

// Linear id -> (split, tile of A, tile of B); false past the last.  Dispatch is
// round-robin over the 8 XCDs: each XCD takes a contiguous range of ids, walked in
// groups of four B tiles, so it re-reads operand tiles from its own L2.  (A workgroup
// that takes several tiles steps its id by the grid's size, a multiple of 8.)
DPC_DEVICE bool mm_tile_of(const MmArgs& g, int id, int* split, int* ta, int* tb) {
  const int tiles = g.tiles_a * g.tiles_b, n = tiles * g.splits;
  if (id >= n) return false;
  const int xcd = id & 7;
  int lin = xcd * (n >> 3) + min(xcd, n & 7) + (id >> 3);
  const int sp = lin / tiles;
  lin -= sp * tiles;
  const int per = 4 * g.tiles_a, grp = lin / per, first = grp * 4;
  const int size = min(g.tiles_b - first, 4), in = lin - grp * per;
  *tb = __builtin_amdgcn_readfirstlane(first + in % size);
  *ta = __builtin_amdgcn_readfirstlane(in / size);
  *split = __builtin_amdgcn_readfirstlane(sp);
  return true;
}

// A wave's accumulators: 128 x 64 of the tile (rows (wave & 1) * 128 of A, columns
// (wave >> 1) * 64 of B), or with kWideB 64 x 128 ((wave & 3) * 64, (wave >> 2) * 128).
// The narrow side's fragments are read half as often: it suits the operand whose
// reads cost more (K-slow ones: 109 against 250 bytes a clock).
template <bool kWideB>
struct MmAcc {
  static constexpr int kA = kWideB ? 4 : 8, kB = kWideB ? 8 : 4;
  f32x4_t v[kA][kB];
  static DPC_DEVICE int row0(int w) { return kWideB ? (w & 3) * 64 : (w & 1) * 128; }
  static DPC_DEVICE int col0(int w) { return kWideB ? (w >> 2) * 128 : (w >> 1) * 64; }
};

constexpr int64_t kMmBlock = kMmTile * kMmStep;  // elements

// A native piece in LDS: as it is where it is read by whole lanes.  For the transposing
// reads, which take 4 rows x 16 columns, slot l ^ 4 (l / 16) holds lane l's 16 bytes.
DPC_DEVICE int mm_native_slot(int row, int q) { return (row ^ (4 * q)) + 16 * q; }

// kPaired (K-contiguous): a tile is 128 rows of the matrix's first half and the same of
// its second, `rows` further on, by 64 in turn: a wave's 128 rows hold both of 64 pairs.
// (The 64 rows of transfer j are of the first half where j is even.)
template <bool kKc, bool kNative, bool kPaired = false>
struct MmStage {
  int voff[4];  // byte offsets of this lane's four 16-byte chunks of a step
  int kchunk;   // K-contiguous: first k of the lane's chunk
  DPC_DEVICE void init(const MmOperand& o, int w, int lane) {
    kchunk = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (kNative) {
        const int from = (kKc ? lane : mm_native_slot(lane & 15, lane >> 4)) * 16;
        // K-contiguous: the block as it is.  K-slow: eight pieces of 32 columns (four
        // blocks) x four of 16 rows.
        voff[j] = kKc ? (w + 8 * j) * 1024 + from
                      : (int)(j * kMmBlock * 2) + (w >> 2) * 16384 + (w & 3) * 1024 + from;
      } else if (kKc) {
        const int row = 8 * (w + 8 * j) + (lane >> 3);
        kchunk = ((lane & 7) ^ ((row >> 1) & 7)) * 8;
        const int from = kPaired ? (row >> 7) * 64 + (row & 63) : row;
        voff[j] = (int)((from * o.ld + kchunk) * 2);
      } else {
        const int row = 2 * (w + 8 * j) + (lane >> 5);
        voff[j] = (int)((row * o.ld + tile_slot_col(row, lane & 31)) * 2);
      }
    }
  }
  // The step at k0 of plane `pl` of tile t: the buffer it reads, and `bad`, out of the
  // buffer's range for lanes whose k is past kl.  Rows past the operand's are out of
  // range too: all such reads give zeros.  (Native blocks are whole; past their matrix
  // they hold zeros.)
  // kPaired: of the matrix's half `half`.
  DPC_DEVICE u32x4_t buffer(const MmOperand& o, int pl, int t, int k0, int kl, int* bad,
                            int half = 0) const {
    const uint16_t* base = o.p + (int64_t)pl * o.plane;
    uint32_t bytes;
    *bad = 0;
    constexpr int kRows = kPaired ? kMmTile / 2 : kMmTile;
    const int i0 = t * kRows;
    if (kNative && kKc) {
      base += (t * o.ld + (k0 >> 6)) * kMmBlock;
      bytes = kMmBlock * 2;
    } else if (kNative) {
      base += ((k0 >> 8) * o.ld + 4 * t) * kMmBlock + ((k0 & 255) >> 4) * 512;
      bytes = (uint32_t)(4 * kMmBlock * 2 - ((k0 & 255) >> 4) * 1024);
    } else if (kKc) {
      base += (int64_t)(kPaired ? half * o.rows + i0 : i0) * o.ld + k0;
      bytes = (uint32_t)((min(o.rows - i0, kRows) * o.ld - k0) * 2);
      *bad = k0 + kchunk >= kl ? kMmOutOfRange : 0;
    } else {
      base += (int64_t)k0 * o.ld + i0;
      bytes = (uint32_t)((min(kl - k0, kMmStep) * o.ld - i0) * 2);
    }
    return rsrc_words(base, bytes);
  }
  DPC_DEVICE void issue(u32x4_t buf, int bad, uint32_t lds, int w, int j) const {
    dma16(buf, lds + (w + 8 * j) * 1024, voff[j] | bad, 0);
  }
};

// Reads the 16 x 32 fragments of a wave's blocks from an operand's tile.  Both of a
// product's operands give the k-slots one order: by rows (K-contiguous), or that of the
// transposing reads (frag16_off: slot 8 q + 4 h + e is k = 16 h + 4 q + e), which a native
// piece has too, and rows with kSlow (two 8-byte reads).  A lane keeps a few byte offsets;
// blocks, sub-steps and stages are added as immediates.
template <bool kKc, bool kNative, int kBlocks, bool kSlow = false>
struct MmFrags {
  static constexpr int kOffsets = kNative ? 1 : kKc ? (kSlow ? 4 : 2) : kBlocks / 2;
  int o[kOffsets];
  // Tile at byte `at` of the workgroup's LDS, first block at index c0.
  DPC_DEVICE void init(int at, int c0, int lane) {
    const int row = c0 + (lane & 15), q = lane >> 4;
#pragma unroll
    for (int i = 0; i < kOffsets; ++i) {
      if (kNative && kKc)
        o[i] = at + (c0 >> 4) * 1024 + lane * 16;
      else if (kNative)  // lane L of 16: row 4 q + L / 4, columns 4 (L % 4) ..
        o[i] = at + (c0 >> 5) * 4096 + mm_native_slot(4 * q + ((lane & 15) >> 2), lane & 3) * 16;
      else if (!kKc)
        o[i] = at + frag16_off(c0 + 32 * i, 0, lane);
      else if (kSlow)  // sub-step i / 2, half i % 2: k = 16 (i % 2) + 4 q ..
        o[i] = at + mm_kc_off(row, 2 * i + (q >> 1)) + 8 * (q & 1);
      else
        o[i] = at + mm_kc_off(row, 4 * i + q);
    }
  }
  // Block i, sub-step kk, `off` bytes on (the stage).
  DPC_DEVICE bf16x8_t read(const uint8_t* lds, int i, int kk, int off) const {
    if (kNative && kKc)
      return *reinterpret_cast<const bf16x8_t*>(lds + o[0] + off + kk * 16384 + i * 1024);
    if (kNative) {  // 32 columns: four pieces of 16 rows, two of them this sub-step's
      const int p = o[0] + off + (i >> 1) * 4096 + (i & 1) * 8 + kk * 2048;
      return join_frag(read_tr(lds, p), read_tr(lds, p + 1024));
    }
    if (!kKc) {  // odd blocks are the other half of a 64-byte LDS block
      const int p = (o[i >> 1] ^ (32 * (i & 1))) + off + kk * 32 * kTileRowBytes;
      return join_frag(read_tr(lds, p), read_tr(lds, p + 16 * kTileRowBytes));
    }
    if constexpr (kSlow) {
      const int p = off + i * 2048;
      return join_frag(*reinterpret_cast<const i16x4_t*>(lds + o[2 * kk] + p),
                       *reinterpret_cast<const i16x4_t*>(lds + o[2 * kk + 1] + p));
    }
    return *reinterpret_cast<const bf16x8_t*>(lds + o[kk] + off + i * 2048);
  }
};

// A place in the K loop: plane pair and first k.  `next` stays at the last step
// past the end, so a pipeline may go on fetching (in range) into a stage that
// nothing reads.
template <bool kHalf>
struct MmPlace {
  int left, pair, k0;
  DPC_DEVICE MmPlace next() const {  // (selects: no branch in the loop)
    const int go = left > 1 ? 1 : 0;
    if (!kHalf) return MmPlace{left - go, 0, k0 + (go ? kMmStep : 0)};
    const int wrap = pair + 1 == kMmPairs ? 1 : 0;
    return MmPlace{left - go, go ? (wrap ? 0 : pair + 1) : pair,
                   k0 + (go & wrap ? kMmStep : 0)};
  }
};

// The K loop of a tile: steps of slice `split` into acc.  Two LDS stages of each
// operand (A, A, B, B: every read is a lane's offset plus a 16-bit immediate), all
// transfers straight from memory into LDS.
//
// A step is two 32-deep sub-steps of two phases of 16 MFMAs: the first and the last
// four blocks of the wide operand against the other's four.  Fragments are read one phase
// ahead.  Before phase 3 a barrier: the other stage has arrived, and this one has
// been read for the last time.  A's transfers of step s + 2 go out right after it,
// B's of step s + 1 at the start of step s, so each has most of a step or more to
// land and the barrier is the only place where a wave waits.
//
// 8192 x 2048 x 32000 in this loop alone runs at 1.34 PFLOP/s at the clocks that the card
// holds under it (1.6 to 1.7 GHz; the matrix cores are busy 68% of the time; the library's
// product of that size reaches 1.43, of 16384^3 1.6).  Without the transfers it would be
// 1.8, without the fragment reads 1.58, with neither 2.2: the 192 KiB of fragments that a
// step's waves read and the 64 KiB that come in keep the LDS as busy as the MFMAs.
// Measured and not better: four waves of 128 x 128 (the accumulators spill), waves in two
// groups that take turns (1.26), transfers through registers (spills), wave priorities,
// earlier transfers.
//
// begin() sends the first transfers, run() does the rest and ends with a barrier,
// after which `lds` is free: the next tile's begin() goes before this one's epilogue,
// so that its first step has arrived when the epilogue ends.
// kPaired: A in pairs (MmStage).  kBSlow: a K-contiguous B beside a K-slow A, whose `rows`
// are then the k that it has (B is zero beyond).
template <bool kAKc, bool kBKc, bool kBNative, bool kWideB, bool kHalf, bool kPaired = false,
          bool kBSlow = false>
struct MmTile {
  const MmArgs& g;
  uint8_t* lds;
  int lane, w, ta, tb, steps;
  MmPlace<kHalf> pa, pb;
  MmStage<kAKc, false, kPaired> sa;
  MmStage<kBKc, kBNative> sb;
  u32x4_t buf, buf2;
  int bad;

  DPC_DEVICE MmTile(const MmArgs& args, uint8_t* l) : g(args), lds(l) {
    lane = threadIdx.x & 63;
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    sa.init(g.a, w, lane);
    sb.init(g.b, w, lane);
  }
  DPC_DEVICE void next_a() {
    const int plane = kHalf ? (kMmPairsA >> (4 * pa.pair)) & 15 : 0;
    const int kl = kBSlow ? g.a.rows : g.kl;
    buf = sa.buffer(g.a, plane, ta, pa.k0, kl, &bad);
    if constexpr (kPaired) buf2 = sa.buffer(g.a, plane, ta, pa.k0, kl, &bad, 1);
    pa = pa.next();
  }
  DPC_DEVICE void next_b() {
    buf = sb.buffer(g.b, kHalf ? (kMmPairsB >> (4 * pb.pair)) & 15 : 0, tb, pb.k0, g.kl, &bad);
    pb = pb.next();
  }
  DPC_DEVICE void fetch_a(int stage, int j) {
    sa.issue(kPaired && (j & 1) ? buf2 : buf, bad, lds_addr(lds) + stage * kMmOperandBytes, w, j);
  }
  DPC_DEVICE void fetch_b(int stage, int j) {
    sb.issue(buf, bad, lds_addr(lds) + (2 + stage) * kMmOperandBytes, w, j);
  }

  static DPC_DEVICE f32x4_t mma(bf16x8_t a, bf16x8_t b, f32x4_t c) {
    typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
    if constexpr (kHalf)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a),
                                                    __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }

  DPC_DEVICE void begin(int tile_a, int tile_b, int split) {
    ta = tile_a;
    tb = tile_b;
    const long long all =
        (long long)((g.kl + kMmStep - 1) / kMmStep) * (kHalf ? kMmPairs : 1);
    const int s0 = __builtin_amdgcn_readfirstlane((int)(all * split / g.splits)),
              s1 = __builtin_amdgcn_readfirstlane((int)(all * (split + 1) / g.splits));
    steps = s1 - s0;
    if (steps <= 0) return;
    const int step0 = kHalf ? s0 / kMmPairs : s0;
    pa = MmPlace<kHalf>{steps, s0 - step0 * (kHalf ? kMmPairs : 1), step0 * kMmStep};
    pb = pa;
    next_a();
#pragma unroll
    for (int j = 0; j < 4; ++j) fetch_a(0, j);
    next_b();
#pragma unroll
    for (int j = 0; j < 4; ++j) fetch_b(0, j);
    next_a();
#pragma unroll
    for (int j = 0; j < 4; ++j) fetch_a(1, j);
  }

  DPC_DEVICE void run(MmAcc<kWideB>& acc) {
#pragma unroll
    for (int i = 0; i < MmAcc<kWideB>::kA; ++i)
#pragma unroll
      for (int j = 0; j < MmAcc<kWideB>::kB; ++j) acc.v[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (steps <= 0) return;
    static_assert(kAKc == (kBKc && !kBNative && !kBSlow), "one order of the k-slots");
    // x: the wide operand's fragments (half of its blocks), y: the narrow one's.
    bf16x8_t x0[4], x1[4], y0[4], y1[4];
    MmFrags<kAKc, false, MmAcc<kWideB>::kA> ra;
    MmFrags<kBKc, kBNative, MmAcc<kWideB>::kB, kBSlow> rb;
    ra.init(0, acc.row0(w), lane);
    rb.init(2 * kMmOperandBytes, acc.col0(w), lane);
    auto read_x = [&](int stage, int kk, int half, bf16x8_t* f, int i)
                      __attribute__((always_inline)) {
      if constexpr (kWideB)
        f[i] = rb.read(lds, 4 * half + i, kk, stage * kMmOperandBytes);
      else
        f[i] = ra.read(lds, 4 * half + i, kk, stage * kMmOperandBytes);
    };
    auto read_y = [&](int stage, int kk, bf16x8_t* f, int i) __attribute__((always_inline)) {
      if constexpr (kWideB)
        f[i] = ra.read(lds, i, kk, stage * kMmOperandBytes);
      else
        f[i] = rb.read(lds, i, kk, stage * kMmOperandBytes);
    };
    // One phase: 16 MFMAs, and after MFMA m what slot(m) issues (a fragment of the next
    // phase, a transfer); the order is the one written.
    auto phase = [&](const bf16x8_t* x, const bf16x8_t* y, int half, auto slot)
        __attribute__((always_inline)) {
#pragma unroll
      for (int m = 0; m < 16; ++m) {
        const int i = m >> 2, j = m & 3;
        if constexpr (kWideB)
          acc.v[j][4 * half + i] = mma(y[j], x[i], acc.v[j][4 * half + i]);
        else
          acc.v[4 * half + i][j] = mma(x[i], y[j], acc.v[4 * half + i][j]);
        slot(m);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto step = [&](int cur, int nxt) __attribute__((always_inline)) {
      next_b();
      __builtin_amdgcn_sched_barrier(0);
      phase(x0, y0, 0, [&](int m) __attribute__((always_inline)) {
        if (m % 2 == 0 && m < 8) read_x(cur, 0, 1, x1, m / 2);
        if (m % 4 == 3) fetch_b(nxt, m / 4);
      });
      phase(x1, y0, 1, [&](int m) __attribute__((always_inline)) {
        if (m < 8) {
          if (m & 1) read_x(cur, 1, 0, x0, m / 2);
          else read_y(cur, 1, y1, m / 2);
        }
      });
      phase(x0, y1, 0, [&](int m) __attribute__((always_inline)) {
        if (m % 2 == 0 && m < 8) read_x(cur, 1, 1, x1, m / 2);
      });
      next_a();
      DPC_WAIT_VMCNT(0);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      phase(x1, y1, 1, [&](int m) __attribute__((always_inline)) {
        if (m < 8) {
          if (m & 1) read_x(nxt, 0, 0, x0, m / 2);
          else read_y(nxt, 0, y0, m / 2);
        }
        if (m % 4 == 3) fetch_a(cur, m / 4);
      });
    };
    DPC_WAIT_VMCNT(4);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      read_y(0, 0, y0, j);
      read_x(0, 0, 0, x0, j);
    }
    int s = 0;
    for (; s + 1 < steps; s += 2) {
      step(0, 1);
      step(1, 0);
    }
    if (s < steps) step(0, 1);
    DPC_WAIT_VMCNT(0);
    __syncthreads();
  }
};
