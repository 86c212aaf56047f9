// Softmax attention with shared key heads, and its gradients.
//
//   s_ij = scale q_i . k_j over the keys j that query i sees,  p = softmax_j(s)
//   o_i = sum_j p_ij v_j,  lse_i = log2 sum_j exp(s_ij)
//   D_i = do_i . o_i,  ds = p (do v^T - D)
//   dq = scale ds k,  dk = scale ds^T q,  dv = p^T do
//
// What a query sees is an interval of keys, [lo, hi], of its position alone (causal,
// windows, lengths; empty for padding).  The heads that share a key head are rows of one
// matrix: row r = token * rep + head, so that a tile of rows reads its keys once for all
// of them and the sums of dk and dv over the heads are sums over rows.
//
// Nothing of size [T, S] is kept: the forward goes over the keys once with a running
// maximum and sum, and the backward forms p again from lse.  The gradients are two launches,
// dq (rows fixed, keys walked; D too) and dk, dv (keys fixed, rows walked): seven products
// where one launch would have five, but then dq would be added up by atomics, whose order
// changes results.
//
// A wave holds 32 columns of the transposed scores (one a lane, twice), so a row's
// statistics are a lane's own and its other half's, and the exponentials are where the
// next product takes them: the scores' tile comes out of the matrix cores as keys 8 a + 4
// (lane / 32) + b, which is made the order of the sum of the second product by reading
// its other operand so (transposing LDS reads).  So probabilities stay in registers.
//
// bf16: probabilities, ds and their operands go to the matrix cores in bf16, 2^-8 of each
// at most, the size of the results' own rounding; scores, statistics and sums are float32.
// float32: the float32 matrix instructions, nothing is rounded to less.
#include <math.h>

#include "common.h"
#include "lds_stage.h"

namespace {

constexpr int kOutOfRange = 0x7ff00000;  // a byte offset past every buffer
constexpr int kBufferBytes = 0x7ff00000;
constexpr int kRowsWave = 32;

extern __shared__ __attribute__((aligned(16))) uint8_t lds_dyn[];

DPC_DEVICE int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A buffer at an address that is the wave's, of which the compiler may not know that.
DPC_DEVICE u32x4_t wave_buffer(const void* base, int bytes) {
  u32x4_t r = rsrc_words(base, bytes);
  r[0] = uniform(r[0]);
  r[1] = uniform(r[1]);
  r[2] = uniform(r[2]);
  return r;
}

// All but the wave's last kLeft transfers into LDS have arrived, and its reads of LDS are
// done (their place may be written again); no access moves across.
template <int kLeft>
DPC_DEVICE void transfers_left() {
  static_assert(kLeft < 64, "six bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLeft) : "memory");
}

// LDS by byte address: with the tile's place a constant, reads take it as their immediate.
template <typename V>
DPC_DEVICE V lds_read(int at) {
  return *(const __attribute__((address_space(3))) V*)(uint32_t)at;
}
DPC_DEVICE i16x4_t lds_read_tr(int at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(uint32_t)at);
}

// n / d for 0 <= n < 2^31 by a multiplication: the factor ceil(2^(31 + s) / d) with 2^(s - 1)
// < d <= 2^s is e / d too large with e < 2^s, so the quotient is n e / (d 2^(31 + s)) < 1 / d.
struct Divisor {
  uint32_t mul;
  int shift, d;
  DPC_DEVICE int of(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};

struct Places {  // of one tensor: elements between examples, tokens and heads
  int64_t b, t, head;
};

struct AttnArgs {
  const void *q, *k, *v, *out, *dout;
  Places pq, pk, pv, pdo;  // out, what is kept and the gradients are contiguous
  void *o, *dq, *dk, *dv;
  // Kept for the backward.  bf16: lse = log2 of a row's sum of exponentials (+inf: it sees
  // nothing) and what rounding took from out (`rest`, by its own places).  float32: the
  // maximum that exponentials are taken against (+inf) and one over their sum, since
  // their logarithm rounded to a float is 2^-20 of the probabilities off.
  float *lse, *inv;        // [B, KV, rows]
  int8_t* rest;
  float* delta;            // -D
  int B, T, S, KV, rep, h;
  int rows;                // of a key head: T * rep
  const int64_t *lengths, *starts;
  int causal, window;
  float scale, c;          // c = scale log2(e)
  int tiles;               // row tiles (dk, dv: key tiles) of a key head
  int per_xcd, chunk;      // key heads of an XCD (0: not divided among them), of a chunk
  int block0;              // workgroups in the launches before (see Launch::go)
  Divisor by_rep, by_kv;
  // Keys in splits (few rows): partial results.
  int splits;
  float* part_o;           // [splits][B * KV * rows][h]
  float2* part_ml;         // [splits][B * KV * rows]: maximum, sum
};

// ---------------------------------------------------------------------------
// What queries see.
// ---------------------------------------------------------------------------

struct Sight {
  int len, start, causal, window;
  DPC_DEVICE Sight(const AttnArgs& a, int b) : causal(a.causal), window(a.window) {
    int64_t n = a.lengths ? a.lengths[b] : a.S;
    n = n < 0 ? 0 : (n < a.S ? n : a.S);
    len = uniform((int)n);
    int64_t s = a.starts ? a.starts[b] : (int64_t)a.S - a.T;
    const int64_t most = 1 << 30;
    s = s < -most ? -most : (s < most ? s : most);
    start = uniform((int)s);
  }
  // The first and last token that see a key at all, of [t0, t1].
  DPC_DEVICE int first(int t0) const { return causal ? max(t0, -start) : t0; }
  DPC_DEVICE int last(int t1) const {
    return len == 0 ? -1 : (causal ? min(t1, len - 1 - start) : t1);
  }
  // Of a token that does (both grow with the token).
  DPC_DEVICE int lo(int t) const {
    return causal && window ? max(0, start + t - window + 1) : 0;
  }
  DPC_DEVICE int hi(int t) const { return causal ? start + t : len - 1; }
};

// The tokens of rows [r0, r1) that see a key (none: t_first > t_last), the keys that one of
// them sees, and those that all of them see.
struct RowRange {
  int t_first, t_last, lo, hi, lo_all, hi_all;
  bool none;
  DPC_DEVICE RowRange(const AttnArgs& a, const Sight& s, int r0, int r1) {
    t_first = uniform(s.first(a.by_rep.of(r0)));
    t_last = uniform(r1 > r0 ? s.last(a.by_rep.of(r1 - 1)) : -1);
    none = t_first > t_last;
    lo = uniform(s.lo(t_first));
    hi = uniform(none ? -1 : s.hi(t_last));
    lo_all = uniform(s.lo(t_last));
    hi_all = uniform(s.hi(t_first));
  }
};

// Linear id -> (key head of the batch, tile).  Each XCD takes its own key heads, so that
// the tiles of one read its operands from one L2, and of those a few (`chunk`) at a time, the
// tiles with most work of all of them first: started last, they would end long after the
// others (8 x 2048 tokens, 32 heads over 8: a quarter of the time with each key head's
// tiles by themselves).
DPC_DEVICE void place_of(const AttnArgs& a, int tiles, int* bk, int* tile) {
  int x = a.block0 + blockIdx.x, first = 0, heads = a.B * a.KV;
  if (a.per_xcd) {
    heads = a.per_xcd;
    first = (x & 7) * heads;
    x >>= 3;
  }
  const uint32_t size = (uint32_t)a.chunk * (uint32_t)tiles;
  const int c = uniform((uint32_t)x / size), r = x - c * (int)size;
  const int now = min(a.chunk, heads - c * a.chunk);
  *tile = uniform((uint32_t)r / (uint32_t)now);
  *bk = first + c * a.chunk + r - *tile * now;
}

// Keys in splits: linear id -> (key head, row tile, split).  Sequences differ in length, so each
// XCD, and with every split each unit, gets another example's heads; the row tiles of a
// split's keys follow each other on one XCD, if the heads are a multiple of eight.  (16
// sequences of 1 to 8192 keys, 8 key heads: 58 us, 4.6 TB/s; each XCD with its own heads 69.)
DPC_DEVICE void place_of_split(const AttnArgs& a, int* bk, int* tile, int* split) {
  const uint32_t heads = a.B * a.KV, all = heads * a.tiles, x = blockIdx.x, s = x / all,
                 r = x - s * all, t = r / heads;
  *split = uniform(s);
  *tile = uniform(t);
  *bk = uniform((r - t * heads + s * 3 * a.KV) % heads);
}

// ---------------------------------------------------------------------------
// Tiles in LDS: rows of kD elements in 16-byte chunks, chunk c of a row at slot
// c ^ swizzle(row).  16 rows of one chunk (fragment reads) lie on distinct groups of four
// banks, and so do the 64-byte blocks of 4 rows that a transposing read takes.
// ---------------------------------------------------------------------------

template <int kChunks>
DPC_DEVICE int swizzle(int row) {
  return kChunks == 8 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
}

template <typename T, int kD>
struct Tile {
  static constexpr int kRow = kD * (int)sizeof(T), kChunks = kRow / 16, kPairs = kChunks / 2,
                       kEach = 16 / (int)sizeof(T), kBlocks = kD / 32;
  static_assert(kChunks >= 8, "rows of 128 bytes at least");
};

// An operand of a lane: its column (lane % 32)'s chunks 2 i + lane / 32.
template <typename T, int kD>
struct RowFrags {
  u32x4_t v[Tile<T, kD>::kPairs];
};

DPC_DEVICE f32x16_t mma_bf16(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// bf16: a lane's places in a tile.  Fragments are read by rows (row lane % 32 of a block
// of 32, pair i of its chunks) or by columns (element lane % 32 of block d of 32, 16 rows in
// the order that row products leave a lane's column in: 4 (lane / 32) + e, then 8 more).
template <int kD>
struct Walk {
  typedef Tile<uint16_t, kD> X;
  int row0, col0[2];  // of pair 0; of block 0, either half
  // `first`: a row that the blocks are counted from.
  DPC_DEVICE void init(int lane, int first) {
    const int row = lane & 31, base = (int)lds_addr(lds_dyn) + first * X::kRow;
    row0 = base + row * X::kRow + ((swizzle<X::kChunks>(row) ^ (lane >> 5)) << 4);
    const int L = lane & 15, r = 4 * (lane >> 5) + (L >> 2);
    const int chunk = ((lane >> 4) & 1) * 2 + ((L & 3) >> 1);
#pragma unroll
    for (int half = 0; half < 2; ++half)
      col0[half] = base + (r + 8 * half) * X::kRow +
                   ((chunk ^ swizzle<X::kChunks>(r + 8 * half)) << 4) + (L & 1) * 8;
  }
  // The places of a phase's reads, made for it: kept, they would take the registers that
  // keep operands from spilling.  (The swizzle turns bits of the chunk's place alone.)
  struct Rows {
    int at[X::kPairs];
  };
  struct Cols {
    int at[2 * X::kBlocks];
  };
  DPC_DEVICE Rows rows() const {
    Rows r;
    int from = row0;
    asm volatile("" : "+v"(from));
#pragma unroll
    for (int i = 0; i < X::kPairs; ++i) r.at[i] = from ^ (i << 5);
    return r;
  }
  DPC_DEVICE Cols cols() const {
    Cols r;
    int a = col0[0], b = col0[1];
    asm volatile("" : "+v"(a), "+v"(b));
#pragma unroll
    for (int d = 0; d < X::kBlocks; ++d) {
      r.at[2 * d] = a ^ (d << 6);
      r.at[2 * d + 1] = b ^ (d << 6);
    }
    return r;
  }
  // Pair i's place from pair 0's, which is opaque so that each use has its own.
  DPC_DEVICE int first_row() const {
    int from = row0;
    asm volatile("" : "+v"(from));
    return from;
  }
  static DPC_DEVICE u32x4_t row_from(int from, int at, int e, int i) {
    return lds_read<u32x4_t>((from ^ (i << 5)) + (at + e * 32 * X::kRow));
  }
  // Block e of 32 rows of the tile at `at`.
  static DPC_DEVICE u32x4_t row(const Rows& r, int at, int e, int i) {
    return lds_read<u32x4_t>(r.at[i] + (at + e * 32 * X::kRow));
  }
  // Rows 16 j .. of block e, columns of block d.
  static DPC_DEVICE u32x4_t col(const Cols& r, int at, int e, int j, int d) {
    const int o = at + (32 * e + 16 * j) * X::kRow;
    return __builtin_bit_cast(u32x4_t, join_frag(lds_read_tr(r.at[2 * d] + o),
                                                 lds_read_tr(r.at[2 * d + 1] + o)));
  }
};

// Half j of a lane's column as the second product takes it.
DPC_DEVICE u32x4_t packed_half(const f32x16_t& x, int j) {
  u32x4_t b;
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = f32x2_to_bf16x2_bits(x[8 * j + 2 * e], x[8 * j + 2 * e + 1]);
  return b;
}

// The same products in float32 (2 matrix instructions of 64 cycles take the place of one of
// 32, so nothing but they needs an order).
template <int kD>
DPC_DEVICE f32x16_t times_rows(int tile, int row0, const RowFrags<float, kD>& b, int lane) {
  typedef Tile<float, kD> X;
  const int row = row0 + (lane & 31), sw = swizzle<X::kChunks>(row) ^ (lane >> 5);
  const uint8_t* at = lds_dyn + tile + row * X::kRow;
  f32x16_t c = {};
#pragma unroll
  for (int i = 0; i < X::kPairs; ++i) {
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(at + (((2 * i) ^ sw) << 4)),
                  y = __builtin_bit_cast(f32x4_t, b.v[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
  }
  return c;
}

template <int kD>
DPC_DEVICE void add_columns(f32x16_t* acc, int tile, int row0, const f32x16_t& x, int lane) {
  typedef Tile<float, kD> X;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = row0 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
    const int sw = swizzle<X::kChunks>(row);
#pragma unroll
    for (int d = 0; d < X::kBlocks; ++d) {
      const int col = 32 * d + (lane & 31);
      const float a = *reinterpret_cast<const float*>(
          lds_dyn + tile + row * X::kRow + (((col >> 2) ^ sw) << 4) + (col & 3) * 4);
      acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x[r], acc[d], 0, 0, 0);
    }
  }
}

// Transfers of a tile of kRows rows by kWaves waves: transfer j of a wave takes 64 chunks.
template <typename T, int kD, int kRows, int kWaves>
struct Loader {
  typedef Tile<T, kD> X;
  static constexpr int kCount = kRows * X::kChunks / (64 * kWaves);
  static_assert(kCount * 64 * kWaves == kRows * X::kChunks, "whole transfers");
  static_assert(64 * kWaves % X::kChunks == 0, "a lane keeps its place in the row");
  int voff[kCount];

  static DPC_DEVICE int row(int j, int w, int lane) {
    return (w * 64 + lane) / X::kChunks + j * (64 * kWaves / X::kChunks);
  }
  // Byte offset of the lane's chunk in its row, or out of range.
  static DPC_DEVICE int chunk(int j, int h, int w, int lane) {
    const int c = ((w * 64 + lane) & (X::kChunks - 1)) ^ swizzle<X::kChunks>(row(j, w, lane));
    return c * X::kEach < h ? c * 16 : kOutOfRange;
  }
  // Rows `stride` bytes apart.
  DPC_DEVICE void init(int stride, int h, int w, int lane) {
#pragma unroll
    for (int j = 0; j < kCount; ++j) {
      const int c = chunk(j, h, w, lane);
      voff[j] = c == kOutOfRange ? c : row(j, w, lane) * stride + c;
    }
  }
  // `limit` rows of them; the others are zeros (their offsets are past the buffer's end:
  // rows do not overlap).
  DPC_DEVICE void rows(const void* base, int stride, int limit, int h, uint32_t lds, int w) const {
    const u32x4_t buf =
        wave_buffer(base, (min(limit, kRows) - 1) * stride + h * (int)sizeof(T));
#pragma unroll
    for (int j = 0; j < kCount; ++j)
      dma16(buf, uniform(lds + (w + kWaves * j) * 1024), voff[j], 0);
  }
};

// A tile of rows of shared key heads: whole tokens of all rep heads, or where rep is over
// kRows, kRows heads of one token at a time.
struct RowTiles {
  int tokens, chunks;  // tokens a tile; tiles a token
  DPC_DEVICE RowTiles(const AttnArgs& a, int rows)
      : tokens(a.rep <= rows ? uniform((int)((unsigned)rows / (unsigned)a.rep)) : 1),
        chunks(a.rep <= rows ? 1 : uniform((int)((unsigned)(a.rep + rows - 1) / (unsigned)rows))) {}
};

// A lane's row of an operand, from memory (zeros where not valid).
template <typename T, int kD>
DPC_DEVICE void load_row(RowFrags<T, kD>& f, const T* row, bool valid, int h, int lane) {
  typedef Tile<T, kD> X;
#pragma unroll
  for (int i = 0; i < X::kPairs; ++i) {
    const int at = (2 * i + (lane >> 5)) * X::kEach;
    f.v[i] = valid && at < h ? *reinterpret_cast<const u32x4_t*>(row + at) : u32x4_t{};
  }
}

// Both halves of the wave: x of lane l and of lane l ^ 32, in either.
DPC_DEVICE void both_halves(float x, float* a, float* b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  *a = __uint_as_float(r[0]);
  *b = __uint_as_float(r[1]);
}
DPC_DEVICE float max_halves(float x) {
  float a, b;
  both_halves(x, &a, &b);
  return fmaxf(a, b);
}
DPC_DEVICE float sum_halves(float x) {
  float a, b;
  both_halves(x, &a, &b);
  return a + b;
}

// Stores a lane's column (kD elements in the row products' order, kD / 32 blocks) times f
// as row `out`, or zeros where !keep; bf16: and `rest`, if not null.
template <typename T, int kD>
DPC_DEVICE void store_row(T* out, int8_t* rest, const f32x16_t* acc, float f, bool keep, bool on,
                          int h, int lane) {
#pragma unroll
  for (int d = 0; d < kD / 32; ++d) {
    if constexpr (sizeof(T) == 2) {
      // A pair of quads of both halves makes 8 elements a lane.
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t p[4], q[2] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = acc[d][8 * j + 2 * e] * f, y = acc[d][8 * j + 2 * e + 1] * f;
          p[e] = keep ? f32x2_to_bf16x2_bits(x, y) : 0u;
          if (rest && keep)
            q[e >> 1] |= ((uint32_t)(rest_of(x, p[e] & 0xffffu) & 255) |
                          (uint32_t)(rest_of(y, p[e] >> 16) & 255) << 8) << (16 * (e & 1));
        }
        const auto lo = __builtin_amdgcn_permlane32_swap(p[0], p[2], false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap(p[1], p[3], false, false);
        const int at = 32 * d + 16 * j + 8 * (lane >> 5);
        if (on && at < h)
          *reinterpret_cast<u32x4_t*>(out + at) = u32x4_t{lo[0], hi[0], lo[1], hi[1]};
        if (rest) {
          const auto r = __builtin_amdgcn_permlane32_swap(q[0], q[1], false, false);
          if (on && at < h) *reinterpret_cast<uint2*>(rest + at) = make_uint2(r[0], r[1]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 32 * d + 8 * j + 4 * (lane >> 5);
        f32x4_t x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = keep ? acc[d][4 * j + e] * f : 0.f;
        if (on && at < h) *reinterpret_cast<f32x4_t*>(out + at) = x;
      }
    }
  }
}

// A lane's row (lane % 32 of a wave's): its token and head, whether it is one, whether it
// sees a key, and which.
struct LaneRow {
  int r, t, g, lo, span;  // keys lo .. lo + span
  bool there, sees;
  DPC_DEVICE LaneRow(const AttnArgs& a, const Sight& s, const RowRange& mine, int w0, int lane) {
    r = w0 + (lane & 31);
    there = r < a.rows;
    t = a.by_rep.of(there ? r : a.rows - 1);
    g = r - t * a.rep;
    sees = there && t >= mine.t_first && t <= mine.t_last;
    lo = sees ? s.lo(t) : 1 << 30;
    span = sees ? s.hi(t) - lo : 0;
  }
};

// Row x of a lane's column of row products, in a block of 32.
DPC_DEVICE int column_row(int x, int lane) { return 8 * (x >> 2) + 4 * (lane >> 5) + (x & 3); }

#define DPC_WALL() __builtin_amdgcn_sched_barrier(0)

// ---------------------------------------------------------------------------
// Forward.  Bound by the matrix cores and by what vector instructions the exponentials
// and the statistics cannot hide behind them; a workgroup takes 6 us before its first
// product.  bf16, causal, h = 128: 1 x 16384 tokens of 16 heads 1117 us (1.0 PFLOP/s of visible
// pairs, the matrix cores half busy, vector instructions 40%), 8 x 2048 of 32 over 8 359 (0.77),
// 16 x 1024 of 16 135 (0.51: half of each key head's tiles cross the diagonal).  float32, 8 x 1024
// of 16: h = 64 214 us, 128 422 (81 TFLOP/s).
// ---------------------------------------------------------------------------

// Row tiles of kWaves x 32 rows.  Stages of key and value tiles in LDS: as many as 128 KiB
// hold, at most four, so that a tile is asked for up to three tiles ahead.
template <typename T, int kD, int kWaves>
struct RowsShape {
  static constexpr int kRow = Tile<T, kD>::kRow;
  static constexpr int kKeys = kRow <= 512 ? 64 : 32;
  static constexpr int kBytes = kKeys * kRow;
  static constexpr int kFit = 131072 / (2 * kBytes);
  static constexpr int kStages = kWaves == 1 ? 2 : (kFit < 4 ? kFit : 4);
  static constexpr int kLds = kStages * 2 * kBytes;
  // Two waves a SIMD: the second half of them a product behind (see `late`), which needs a
  // tile for one step longer.
  static constexpr bool kLate = kWaves == 8;
  static constexpr int kNext = kStages - (kLate ? 2 : 1);
};
// Keys in splits: a wave takes 32 keys at a time into LDS of its own.
template <typename T, int kD>
struct SplitShape {
  static constexpr int kRow = Tile<T, kD>::kRow;
  static constexpr int kWaves = kRow <= 128 ? 4 : (kRow == 256 ? 2 : 1);
  static constexpr int kLds = kWaves * 4 * 32 * kRow;
};
// Rows of whose tiles two waves share a SIMD (256 registers each) and take turns: one has
// products while the other has exponentials (forward of 16 x 1024 tokens of 16 heads, h =
// 128: 144 us with one wave, 132 with two; 8 x 2048 of 32 over 8: 372 and 358).
template <typename T, int kD>
constexpr int kMostWaves = sizeof(T) == 2 && kD <= 128 ? 8 : 4;

// Fragments in flight between LDS and the matrix cores: a read is issued that many
// instructions (of 32 cycles) before its product.  (Reads waited for one by one: 170 us
// for the 16 x 1024 tokens above, 156 with these; longer rings spill.)
constexpr int kAheadRows = 8, kAheadDq = 5, kAheadKeys = 4;

template <typename T, int kD, int kWaves, bool kSplit>
__global__ void __launch_bounds__(64 * kWaves, (kWaves == 8 ? 2 : 1))
    attn_forward_kernel(AttnArgs a) {
  typedef Tile<T, kD> X;
  typedef RowsShape<T, kD, kWaves> Sh;
  constexpr int kKeys = kSplit ? 32 : Sh::kKeys, kStages = kSplit ? 2 : Sh::kStages;
  constexpr int kBytes = kKeys * X::kRow, kParts = kKeys / 32, kNext = kSplit ? 1 : Sh::kNext;
  constexpr bool kLate = !kSplit && Sh::kLate;
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  int bk, tile, split = 0;
  if (kSplit) {
    place_of_split(a, &bk, &tile, &split);
    split = split * kWaves + w;
  } else {
    place_of(a, a.tiles, &bk, &tile);
  }
  tile = a.tiles - 1 - tile;  // the longest first
  const int b = uniform(a.by_kv.of(bk)), kv = bk - b * a.KV;
  const Sight sight(a, b);
  constexpr int kTileRows = kSplit ? kRowsWave : kRowsWave * kWaves;
  const int t0 = tile * kTileRows, t1 = min(t0 + kTileRows, a.rows);
  const int w0 = kSplit ? t0 : t0 + w * kRowsWave, w1 = min(w0 + kRowsWave, t1);
  const RowRange all(a, sight, t0, t1), mine(a, sight, min(w0, a.rows), w1);
  const LaneRow me(a, sight, mine, w0, lane);
  const int64_t head = (int64_t)kv * a.rep + me.g;
  RowFrags<T, kD> q;
  load_row<T, kD>(q, static_cast<const T*>(a.q) + b * a.pq.b + me.t * a.pq.t + head * a.pq.head,
                  me.sees, a.h, lane);

  const T* kbase = static_cast<const T*>(a.k) + b * a.pk.b + kv * a.pk.head;
  const T* vbase = static_cast<const T*>(a.v) + b * a.pv.b + kv * a.pv.head;
  const int kstride = (int)(a.pk.t * sizeof(T)), vstride = (int)(a.pv.t * sizeof(T));
  const int lw = kSplit ? 0 : w;
  Loader<T, kD, kKeys, (kSplit ? 1 : kWaves)> kload, vload;
  kload.init(kstride, a.h, lw, lane);
  vload.init(vstride, a.h, lw, lane);
  const int lds0 = kSplit ? w * 4 * kBytes : 0;  // in lds_dyn
  const uint32_t lds_base = lds_addr(lds_dyn);
  Walk<(sizeof(T) == 2 ? kD : 64)> walk;
  if constexpr (sizeof(T) == 2) walk.init(lane, 0);

  f32x16_t o[X::kBlocks] = {};
  float m = -INFINITY, l = 0.f, l2 = 0.f;
  int first = all.lo / kKeys, n = all.none ? 0 : all.hi / kKeys - first + 1;
  if (kSplit && n > 0) {  // this wave's share of the row tile's keys
    const int parts = a.splits * kWaves;
    const int s0 = (int)((uint32_t)n * (uint64_t)split / (uint32_t)parts),
              s1 = (int)((uint32_t)n * (uint64_t)(split + 1) / (uint32_t)parts);
    first += s0;
    n = s1 - s0;
  }
  first = uniform(first);
  n = uniform(n);
  const int limit = min(sight.len, all.hi + 1);
  // Tile i into a stage (past the last: that again, so that the number of transfers in
  // flight is always the same).
  constexpr int kCount = 2 * decltype(kload)::kCount;
  auto fetch = [&](int i, int stage) __attribute__((always_inline)) {
    const int j0 = (first + min(i, n - 1)) * kKeys;
    const uint32_t at = lds_base + lds0 + stage * 2 * kBytes;
    kload.rows(kbase + j0 * a.pk.t, kstride, limit - j0, a.h, at, lw);
    vload.rows(vbase + j0 * a.pv.t, vstride, limit - j0, a.h, at + kBytes, lw);
  };
  // The tile's statistics go into the lane's: what the exponentials are taken against.
  auto statistics = [&](f32x16_t* s, int j0) __attribute__((always_inline)) {
    if (j0 < mine.lo_all || j0 + kKeys - 1 > mine.hi_all) {
      const int from = j0 + 4 * (lane >> 5) - me.lo;
#pragma unroll
      for (int e = 0; e < kParts; ++e)
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if ((uint32_t)(from + 32 * e + 8 * (x >> 2) + (x & 3)) > (uint32_t)me.span)
            s[e][x] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int e = 0; e < kParts; ++e)
#pragma unroll
      for (int x = 0; x < 16; ++x) top = fmaxf(top, s[e][x]);
    top = max_halves(top) * a.c;
    // The maximum follows only where exponentials would pass 2^8: sums and products
    // hold that much more easily than they are rescaled.
    if (__any(top > m + 8.f)) {
      const float to = fmaxf(m, top);
      const float f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= f;
      l2 *= f;
#pragma unroll
      for (int d = 0; d < X::kBlocks; ++d) o[d] *= f;
    }
    return m == -INFINITY ? 0.f : m;
  };
  // A tile in three: its scores, their probabilities, and the product with the values.
  f32x16_t s[kParts];
  u32x4_t p[2 * kParts];
  auto front = [&](int stage) __attribute__((always_inline)) {
    const int kt = lds0 + stage * 2 * kBytes;
#pragma unroll
    for (int e = 0; e < kParts; ++e) s[e] = f32x16_t{};
    if constexpr (sizeof(T) == 2) {
      constexpr int kAll = kParts * X::kPairs;
      const auto at = walk.rows();
      u32x4_t ring[kAheadRows];
      auto read = [&](int u) __attribute__((always_inline)) {
        if (u < kAll) ring[u % kAheadRows] = walk.row(at, kt, u / X::kPairs, u % X::kPairs);
      };
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAheadRows; ++u) read(u);
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAll; ++u) {
        s[u / X::kPairs] = mma_bf16(ring[u % kAheadRows], q.v[u % X::kPairs], s[u / X::kPairs]);
        read(u + kAheadRows);
        DPC_WALL();
      }
    } else {
#pragma unroll
      for (int e = 0; e < kParts; ++e) s[e] = times_rows<kD>(kt, 32 * e, q, lane);
    }
  };
  auto middle = [&](int i) __attribute__((always_inline)) {
    const float from = statistics(s, (first + i) * kKeys);
#pragma unroll
    for (int e = 0; e < kParts; ++e) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        s[e][x] = __builtin_amdgcn_exp2f(fmaf(s[e][x], a.c, -from));
        (x & 1 ? l2 : l) += s[e][x];
      }
      if constexpr (sizeof(T) == 2) {
        p[2 * e] = packed_half(s[e], 0);
        p[2 * e + 1] = packed_half(s[e], 1);
      }
    }
  };
  auto back = [&](int stage) __attribute__((always_inline)) {
    const int vt = lds0 + stage * 2 * kBytes + kBytes;
    if constexpr (sizeof(T) == 2) {
      constexpr int kAll = 2 * kParts * X::kBlocks;
      const auto at = walk.cols();
      u32x4_t ring[kAheadRows];
      auto read = [&](int u) __attribute__((always_inline)) {
        if (u < kAll)
          ring[u % kAheadRows] = walk.col(at, vt, u / (2 * X::kBlocks), u / X::kBlocks % 2, u % X::kBlocks);
      };
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAheadRows; ++u) read(u);
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAll; ++u) {
        o[u % X::kBlocks] = mma_bf16(ring[u % kAheadRows], p[u / X::kBlocks], o[u % X::kBlocks]);
        read(u + kAheadRows);
        DPC_WALL();
      }
    } else {
#pragma unroll
      for (int e = 0; e < kParts; ++e) add_columns<kD>(o, vt, 32 * e, s[e], lane);
    }
  };
  // Two waves a SIMD take turns: the first half of them have products (of the last tile's
  // probabilities, then scores) while the second have probabilities to form of the scores
  // that they left the step before, and then the other way round.  In step with each
  // other both would wait for the same unit.  One wave a SIMD goes tile by tile.
  const bool late = kLate && w >= kWaves / 2;
  bool pending = false;  // a tile is not through
  auto step = [&](int i, int stage) __attribute__((always_inline)) {
    transfers_left<(kNext - 1) * kCount>();
    if (!kSplit) __syncthreads();
    const int before = (stage + kStages - 1) % kStages, j0 = (first + i) * kKeys;
    const bool now = !(j0 > mine.hi || j0 + kKeys <= mine.lo);
    if (late || !kLate) fetch(i + kNext, (stage + kNext) % kStages);
    if (kLate && pending) {
      if (late) middle(i - 1);
      back(before);
    }
    if (now) front(stage);
    if (kLate && !late) fetch(i + kNext, (stage + kNext) % kStages);
    if (now && !late) middle(i);
    if (now && !kLate) back(stage);
    pending = now;
  };
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < kNext; ++i) fetch(i, i);
  }
  for (int i = 0; i < n; i += kStages) {
#pragma unroll
    for (int x = 0; x < kStages; ++x)
      if (x == 0 || i + x < n) step(i + x, x);
  }
  if (kLate && pending) {
    if (late) middle(n - 1);
    const int stage = uniform((n - 1) % kStages);
#pragma unroll
    for (int x = 0; x < kStages; ++x)
      if (x == stage) back(x);
  }
  transfers_left<0>();  // none may land in LDS that is another's
  l = sum_halves(l + l2);
  const int64_t row = (int64_t)bk * a.rows + me.r;
  if (kSplit) {
    const int64_t at = (int64_t)split * a.B * a.KV * a.rows + row;
    if (me.there && lane < 32)
      a.part_ml[at] = make_float2(me.sees ? m : -INFINITY, me.sees ? l : 0.f);
    store_row<float, kD>(a.part_o + at * a.h, nullptr, o, 1.f, me.sees, me.there, a.h, lane);
    return;
  }
  // (A row that sees keys has l > 0, but where all of its scores are -inf: NaN there.)
  if (me.there && lane < 32 && a.lse) {
    if constexpr (sizeof(T) == 2) {
      a.lse[row] = me.sees ? m + __builtin_amdgcn_logf(l) : INFINITY;
    } else {
      a.lse[row] = me.sees ? m : INFINITY;
      a.inv[row] = me.sees ? 1.f / l : 0.f;
    }
  }
  const int64_t flat = (((int64_t)b * a.T + me.t) * a.KV * a.rep + head) * a.h;
  store_row<T, kD>(static_cast<T*>(a.o) + flat, a.rest ? a.rest + flat : nullptr, o, 1.f / l,
                   me.sees, me.there, a.h, lane);
}

// The splits of a row joined: one wave a row.  Lane p has parts p, p + 64, ... weighed
// (kMostParts), then the wave adds up the parts' outputs, eight loads in flight.
constexpr int kMostParts = 256;

DPC_DEVICE float wave_max(float x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
DPC_DEVICE float wave_sum(float x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a, int parts) {
  __shared__ float weights[4][kMostParts];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t n = (int64_t)a.B * a.KV * a.rows;
  const int64_t row = (int64_t)blockIdx.x * 4 + w;
  if (row >= n) return;
  float2 x[kMostParts / 64];
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < kMostParts / 64; ++e) {
    const int p = lane + 64 * e;
    x[e] = p < parts ? a.part_ml[p * n + row] : make_float2(-INFINITY, 0.f);
    m = fmaxf(m, x[e].x);
  }
  m = wave_max(m);
  const float from = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[4] = {};
#pragma unroll
  for (int e = 0; e < kMostParts / 64; ++e) {
    const float f = __builtin_amdgcn_exp2f(x[e].x - from);
    l += x[e].y * f;
    weights[w][lane + 64 * e] = f;  // (the wave's own)
  }
  l = wave_sum(l);
  const int blocks = (a.h + 63) >> 6;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (e >= blocks) break;
    const int c = min(lane + 64 * e, a.h - 1);
    const float* from_o = a.part_o + row * a.h + c;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) o[e] = fmaf(from_o[p * n * a.h], weights[w][p], o[e]);
  }
  const int64_t bk = row / a.rows, r = row - bk * a.rows, b = bk / a.KV, kv = bk - b * a.KV,
                t = r / a.rep, g = r - t * a.rep;
  const Sight sight(a, uniform((int)b));
  const bool some = sight.first((int)t) == (int)t && sight.last((int)t) == (int)t;
  if (a.lse && lane == 0) {
    if constexpr (sizeof(T) == 2) {
      a.lse[row] = some ? m + __builtin_amdgcn_logf(l) : INFINITY;
    } else {
      a.lse[row] = some ? m : INFINITY;
      a.inv[row] = some ? 1.f / l : 0.f;
    }
  }
  const int64_t flat = ((b * a.T + t) * a.KV * a.rep + kv * a.rep + g) * a.h;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 64 * e < a.h) {
      const float x = some ? o[e] / l : 0.f;
      const int64_t at = flat + lane + 64 * e;
      if constexpr (sizeof(T) == 2) {
        const uint16_t hi = f32_to_bf16_bits(x);
        static_cast<uint16_t*>(a.o)[at] = hi;
        if (a.rest) a.rest[at] = (int8_t)rest_of(x, hi);
      } else {
        static_cast<float*>(a.o)[at] = x;
      }
    }
}

// ---------------------------------------------------------------------------
// dq and D: rows fixed, keys walked.  The forward's walk with a product more; what bounds
// it is the same: 8 x 2048 tokens of 32 heads over 8 515 us (0.80 PFLOP/s of its three
// products), 16 x 1024 of 16 199 (0.52).  float32, 8 x 1024 of 16: h = 64 286 us, 128 559.
// ---------------------------------------------------------------------------

template <typename T, int kD, int kWaves>
__global__ void __launch_bounds__(64 * kWaves, (kWaves == 8 ? 2 : 1))
    attn_dq_kernel(AttnArgs a) {
  typedef Tile<T, kD> X;
  typedef RowsShape<T, kD, kWaves> Sh;
  constexpr int kKeys = Sh::kKeys, kBytes = Sh::kBytes, kStages = Sh::kStages;
  constexpr int kParts = kKeys / 32, kNext = Sh::kNext;
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  int bk, tile;
  place_of(a, a.tiles, &bk, &tile);
  tile = a.tiles - 1 - tile;
  const int b = uniform(a.by_kv.of(bk)), kv = bk - b * a.KV;
  const Sight sight(a, b);
  const int t0 = tile * kRowsWave * kWaves, t1 = min(t0 + kRowsWave * kWaves, a.rows);
  const int w0 = t0 + w * kRowsWave, w1 = min(w0 + kRowsWave, t1);
  const RowRange all(a, sight, t0, t1), mine(a, sight, min(w0, a.rows), w1);
  const LaneRow me(a, sight, mine, w0, lane);
  const int64_t head = (int64_t)kv * a.rep + me.g, row = (int64_t)bk * a.rows + me.r;
  const int64_t flat = (((int64_t)b * a.T + me.t) * a.KV * a.rep + head) * a.h;

  const T* kbase = static_cast<const T*>(a.k) + b * a.pk.b + kv * a.pk.head;
  const T* vbase = static_cast<const T*>(a.v) + b * a.pv.b + kv * a.pv.head;
  const int kstride = (int)(a.pk.t * sizeof(T)), vstride = (int)(a.pv.t * sizeof(T));
  Loader<T, kD, kKeys, kWaves> kload, vload;
  kload.init(kstride, a.h, w, lane);
  vload.init(vstride, a.h, w, lane);
  const uint32_t lds_base = lds_addr(lds_dyn);
  const int first = uniform(all.lo / kKeys),
            n = uniform(all.none ? 0 : all.hi / kKeys - first + 1);
  const int limit = min(sight.len, all.hi + 1);
  constexpr int kCount = 2 * decltype(kload)::kCount;
  auto fetch = [&](int i, int stage) __attribute__((always_inline)) {
    const int j0 = (first + min(i, n - 1)) * kKeys;
    const uint32_t at = lds_base + stage * 2 * kBytes;
    kload.rows(kbase + j0 * a.pk.t, kstride, limit - j0, a.h, at, w);
    vload.rows(vbase + j0 * a.pv.t, vstride, limit - j0, a.h, at + kBytes, w);
  };
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < kNext; ++i) fetch(i, i);
  }

  RowFrags<T, kD> q, dout;
  load_row<T, kD>(q, static_cast<const T*>(a.q) + b * a.pq.b + me.t * a.pq.t + head * a.pq.head,
                  me.sees, a.h, lane);
  load_row<T, kD>(dout, static_cast<const T*>(a.dout) + b * a.pdo.b + me.t * a.pdo.t +
                            head * a.pdo.head, me.sees, a.h, lane);
  float D = 0.f;
#pragma unroll
  for (int i = 0; i < X::kPairs; ++i) {
    const int at = (2 * i + (lane >> 5)) * X::kEach;
    const bool on = me.sees && at < a.h;
    const u32x4_t x = on ? *reinterpret_cast<const u32x4_t*>(static_cast<const T*>(a.out) + flat +
                                                            at) : u32x4_t{};
    if constexpr (sizeof(T) == 2) {
      const uint2 y = on ? *reinterpret_cast<const uint2*>(a.rest + flat + at) : uint2{};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t word = e < 4 ? y.x : y.y;
        const int rest = (int)(word << (24 - 8 * (e & 3))) >> 24;
        const uint32_t hi = (x[e >> 1] >> (16 * (e & 1))) & 0xffffu,
                       g = (dout.v[i][e >> 1] >> (16 * (e & 1))) & 0xffffu;
        D = fmaf(with_rest(hi, rest), bf16_bits_to_f32((uint16_t)g), D);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        D = fmaf(__uint_as_float(x[e]), __uint_as_float(dout.v[i][e]), D);
    }
  }
  D = sum_halves(D);
  if (me.there && lane < 32) a.delta[row] = -D;
  const float lse = me.sees ? a.lse[row] : INFINITY;
  const float inv = sizeof(T) == 4 && me.sees ? a.inv[row] : 0.f;
  Walk<(sizeof(T) == 2 ? kD : 64)> walk;
  if constexpr (sizeof(T) == 2) walk.init(lane, 0);
  f32x16_t dq[X::kBlocks] = {};

  // A tile in three: the two products, ds of them, and its product.
  f32x16_t s[kParts], dp[kParts];
  u32x4_t p[2 * kParts];
  auto front = [&](int stage) __attribute__((always_inline)) {
    const int kt = stage * 2 * kBytes, vt = kt + kBytes;
    if constexpr (sizeof(T) == 2) {
      // Fragment u: of each block of 32 keys the keys' rows, then the values'.
      constexpr int kFront = 2 * X::kPairs;
      const auto at = walk.rows();
      u32x4_t ring[kAheadDq];
      auto read = [&](int u) __attribute__((always_inline)) {
        const int e = u / kFront, v = u % kFront;
        if (e < kParts)
          ring[u % kAheadDq] = walk.row(at, v < X::kPairs ? kt : vt, e, v % X::kPairs);
      };
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAheadDq; ++u) read(u);
      DPC_WALL();
#pragma unroll
      for (int e = 0; e < kParts; ++e) {
        s[e] = dp[e] = f32x16_t{};
#pragma unroll
        for (int v = 0; v < kFront; ++v) {
          const int u = e * kFront + v, i = v % X::kPairs;
          if (v < X::kPairs)
            s[e] = mma_bf16(ring[u % kAheadDq], q.v[i], s[e]);
          else
            dp[e] = mma_bf16(ring[u % kAheadDq], dout.v[i], dp[e]);
          read(u + kAheadDq);
          DPC_WALL();
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < kParts; ++e) {
        s[e] = times_rows<kD>(kt, 32 * e, q, lane);
        dp[e] = times_rows<kD>(vt, 32 * e, dout, lane);
      }
    }
  };
  auto middle = [&](int i) __attribute__((always_inline)) {
    const int j0 = (first + i) * kKeys;
    const bool whole = j0 >= mine.lo_all && j0 + kKeys - 1 <= mine.hi_all;
#pragma unroll
    for (int e = 0; e < kParts; ++e) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        float p = __builtin_amdgcn_exp2f(fmaf(s[e][x], a.c, -lse));
        if (sizeof(T) == 4) p *= inv;
        s[e][x] = p * (dp[e][x] - D);
      }
      if (!whole) {
        const int from = j0 + 32 * e + 4 * (lane >> 5) - me.lo;
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if ((uint32_t)(from + 8 * (x >> 2) + (x & 3)) > (uint32_t)me.span) s[e][x] = 0.f;
      }
      if constexpr (sizeof(T) == 2) {
        p[2 * e] = packed_half(s[e], 0);
        p[2 * e + 1] = packed_half(s[e], 1);
      }
    }
  };
  auto back = [&](int stage) __attribute__((always_inline)) {
    const int kt = stage * 2 * kBytes;
    if constexpr (sizeof(T) == 2) {
      constexpr int kAll = 2 * kParts * X::kBlocks;
      const auto at = walk.cols();
      u32x4_t ring[kAheadDq];
      auto read = [&](int u) __attribute__((always_inline)) {
        if (u < kAll)
          ring[u % kAheadDq] = walk.col(at, kt, u / (2 * X::kBlocks), u / X::kBlocks % 2, u % X::kBlocks);
      };
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAheadDq; ++u) read(u);
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAll; ++u) {
        dq[u % X::kBlocks] = mma_bf16(ring[u % kAheadDq], p[u / X::kBlocks], dq[u % X::kBlocks]);
        read(u + kAheadDq);
        DPC_WALL();
      }
    } else {
#pragma unroll
      for (int e = 0; e < kParts; ++e) add_columns<kD>(dq, kt, 32 * e, s[e], lane);
    }
  };
  const bool late = Sh::kLate && w >= kWaves / 2;  // as in the forward
  bool pending = false;
  auto step = [&](int i, int stage) __attribute__((always_inline)) {
    transfers_left<(kNext - 1) * kCount>();
    __syncthreads();
    const int before = (stage + kStages - 1) % kStages, j0 = (first + i) * kKeys;
    const bool now = !(j0 > mine.hi || j0 + kKeys <= mine.lo);
    if (late || !Sh::kLate) fetch(i + kNext, (stage + kNext) % kStages);
    if (Sh::kLate && pending) {
      if (late) middle(i - 1);
      back(before);
    }
    if (now) front(stage);
    if (Sh::kLate && !late) fetch(i + kNext, (stage + kNext) % kStages);
    if (now && !late) middle(i);
    if (now && !Sh::kLate) back(stage);
    pending = now;
  };
  for (int i = 0; i < n; i += kStages) {
#pragma unroll
    for (int x = 0; x < kStages; ++x)
      if (x == 0 || i + x < n) step(i + x, x);
  }
  if (Sh::kLate && pending) {
    if (late) middle(n - 1);
    const int stage = uniform((n - 1) % kStages);
#pragma unroll
    for (int x = 0; x < kStages; ++x)
      if (x == stage) back(x);
  }
  transfers_left<0>();
  // One key alone: its probability is one, and ds zero, whatever rounding left of it; but not
  // where D is no number (do, its value or its score is not finite), and so ds neither.
  const bool keep = me.span > 0 || (me.sees && !(fabsf(D) < INFINITY));
  store_row<T, kD>(static_cast<T*>(a.dq) + flat, nullptr, dq, a.scale, keep, me.there, a.h, lane);
}

// ---------------------------------------------------------------------------
// dk and dv: keys fixed, rows walked.  Four products: 8 x 2048 tokens of 32 heads over 8
// 638 us (0.86 PFLOP/s), 16 x 1024 of 16 273 (0.50).  float32, 8 x 1024 of 16: h = 64 418 us, 128
// 844.
// ---------------------------------------------------------------------------

// Key tiles of 32 keys a wave, or of 4 x 32 keys for 8 waves: then the wave and the one four on
// have the same keys, and every tile's first and second 32 rows (their sums are added
// up at the end).  Stages of row tiles as RowsShape's.
template <typename T, int kD, int kWaves>
struct KeysShape {
  static constexpr int kRow = Tile<T, kD>::kRow;
  static constexpr int kRows = kRow < 512 ? 64 : 32;  // of queries, a tile
  static constexpr int kBytes = kRows * kRow;
  static constexpr int kStats = 4 * 256;  // 64 of lse, -D, inv; and a place for nothing
  static constexpr int kStage = 2 * kBytes + kStats;
  static constexpr bool kTwo = kWaves == 8;
  static constexpr int kKeys = kTwo ? 128 : 32 * kWaves;
  // Operands of a lane's key in registers, beside 2 kD / 2 of its gradients; two waves a SIMD
  // have room for one of them, and the values stay in LDS.
  static constexpr bool kHoldK = kRow <= 512, kHoldV = kHoldK && !kTwo;
  static constexpr int kValues = kTwo ? kKeys * kRow : 0;
  static constexpr int kFit = (135168 - kValues) / kStage;
  static constexpr int kStages = kWaves == 1 ? 2 : (kFit < 4 ? kFit : 4);
  static constexpr bool kLate = kTwo;
  static constexpr int kNext = kStages - (kLate ? 2 : 1);
  static constexpr int kLds = kStages * kStage + kValues;
};

template <typename T, int kD, int kWaves>
__global__ void __launch_bounds__(64 * kWaves, (kWaves == 8 ? 2 : 1)) attn_dkv_kernel(AttnArgs a) {
  typedef Tile<T, kD> X;
  typedef KeysShape<T, kD, kWaves> Sh;
  constexpr int kRows = Sh::kRows, kBytes = Sh::kBytes;
  constexpr int kParts = kRows / 32 / (Sh::kTwo ? 2 : 1);  // of a tile, this wave's blocks
  constexpr int kStages = Sh::kStages, kNext = Sh::kNext;
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const int group = Sh::kTwo ? w >> 2 : 0, own = Sh::kTwo ? w & 3 : w;
  int bk, tile;  // the first keys are seen by most rows
  place_of(a, a.tiles, &bk, &tile);
  const int b = uniform(a.by_kv.of(bk)), kv = bk - b * a.KV;
  const Sight sight(a, b);
  const int j0 = tile * Sh::kKeys, jw = j0 + own * 32;
  const int key = jw + (lane & 31);
  const bool there = key < a.S, seen = key < sight.len;
  const T* krow = static_cast<const T*>(a.k) + b * a.pk.b + kv * a.pk.head + key * a.pk.t;
  const T* vbase = static_cast<const T*>(a.v) + b * a.pv.b + kv * a.pv.head;
  const T* vrow = vbase + key * a.pv.t;

  // The tokens that may see one of these keys.
  int ta = sight.first(0), tb = sight.last(a.T - 1);
  const int j1 = min(j0 + Sh::kKeys, sight.len) - 1;
  if (sight.causal) {
    ta = max(ta, j0 - sight.start);
    if (sight.window) tb = min(tb, j1 + sight.window - 1 - sight.start);
  }
  if (j0 > j1) tb = ta - 1;
  ta = uniform(ta);
  tb = uniform(tb);
  const RowTiles tiles(a, kRows);
  const bool grouped = a.rep <= kRows;
  const int n = tb < ta ? 0
      : uniform((int)((unsigned)(tb - ta + tiles.tokens) / (unsigned)tiles.tokens)) * tiles.chunks;

  const T* qbase = static_cast<const T*>(a.q) + b * a.pq.b + (int64_t)kv * a.rep * a.pq.head;
  const T* dbase = static_cast<const T*>(a.dout) + b * a.pdo.b + (int64_t)kv * a.rep * a.pdo.head;
  const uint32_t lds_base = lds_addr(lds_dyn);
  constexpr int kValuesAt = kStages * Sh::kStage;
  if (Sh::kTwo && n > 0) {
    Loader<T, kD, Sh::kKeys, kWaves> vload;
    const int stride = (int)(a.pv.t * sizeof(T));
    vload.init(stride, a.h, w, lane);
    vload.rows(vbase + j0 * a.pv.t, stride, sight.len - j0, a.h, lds_base + kValuesAt, w);
  }
  Loader<T, kD, kRows, kWaves> qload, dload;
  int unit[Loader<T, kD, kRows, kWaves>::kCount];  // a row's token (or head) in the tile
#pragma unroll
  for (int j = 0; j < qload.kCount; ++j) {
    const int r = qload.row(j, w, lane), c = qload.chunk(j, a.h, w, lane);
    const int t = grouped ? a.by_rep.of(r) : 0, g = r - t * a.rep;
    unit[j] = grouped ? t : g;
    const bool on = c != kOutOfRange && t < tiles.tokens;
    qload.voff[j] = on ? (int)((t * a.pq.t + g * a.pq.head) * sizeof(T)) + c : kOutOfRange;
    dload.voff[j] = on ? (int)((t * a.pdo.t + g * a.pdo.head) * sizeof(T)) + c : kOutOfRange;
  }
  const int64_t stat0 = (int64_t)bk * a.rows;
  // Tile (t, c): tokens from t on (heads from c kRows on).  Rows past the last are zeros in
  // all of their operands, and so is what comes of them.
  auto fetch = [&](int t, int c, int stage) __attribute__((always_inline)) {
    const uint32_t at = lds_base + stage * Sh::kStage;
    const int left = grouped ? tb - t + 1 : a.rep - c * kRows;  // tokens, or heads
    const int full = grouped ? tiles.tokens : kRows;
    const u32x4_t qb = wave_buffer(qbase + t * a.pq.t + c * kRows * a.pq.head, kBufferBytes),
                  db = wave_buffer(dbase + t * a.pdo.t + c * kRows * a.pdo.head, kBufferBytes);
#pragma unroll
    for (int j = 0; j < qload.kCount; ++j) {
      const uint32_t to = uniform(at + (w + kWaves * j) * 1024);
      const bool on = unit[j] < left;
      dma16(qb, to, on ? qload.voff[j] : kOutOfRange, 0);
      dma16(db, to + kBytes, on ? dload.voff[j] : kOutOfRange, 0);
    }
    // (One transfer a wave, so that all of them count the same.)
#pragma unroll
    for (int x = 0; x < (kWaves == 1 ? 3 : 1); ++x) {
      const int which = kWaves == 1 ? x : w;
      const bool some = which < (sizeof(T) == 4 ? 3 : 2);
      const float* from = (which == 0 ? a.lse : which == 1 ? a.delta : a.inv);
      const int count = some ? min(left, full) * (grouped ? a.rep : 1) : 0;
      dma4(wave_buffer(some ? from + stat0 + t * a.rep + c * kRows : a.lse, count * 4),
           uniform(at + 2 * kBytes + min(which, 3) * 256), lane * 4, 0);
    }
  };
  constexpr int kCount = 2 * decltype(qload)::kCount + (kWaves == 1 ? 3 : 1);
  int ft = ta, fc = 0, t = ta, c = 0;  // the tile that is fetched next, and the current one
  auto next = [&](int* t, int* c) __attribute__((always_inline)) {
    if (++*c >= tiles.chunks) {
      *c = 0;
      *t += tiles.tokens;
    }
  };
  // (Past the last tile: that again.)
  auto fetch_next = [&](int stage) __attribute__((always_inline)) {
    fetch(ft, fc, stage);
    if (ft + tiles.tokens <= tb || fc + 1 < tiles.chunks) next(&ft, &fc);
  };
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < kNext; ++i) fetch_next(i);
  }
  RowFrags<T, kD> k, v;
  if constexpr (Sh::kHoldK) load_row<T, kD>(k, krow, seen, a.h, lane);
  if constexpr (Sh::kHoldV) load_row<T, kD>(v, vrow, seen, a.h, lane);
  f32x16_t dk[X::kBlocks] = {}, dv[X::kBlocks] = {};
  Walk<(sizeof(T) == 2 ? kD : 64)> walk;
  if constexpr (sizeof(T) == 2) walk.init(lane, group * 32);
  const int stat_at = (int)lds_base + 16 * (lane >> 5) + 128 * group;
  const int values_at = uniform(kValuesAt + (own - group) * 32 * X::kRow);  // (walk: group's)

  // A tile in three: the two products, probabilities and ds, and their products.
  f32x16_t s[kParts], dp[kParts];
  u32x4_t p[4 * kParts];
  auto quad = [&](int which, int stage, int e, int x) __attribute__((always_inline)) {
    return lds_read<f32x4_t>(stat_at + (stage * Sh::kStage + 2 * kBytes + which * 256 +
                                        (32 * e + 8 * x) * 4));
  };
  auto front = [&](int stage) __attribute__((always_inline)) {
    const int qt = stage * Sh::kStage, dt = qt + kBytes;
    if constexpr (sizeof(T) == 2) {
      // Fragment u: of each block of 32 rows the queries' rows, then the output gradients'
      // (and the values' before each, if they are not held).
      constexpr int kEach = (Sh::kHoldV ? 2 : 3) * X::kPairs, kAll = kParts * kEach;
      const int q0 = walk.first_row(), d0 = walk.first_row(), v0 = walk.first_row() + values_at;
      u32x4_t ring[kAheadKeys];
      auto read = [&](int u) __attribute__((always_inline)) {
        if (u >= kAll) return;
        const int e = u / kEach, x = u % kEach, y = x - X::kPairs;
        if (x < X::kPairs)
          ring[u % kAheadKeys] = walk.row_from(q0, qt, e, x);
        else if (Sh::kHoldV)
          ring[u % kAheadKeys] = walk.row_from(d0, dt, e, y);
        else
          ring[u % kAheadKeys] = y & 1 ? walk.row_from(d0, dt, e, y >> 1)
                                       : walk.row_from(v0, 0, 0, y >> 1);
      };
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAheadKeys; ++u) read(u);
#pragma unroll
      for (int e = 0; e < kParts; ++e) {
        // The output gradients' product starts at -D.
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const f32x4_t d = quad(1, stage, e, x >> 2);
          dp[e][x] = d[x & 3];
        }
        s[e] = f32x16_t{};
        DPC_WALL();
#pragma unroll
        for (int x = 0; x < X::kPairs; ++x) {
          const int u = e * kEach + x;
          s[e] = mma_bf16(ring[u % kAheadKeys], k.v[x], s[e]);
          read(u + kAheadKeys);
          DPC_WALL();
        }
#pragma unroll
        for (int x = 0; x < X::kPairs; ++x) {
          if constexpr (Sh::kHoldV) {
            const int u = e * kEach + X::kPairs + x;
            dp[e] = mma_bf16(ring[u % kAheadKeys], v.v[x], dp[e]);
            read(u + kAheadKeys);
          } else {
            const int u = e * kEach + X::kPairs + 2 * x;
            dp[e] = mma_bf16(ring[(u + 1) % kAheadKeys], ring[u % kAheadKeys], dp[e]);
            read(u + kAheadKeys);
            read(u + 1 + kAheadKeys);
          }
          DPC_WALL();
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < kParts; ++e) {
        if constexpr (!Sh::kHoldK) load_row<T, kD>(k, krow, seen, a.h, lane);
        s[e] = times_rows<kD>(qt, 32 * e, k, lane);
        if constexpr (!Sh::kHoldK) load_row<T, kD>(v, vrow, seen, a.h, lane);
        dp[e] = times_rows<kD>(dt, 32 * e, v, lane);
      }
    }
  };
  // Of the tile of tokens ti .. tj.
  auto middle = [&](int ti, int tj, int stage) __attribute__((always_inline)) {
    const bool whole = jw >= sight.lo(tj) && jw + kRowsWave - 1 <= sight.hi(ti);
#pragma unroll
    for (int e = 0; e < kParts; ++e) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        s[e][x] = __builtin_amdgcn_exp2f(fmaf(s[e][x], a.c, -quad(0, stage, e, x >> 2)[x & 3]));
        if (sizeof(T) == 4) {
          s[e][x] *= quad(2, stage, e, x >> 2)[x & 3];
          dp[e][x] += quad(1, stage, e, x >> 2)[x & 3];
        }
        dp[e][x] *= s[e][x];
      }
      // Rows that do not see the key: zero, and then so is ds; it is zero too where a row sees one
      // key alone (never in a whole tile), whatever the rounding of dp - D left, if it is finite.
      if (!whole) {
        int r0 = 32 * (e + group) + column_row(0, lane);
        asm volatile("" : "+v"(r0));  // (its rows' tokens are not kept between tiles)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int at = ti + (grouped ? a.by_rep.of(r0 + column_row(x, 0)) : 0);
          const int lo = sight.lo(at), hi = sight.hi(at);
          if (key < lo || key > hi) s[e][x] = 0.f;
          if (key < lo || key > hi || (lo == hi && fabsf(dp[e][x]) < INFINITY)) dp[e][x] = 0.f;
        }
      }
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          p[4 * e + x] = packed_half(s[e], x);
          p[4 * e + 2 + x] = packed_half(dp[e], x);
        }
      }
    }
  };
  auto back = [&](int stage) __attribute__((always_inline)) {
    const int qt = stage * Sh::kStage, dt = qt + kBytes;
    if constexpr (sizeof(T) == 2) {
      // Fragment u: of each block the output gradients' columns, then the queries'.
      constexpr int kHalf = 2 * X::kBlocks, kAll = 2 * kParts * kHalf;
      const auto at = walk.cols();
      u32x4_t ring[kAheadKeys];
      auto read = [&](int u) __attribute__((always_inline)) {
        const int e = u / (2 * kHalf), x = u % (2 * kHalf);
        if (u < kAll)
          ring[u % kAheadKeys] = walk.col(at, x < kHalf ? dt : qt, e, x / X::kBlocks % 2, x % X::kBlocks);
      };
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAheadKeys; ++u) read(u);
      DPC_WALL();
#pragma unroll
      for (int u = 0; u < kAll; ++u) {
        const int d = u % X::kBlocks;
        if (u % (2 * kHalf) < kHalf)
          dv[d] = mma_bf16(ring[u % kAheadKeys], p[u / X::kBlocks], dv[d]);
        else
          dk[d] = mma_bf16(ring[u % kAheadKeys], p[u / X::kBlocks], dk[d]);
        read(u + kAheadKeys);
        DPC_WALL();
      }
    } else {
#pragma unroll
      for (int e = 0; e < kParts; ++e) {
        add_columns<kD>(dv, dt, 32 * e, s[e], lane);
        add_columns<kD>(dk, qt, 32 * e, dp[e], lane);
      }
    }
  };
  const bool late = Sh::kLate && group > 0;  // as in the forward
  bool pending = false;
  int pi = 0, pj = 0;  // the tokens of the tile that is not through
  auto step = [&](int i, int stage) __attribute__((always_inline)) {
    transfers_left<(kNext - 1) * kCount>();
    __syncthreads();
    const int before = (stage + kStages - 1) % kStages;
    const int ti = t, tj = min(tb, t + tiles.tokens - 1);
    next(&t, &c);
    const bool now = !(jw > sight.hi(tj) || jw + kRowsWave <= sight.lo(ti) || jw >= sight.len);
    if (late || !Sh::kLate) fetch_next((stage + kNext) % kStages);
    if (Sh::kLate && pending) {
      if (late) middle(pi, pj, before);
      back(before);
    }
    if (now) front(stage);
    if (Sh::kLate && !late) fetch_next((stage + kNext) % kStages);
    if (now && !late) middle(ti, tj, stage);
    if (now && !Sh::kLate) back(stage);
    pending = now;
    pi = ti;
    pj = tj;
  };
  for (int i = 0; i < n; i += kStages) {
#pragma unroll
    for (int x = 0; x < kStages; ++x)
      if (x == 0 || i + x < n) step(i + x, x);
  }
  if (Sh::kLate && pending) {
    const int stage = uniform((n - 1) % kStages);
#pragma unroll
    for (int x = 0; x < kStages; ++x)
      if (x == stage) {
        if (late) middle(pi, pj, x);
        back(x);
      }
  }
  transfers_left<0>();
  const int64_t flat = (((int64_t)b * a.S + key) * a.KV + kv) * a.h;
  if constexpr (Sh::kTwo) {
    // The first wave of two gives its dv away and adds the other's dk to its own.
    __syncthreads();
    constexpr int kWords = X::kBlocks * 16;
    static_assert(kWaves * kWords * 256 <= Sh::kLds, "LDS holds what is exchanged");
    float* to = reinterpret_cast<float*>(lds_dyn) + w * kWords * 64 + lane;
    const float* from = reinterpret_cast<const float*>(lds_dyn) + (w ^ 4) * kWords * 64 + lane;
#pragma unroll
    for (int d = 0; d < X::kBlocks; ++d)
#pragma unroll
      for (int x = 0; x < 16; ++x) to[(d * 16 + x) * 64] = group ? dk[d][x] : dv[d][x];
    __syncthreads();
#pragma unroll
    for (int d = 0; d < X::kBlocks; ++d)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float other = from[(d * 16 + x) * 64];
        dk[d][x] = group ? other + dv[d][x] : dk[d][x] + other;
      }
    store_row<T, kD>(static_cast<T*>(group ? a.dv : a.dk) + flat, nullptr, dk,
                     group ? 1.f : a.scale, seen, there, a.h, lane);
  } else {
    store_row<T, kD>(static_cast<T*>(a.dk) + flat, nullptr, dk, a.scale, seen, there, a.h, lane);
    store_row<T, kD>(static_cast<T*>(a.dv) + flat, nullptr, dv, 1.f, seen, there, a.h, lane);
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

constexpr int kUnits = 256;

Divisor divisor(int d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  return Divisor{(uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s, d};
}

// Key heads of an XCD, and as many of them at a time as make four rounds of its 32 units.
void spread(AttnArgs& a, int tiles) {
  const int heads = a.B * a.KV;
  a.per_xcd = heads % 8 ? 0 : heads / 8;
  const int most = a.per_xcd ? a.per_xcd : heads, want = (a.per_xcd ? 128 : 1024) / tiles + 1;
  a.chunk = want < most ? want : most;
}

template <typename T, int kD>
struct Launch {
  static constexpr int kSplitWaves = SplitShape<T, kD>::kWaves;

  template <typename K>
  static int go(K kernel, AttnArgs& a, int64_t grid, int threads, int lds, hipStream_t s) {
    if (lds > 65536)
      DPC_HIP_CHECK(hipFuncSetAttribute((const void*)kernel,
                                        hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    // A launch has fewer than 2^32 threads; whole rounds of the XCDs keep place_of's heads there.
    const int64_t most = UINT32_MAX / threads / 8 * 8;
    for (int64_t at = 0; at < grid; at += most) {
      a.block0 = (int)at;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(grid - at < most ? grid - at : most)),
                         dim3(threads), lds, s, a);
      DPC_HIP_CHECK(hipGetLastError());
    }
    return DPC_OK;
  }
  static int64_t heads(const AttnArgs& a) { return (int64_t)a.B * a.KV; }

  template <int kWaves>
  static int forward_rows(AttnArgs& a, hipStream_t s) {
    a.tiles = (a.rows + 32 * kWaves - 1) / (32 * kWaves);
    spread(a, a.tiles);
    return go(attn_forward_kernel<T, kD, kWaves, false>, a, heads(a) * a.tiles, 64 * kWaves,
              RowsShape<T, kD, kWaves>::kLds, s);
  }
  static int forward(AttnArgs& a, hipStream_t s) {
    if (a.splits == 0)
      return fills(a, a.rows, kMostWaves<T, kD>) ? forward_rows<kMostWaves<T, kD>>(a, s)
                                                 : forward_rows<4>(a, s);
    a.tiles = (a.rows + kRowsWave - 1) / kRowsWave;
    const int rc = go(attn_forward_kernel<T, kD, kSplitWaves, true>, a,
                      heads(a) * a.tiles * a.splits, 64 * kSplitWaves, SplitShape<T, kD>::kLds, s);
    if (rc) return rc;
    const int64_t rows = heads(a) * a.rows;
    hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a,
                       a.splits * kSplitWaves);
    DPC_HIP_CHECK(hipGetLastError());
    return DPC_OK;
  }

  template <int kWaves>
  static int dq(AttnArgs& a, hipStream_t s) {
    a.tiles = (a.rows + 32 * kWaves - 1) / (32 * kWaves);
    spread(a, a.tiles);
    return go(attn_dq_kernel<T, kD, kWaves>, a, heads(a) * a.tiles, 64 * kWaves,
              RowsShape<T, kD, kWaves>::kLds, s);
  }
  template <int kWaves>
  static int dkv(AttnArgs& a, hipStream_t s) {
    constexpr int kKeys = KeysShape<T, kD, kWaves>::kKeys;
    a.tiles = (a.S + kKeys - 1) / kKeys;
    spread(a, a.tiles);
    return go(attn_dkv_kernel<T, kD, kWaves>, a, heads(a) * a.tiles, 64 * kWaves,
              KeysShape<T, kD, kWaves>::kLds, s);
  }
  // The widest tiles that give every compute unit one; else the narrowest (dq: 128 rows between
  // the two).  bf16, h = 128, us of 256 / 128 / 32 rows: dq of 1 x 1024 tokens of 8 heads 40 / 33 /
  // 32, of 4 x 1024 46 / 36 / 41; the forward of 4 x 1024 33 / 31.  dk and dv, 128 / 32 keys:
  // 4 x 1024 39 / 58.  Below a tile a unit 32 keys win where few rows see a key (9 x 443, 6 heads of
  // 80 over 2, a window of 200: 49 / 42), and lose without a window (1 x 1024 of 8 heads: 37 / 45,
  // of 32 over 8: 116 / 153).
  static bool fills(const AttnArgs& a, int64_t n, int waves) {
    return heads(a) * ((n + 32 * waves - 1) / (32 * waves)) >= kUnits;
  }
  static int backward(AttnArgs& a, hipStream_t s) {
    if (a.rows > 0) {
      constexpr int kMost = kMostWaves<T, kD>;
      const int rc = fills(a, a.rows, kMost) ? dq<kMost>(a, s)
                     : fills(a, a.rows, 4)   ? dq<4>(a, s)
                                             : dq<1>(a, s);
      if (rc) return rc;
    }
    if (a.S > 0 && a.dk) return fills(a, a.S, 4) ? dkv<kMostWaves<T, kD>>(a, s) : dkv<1>(a, s);
    return DPC_OK;
  }
};

template <typename F>
int by_width(int dtype, int h, F f) {
  if (dtype == DPC_BF16) {
    if (h <= 64) return f(Launch<uint16_t, 64>());
    if (h <= 128) return f(Launch<uint16_t, 128>());
    return f(Launch<uint16_t, 256>());
  }
  if (h <= 64) return f(Launch<float, 64>());
  if (h <= 128) return f(Launch<float, 128>());
  return f(Launch<float, 256>());
}

int split_waves(int dtype, int h) {
  return by_width(dtype, h, [](auto l) { return decltype(l)::kSplitWaves; });
}

constexpr int64_t kMostTokens = 1ll << 24;

bool valid_sizes(int64_t B, int64_t T, int64_t S, int H, int KV, int h, int dtype) {
  if (B < 0 || T < 0 || S < 0 || T > kMostTokens || S > kMostTokens || H < 1 || KV < 1 || H % KV ||
      H > (1 << 16) || h < 1 || h > 256 || (dtype != DPC_F32 && dtype != DPC_BF16))
    return false;
  if (h % (dtype == DPC_F32 ? 4 : 8)) return false;
  if (B > (1ll << 30)) return false;
  // Workgroups of a launch, by rows, by keys, and by rows in splits.
  const int64_t most = INT32_MAX, rows = T * (H / KV);
  if (rows > 1 << 30) return false;
  return B * KV <= most / ((rows + 31) / 32 + 1) && B * KV <= most / ((S + 31) / 32 + 1);
}

// Splits of the keys (0: none).  Where tiles of 256 rows leave compute units idle, either of
// two is taken that costs less: tiles of 128 rows (6 us and 1.1 a round's 64 keys), or rows by
// 32 with their keys in splits, which are joined (12 us and 1.2 for 32 keys of 32 rows, four
// waves a unit): then enough splits for four workgroups a unit, none with fewer than four tiles of
// 32 keys a wave.  (9 x 443 tokens, 6 heads over 2: 18 us in 198 tiles, 29 in splits.  16
// tokens of 32 heads over 8, 8192 keys at most: 228 us in tiles, 64 in 8 splits.)  The prices are
// bf16's at h = 128, and S is counted whatever a window or the lengths leave of it.
int splits_of(int64_t B, int64_t T, int64_t S, int H, int KV, int h, int dtype) {
  const int64_t rows = T * (H / KV), heads = B * KV;
  if (heads * ((rows + 255) / 256) >= kUnits) return 0;
  const int64_t groups = heads * ((rows + 31) / 32);
  const int64_t rounds = (heads * ((rows + 127) / 128) + kUnits - 1) / kUnits;
  const double tiled = 6.0 + 1.1 * (double)(rounds * S) / 64,
               split = 12.0 + 1.2 * (double)(groups * S) / (32.0 * 4 * kUnits);
  if (tiled <= split) return 0;
  int64_t n = (4 * kUnits + groups - 1) / groups;
  const int64_t most = S / (32 * 4 * split_waves(dtype, h));
  if (n > most) n = most;
  return n < 1 ? 1 : (n > 64 ? 64 : (int)n);
}

}  // namespace

namespace {

// `rows`: of keys and values, of which more than one may not overlap.
int tensor_places(const int64_t* s, int bytes, int rep, int64_t rows, int h, Places* p) {
  *p = Places{s[0], s[1], s[2]};
  if (rows > 1 && s[1] < h) return DPC_ENOTSUP;
  const int64_t most = (int64_t)kOutOfRange - (1 << 20);
  if (s[1] < 0 || s[2] < 0 || s[1] > most || s[2] > most) return DPC_ENOTSUP;
  // A tile's 64 rows (of shared key heads: 65 tokens at most) in one buffer.
  if ((65 * s[1] + rep * s[2]) * bytes > most) return DPC_ENOTSUP;
  return (s[0] * bytes | s[1] * bytes | s[2] * bytes) & 15 ? DPC_EINVAL : DPC_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

void keep_in(AttnArgs& a, void* state, int64_t n, int dtype) {
  if (!state) return;
  a.lse = static_cast<float*>(state);
  uint8_t* second = static_cast<uint8_t*>(state) + up256(n * 4);
  if (dtype == DPC_F32)
    a.inv = reinterpret_cast<float*>(second);
  else
    a.rest = reinterpret_cast<int8_t*>(second);
}

}  // namespace

extern "C" size_t dpc_attention_state_bytes(int64_t B, int64_t T, int H, int h, int dtype) {
  if (B <= 0 || T <= 0 || H <= 0 || h <= 0) return 0;
  const size_t n = (size_t)(B * T * H);
  return up256(n * 4) + n * (dtype == DPC_F32 ? 4 : h);
}

extern "C" size_t dpc_attention_workspace_bytes(int64_t B, int64_t T, int64_t S, int H, int KV,
                                                int h, int dtype) {
  if (!valid_sizes(B, T, S, H, KV, h, dtype) || B == 0 || T == 0) return 0;
  const int64_t parts = (int64_t)splits_of(B, T, S, H, KV, h, dtype) * split_waves(dtype, h);
  return (size_t)(parts * B * T * H * (h * 4 + 8));
}

extern "C" int dpc_attention(const void* q, const void* k, const void* v, const int64_t* strides,
                             int64_t B, int64_t T, int64_t S, int H, int KV, int h, int dtype,
                             const int64_t* lengths, const int64_t* starts, int causal, int window,
                             double scale, void* out, void* state, size_t state_bytes, void* ws,
                             size_t ws_bytes, void* stream) {
  if (!valid_sizes(B, T, S, H, KV, h, dtype) || !strides || window < 0 || (window && !causal) ||
      !((float)scale > 0.f) || !isfinite((float)scale))
    return DPC_EINVAL;
  if (B == 0 || T == 0) return DPC_OK;
  if (!q || !out || (S && (!k || !v)) || !aligned16(q) || !aligned16(k) || !aligned16(v) ||
      !aligned16(out))
    return DPC_EINVAL;
  AttnArgs a = {};
  const int bytes = dtype == DPC_F32 ? 4 : 2;
  a.rep = H / KV;
  if (const int rc = tensor_places(strides, bytes, a.rep, 0, h, &a.pq)) return rc;
  if (const int rc = tensor_places(strides + 3, bytes, 1, S, h, &a.pk)) return rc;
  if (const int rc = tensor_places(strides + 6, bytes, 1, S, h, &a.pv)) return rc;
  const size_t need = dpc_attention_workspace_bytes(B, T, S, H, KV, h, dtype);
  if (ws_bytes < need ||
      (state && state_bytes < dpc_attention_state_bytes(B, T, H, h, dtype)))
    return DPC_ENOSPC;
  if ((need && (!ws || ((uintptr_t)ws & 255))) || ((uintptr_t)state & 255)) return DPC_EINVAL;
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = out;
  keep_in(a, state, B * T * H, dtype);
  a.B = (int)B;
  a.T = (int)T;
  a.S = (int)S;
  a.KV = KV;
  a.h = h;
  a.rows = (int)(T * a.rep);
  a.by_rep = divisor(a.rep);
  a.by_kv = divisor(KV);
  a.lengths = lengths;
  a.starts = starts;
  a.causal = causal != 0;
  a.window = window < kMostTokens ? window : (int)kMostTokens;
  a.scale = (float)scale;
  a.c = (float)(scale * 1.44269504088896340736);
  a.splits = splits_of(B, T, S, H, KV, h, dtype);
  const int64_t parts = (int64_t)a.splits * split_waves(dtype, h);
  a.part_o = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + parts * B * T * H * h);
  hipStream_t s = (hipStream_t)stream;
  return by_width(dtype, h, [&](auto l) { return decltype(l)::forward(a, s); });
}

extern "C" size_t dpc_attention_grad_workspace_bytes(int64_t B, int64_t T, int H) {
  return B > 0 && T > 0 && H > 0 ? (size_t)(B * T * H * 4) : 0;
}

extern "C" int dpc_attention_grad(const void* q, const void* k, const void* v, const void* out,
                                  const void* dout, const int64_t* strides, int64_t B, int64_t T,
                                  int64_t S, int H, int KV, int h, int dtype,
                                  const int64_t* lengths, const int64_t* starts, int causal,
                                  int window, double scale, const void* state, size_t state_bytes,
                                  void* dq, void* dk, void* dv, void* ws, size_t ws_bytes,
                                  void* stream) {
  if (!valid_sizes(B, T, S, H, KV, h, dtype) || !strides || window < 0 || (window && !causal) ||
      !((float)scale > 0.f) || !isfinite((float)scale))
    return DPC_EINVAL;
  if (B == 0 || (T == 0 && S == 0)) return DPC_OK;
  if ((T && (!q || !out || !dout || !state || !dq)) || (S && (!k || !v)) || (!dk != !dv) ||
      !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(dout) ||
      !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return DPC_EINVAL;
  AttnArgs a = {};
  const int bytes = dtype == DPC_F32 ? 4 : 2;
  a.rep = H / KV;
  if (const int rc = tensor_places(strides, bytes, a.rep, 0, h, &a.pq)) return rc;
  if (const int rc = tensor_places(strides + 3, bytes, 1, S, h, &a.pk)) return rc;
  if (const int rc = tensor_places(strides + 6, bytes, 1, S, h, &a.pv)) return rc;
  if (const int rc = tensor_places(strides + 9, bytes, a.rep, 0, h, &a.pdo)) return rc;
  const size_t need = dpc_attention_grad_workspace_bytes(B, T, H);
  if (ws_bytes < need || state_bytes < dpc_attention_state_bytes(B, T, H, h, dtype))
    return DPC_ENOSPC;
  if ((need && (!ws || ((uintptr_t)ws & 255))) || ((uintptr_t)state & 255)) return DPC_EINVAL;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.dout = dout;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  keep_in(a, const_cast<void*>(state), B * T * H, dtype);
  a.delta = static_cast<float*>(ws);
  a.B = (int)B;
  a.T = (int)T;
  a.S = (int)S;
  a.KV = KV;
  a.h = h;
  a.rows = (int)(T * a.rep);
  a.by_rep = divisor(a.rep);
  a.by_kv = divisor(KV);
  a.lengths = lengths;
  a.starts = starts;
  a.causal = causal != 0;
  a.window = window < kMostTokens ? window : (int)kMostTokens;
  a.scale = (float)scale;
  a.c = (float)(scale * 1.44269504088896340736);
  hipStream_t s = (hipStream_t)stream;
  return by_width(dtype, h, [&](auto l) { return decltype(l)::backward(a, s); });
}
