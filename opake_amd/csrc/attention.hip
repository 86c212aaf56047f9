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

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kOutOfRange = 0x7ff00000;  // a byte offset past every buffer
constexpr int kBufferBytes = 0x7ff00000;
constexpr int kRowsWave = 32;

extern __shared__ __attribute__((aligned(16))) uint8_t lds_dyn[];

// A buffer at an address that is the wave's, of which the compiler may not know that.
DPC_DEVICE u32x4_t wave_buffer(const void* base, uint32_t bytes) {
  u32x4_t r = rsrc_words(base, bytes);
  r[0] = __builtin_amdgcn_readfirstlane(r[0]);
  r[1] = __builtin_amdgcn_readfirstlane(r[1]);
  r[2] = __builtin_amdgcn_readfirstlane(r[2]);
  return r;
}

// The wave's transfers into LDS have arrived and its reads of LDS are done (their place may
// be written again); no access moves across.
DPC_DEVICE void transfers_done() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

struct Places {  // of one tensor: elements between examples, tokens and heads
  int64_t b, t;
  int64_t head;
};

struct AttnArgs {
  const void *q, *k, *v, *out, *dout;
  Places pq, pk, pv, pdo;  // out, lse and the gradients are contiguous
  void *o, *dq, *dk, *dv;
  float *lse, *delta;      // [B, KV, rows]
  int B, T, S, KV, rep, h;
  int64_t rows;            // of a key head: T * rep
  const int64_t *lengths, *starts;
  int causal, window;
  float scale, c;          // c = scale log2(e)
  int tiles;               // row tiles (dk, dv: key tiles) of a key head
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
    len = __builtin_amdgcn_readfirstlane((int)n);
    int64_t s = a.starts ? a.starts[b] : (int64_t)a.S - a.T;
    const int64_t most = 1 << 30;
    s = s < -most ? -most : (s < most ? s : most);
    start = __builtin_amdgcn_readfirstlane((int)s);
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

// Linear id -> (key head of the batch, tile): each XCD takes a contiguous range, so that
// the tiles of a key head read its operands from one L2.
DPC_DEVICE void place_of(int id, int n, int tiles, int* bk, int* tile) {
  const int xcd = id & 7;
  const int lin = xcd * (n >> 3) + min(xcd, n & 7) + (id >> 3);
  *bk = __builtin_amdgcn_readfirstlane(lin / tiles);
  *tile = __builtin_amdgcn_readfirstlane(lin % tiles);
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

// The two products' operands of a lane: column (or row) lane % 32, the chunks 2 i + lane /
// 32 of it.
template <typename T, int kD>
struct RowFrags {
  u32x4_t v[Tile<T, kD>::kPairs];
};

DPC_DEVICE f32x16_t mma(u32x4_t a, u32x4_t b, f32x16_t c, uint16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
DPC_DEVICE f32x16_t mma(u32x4_t a, u32x4_t b, f32x16_t c, float) {
  const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
  return c;
}

// 32 rows of an LDS tile times a lane's column: c[r] is row 8 (r / 4) + 4 (lane / 32) + r % 4.
template <typename T, int kD>
DPC_DEVICE f32x16_t times_rows(const uint8_t* tile, int row0, const RowFrags<T, kD>& b, int lane) {
  typedef Tile<T, kD> X;
  const int row = row0 + (lane & 31), hl = lane >> 5;
  const uint8_t* at = tile + row * X::kRow;
  const int sw = swizzle<X::kChunks>(row) ^ hl;
  f32x16_t c = {};
#pragma unroll
  for (int i = 0; i < X::kPairs; ++i)
    c = mma(*reinterpret_cast<const u32x4_t*>(at + (((2 * i) ^ sw) << 4)), b.v[i], c, T());
  return c;
}

// acc[d] += sum over the tile's 32 rows from row0 of (element d of the row) x[row]: x in
// times_rows' order.
template <typename T, int kD>
DPC_DEVICE void add_columns(f32x16_t* acc, const uint8_t* tile, int row0, const f32x16_t& x,
                            int lane) {
  typedef Tile<T, kD> X;
  if constexpr (sizeof(T) == 2) {
    const int L = lane & 15, hl = lane >> 5;
    const int row = 4 * hl + (L >> 2), chunk = ((lane >> 4) & 1) * 2 + ((L & 3) >> 1);
    const int s0 = swizzle<X::kChunks>(row), s1 = swizzle<X::kChunks>(row + 8);
    const int at = (row0 + row) * X::kRow + (L & 1) * 8;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      u32x4_t b;
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = f32x2_to_bf16x2_bits(x[8 * j + 2 * e], x[8 * j + 2 * e + 1]);
#pragma unroll
      for (int d = 0; d < X::kBlocks; ++d) {
        const int o = at + j * 16 * X::kRow;
        const bf16x8_t a =
            join_frag(read_tr(tile, o + (((4 * d + chunk) ^ s0) << 4)),
                      read_tr(tile, o + 8 * X::kRow + (((4 * d + chunk) ^ s1) << 4)));
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8_t, b),
                                                         acc[d], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = row0 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
      const int sw = swizzle<X::kChunks>(row);
#pragma unroll
      for (int d = 0; d < X::kBlocks; ++d) {
        const int col = 32 * d + (lane & 31);
        const float a = *reinterpret_cast<const float*>(
            tile + row * X::kRow + (((col >> 2) ^ sw) << 4) + (col & 3) * 4);
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x[r], acc[d], 0, 0, 0);
      }
    }
  }
}

// Transfers of a tile of kRows rows by kWaves waves.
template <typename T, int kD, int kRows, int kWaves>
struct Loader {
  typedef Tile<T, kD> X;
  static constexpr int kCount = kRows * X::kChunks / (64 * kWaves);
  static_assert(kCount * 64 * kWaves == kRows * X::kChunks, "whole transfers");
  int chunk[kCount];  // byte offset in the row; out of range past the head's elements
  int row0;           // of the lane's first
  static constexpr int kRowStep = 64 * kWaves / X::kChunks;
  static_assert(64 * kWaves % X::kChunks == 0 || X::kChunks % (64 * kWaves) == 0, "");

  DPC_DEVICE void init(int h, int w, int lane) {
    row0 = (w * 64 + lane) / X::kChunks;
#pragma unroll
    for (int j = 0; j < kCount; ++j) {
      const int c = ((w * 64 + lane) & (X::kChunks - 1)) ^ swizzle<X::kChunks>(row(j));
      chunk[j] = c * X::kEach < h ? c * 16 : kOutOfRange;
    }
  }
  DPC_DEVICE int row(int j) const { return row0 + j * kRowStep; }
  // Rows `stride` bytes apart; rows from `limit` on are zeros.
  DPC_DEVICE void rows(const void* base, int stride, int limit, uint32_t lds, int w) const {
    const u32x4_t buf = wave_buffer(base, kBufferBytes);
#pragma unroll
    for (int j = 0; j < kCount; ++j) {
      const int off = row(j) < limit ? row(j) * stride + chunk[j] : kOutOfRange;
      dma16(buf, __builtin_amdgcn_readfirstlane(lds + (w + kWaves * j) * 1024), chunk[j] == kOutOfRange ? kOutOfRange : off, 0);
    }
  }
  // Rows of shared key heads: row r is token (g0 + r) / rep of `base`, head (g0 + r) % rep.
  DPC_DEVICE void shared(const void* base, int g0, int rep, float inv, int token, int head,
                         int limit, uint32_t lds, int w) const {
    const u32x4_t buf = wave_buffer(base, kBufferBytes);
#pragma unroll
    for (int j = 0; j < kCount; ++j) {
      const int r = g0 + row(j);
      int t = (int)((float)r * inv);  // (r < 2^20: off by one at most)
      t -= t * rep > r;
      t += (t + 1) * rep <= r;
      const int off = t * token + (r - t * rep) * head + chunk[j];
      dma16(buf, __builtin_amdgcn_readfirstlane(lds + (w + kWaves * j) * 1024),
            row(j) < limit && chunk[j] != kOutOfRange ? off : kOutOfRange, 0);
    }
  }
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

// Stores a lane's column (kD elements in times_rows' order, over kD / 32 blocks) times f
// as row `out`, or zeros where !keep.
template <typename T, int kD>
DPC_DEVICE void store_row(T* out, const f32x16_t* acc, float f, bool keep, bool on, int h,
                          int lane) {
#pragma unroll
  for (int d = 0; d < kD / 32; ++d) {
    if constexpr (sizeof(T) == 2) {
      // A pair of quads of both halves makes 8 elements a lane.
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = acc[d][8 * j + 2 * e] * f, y = acc[d][8 * j + 2 * e + 1] * f;
          p[e] = keep ? f32x2_to_bf16x2_bits(x, y) : 0u;
        }
        const auto lo = __builtin_amdgcn_permlane32_swap(p[0], p[2], false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap(p[1], p[3], false, false);
        const int at = 32 * d + 16 * j + 8 * (lane >> 5);
        if (on && at < h)
          *reinterpret_cast<u32x4_t*>(out + at) = u32x4_t{lo[0], hi[0], lo[1], hi[1]};
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

// A row tile's place: its rows, its tokens' keys, and the wave's own of both.
struct RowRange {
  int t_first, t_last;  // tokens that see a key (t_first > t_last: none)
  int lo, hi;           // keys that one of them sees
  int lo_all, hi_all;   // keys that all of them see
  DPC_DEVICE RowRange(const AttnArgs& a, const Sight& s, int64_t r0, int64_t r1) {
    t_first = s.first((int)(r0 / a.rep));
    t_last = r1 > r0 ? s.last((int)((r1 - 1) / a.rep)) : -1;
    if (t_first > t_last) {
      lo = lo_all = 0;
      hi = hi_all = -1;
      return;
    }
    lo = s.lo(t_first);
    hi = s.hi(t_last);
    lo_all = s.lo(t_last);
    hi_all = s.hi(t_first);
  }
  DPC_DEVICE bool none() const { return t_first > t_last; }
};

// ---------------------------------------------------------------------------
// Forward.
// ---------------------------------------------------------------------------

template <typename T, int kD>
struct ForwardShape {
  static constexpr int kRow = Tile<T, kD>::kRow;
  static constexpr int kKeys = kRow <= 512 ? 64 : 32;
  static constexpr int kWaves = 4;
  static constexpr int kLds = 4 * kKeys * kRow;  // two stages of keys and values
  // Keys in splits: a wave takes 32 keys at a time into LDS of its own.
  static constexpr int kSplitWaves = kRow <= 256 ? 4 : (kRow == 512 ? 2 : 1);
  static constexpr int kSplitLds = kSplitWaves * 4 * 32 * kRow;
};

template <typename T, int kD, bool kSplit>
__global__ void __launch_bounds__((kSplit ? 64 * ForwardShape<T, kD>::kSplitWaves : 256),
                                  (Tile<T, kD>::kRow <= 256 && !kSplit ? 2 : 1))
    attn_forward_kernel(AttnArgs a) {
  typedef Tile<T, kD> X;
  typedef ForwardShape<T, kD> Sh;
  constexpr int kKeys = kSplit ? 32 : Sh::kKeys, kWaves = kSplit ? Sh::kSplitWaves : Sh::kWaves;
  constexpr int kBytes = kKeys * X::kRow;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bk, tile, split = 0;
  {
    const int per = a.tiles * (kSplit ? a.splits : 1);
    place_of(blockIdx.x, a.B * a.KV * per, per, &bk, &tile);
    if (kSplit) {
      split = tile % a.splits * kWaves + w;
      tile /= a.splits;
    }
    tile = a.tiles - 1 - tile;  // the longest first
  }
  const int b = bk / a.KV, kv = bk - b * a.KV;
  const Sight sight(a, b);
  constexpr int kTileRows = kSplit ? kRowsWave : kRowsWave * kWaves;
  const int64_t t0 = (int64_t)tile * kTileRows, t1 = min(t0 + kTileRows, a.rows);
  const int64_t w0 = kSplit ? t0 : t0 + w * kRowsWave, w1 = min(w0 + kRowsWave, t1);
  const RowRange all(a, sight, t0, t1), mine(a, sight, w0, w1 > w0 ? w1 : w0);

  // The lane's row.
  const int64_t r = w0 + (lane & 31);
  const int t = (int)(min(r, a.rows - 1) / a.rep), g = (int)(r - (int64_t)t * a.rep);
  const bool there = r < a.rows, sees = there && t >= mine.t_first && t <= mine.t_last;
  const int lo = sees ? sight.lo(t) : 0, hi = sees ? sight.hi(t) : -1;
  RowFrags<T, kD> q;
  load_row<T, kD>(q, static_cast<const T*>(a.q) + b * a.pq.b + t * a.pq.t +
                         ((int64_t)kv * a.rep + g) * a.pq.head, sees, a.h, lane);

  const T* kbase = static_cast<const T*>(a.k) + b * a.pk.b + kv * a.pk.head;
  const T* vbase = static_cast<const T*>(a.v) + b * a.pv.b + kv * a.pv.head;
  const int kstride = (int)(a.pk.t * sizeof(T)), vstride = (int)(a.pv.t * sizeof(T));
  constexpr int kLoaders = kSplit ? 1 : kWaves;
  Loader<T, kD, kKeys, kLoaders> loader;
  const int lw = kSplit ? 0 : w;
  loader.init(a.h, lw, lane);
  uint8_t* lds = lds_dyn + (kSplit ? w * 4 * kBytes : 0);
  const uint32_t lds0 = lds_addr(lds);

  f32x16_t o[X::kBlocks] = {};
  float m = -INFINITY, l = 0.f;
  int n = all.none() ? 0 : all.hi / kKeys - all.lo / kKeys + 1, first = all.lo / kKeys;
  if (kSplit && n > 0) {  // this wave's share of the row tile's keys
    const int parts = a.splits * kWaves, s0 = (int)((int64_t)n * split / parts),
              s1 = (int)((int64_t)n * (split + 1) / parts);
    first += s0;
    n = s1 - s0;
  }
  const int limit = min(sight.len, all.hi + 1);
  auto fetch = [&](int i) __attribute__((always_inline)) {
    const int j0 = (first + i) * kKeys;
    const uint32_t at = lds0 + (i & 1) * 2 * kBytes;
    loader.rows(kbase + (int64_t)j0 * a.pk.t, kstride, limit - j0, at, lw);
    loader.rows(vbase + (int64_t)j0 * a.pv.t, vstride, limit - j0, at + kBytes, lw);
  };
  if (n > 0) fetch(0);
  for (int i = 0; i < n; ++i) {
    transfers_done();
    if (!kSplit) __syncthreads();
    if (i + 1 < n) fetch(i + 1);
    const int j0 = (first + i) * kKeys;
    if (mine.none() || j0 > mine.hi || j0 + kKeys <= mine.lo) continue;
    const bool whole = j0 >= mine.lo_all && j0 + kKeys - 1 <= mine.hi_all;
    const uint8_t* kt = lds + (i & 1) * 2 * kBytes;
    const uint8_t* vt = kt + kBytes;
    f32x16_t s[kKeys / 32];
#pragma unroll
    for (int e = 0; e < kKeys / 32; ++e) s[e] = times_rows<T, kD>(kt, 32 * e, q, lane);
    if (!whole) {
#pragma unroll
      for (int e = 0; e < kKeys / 32; ++e)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int j = j0 + 32 * e + 8 * (x >> 2) + 4 * (lane >> 5) + (x & 3);
          if (j < lo || j > hi) s[e][x] = -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int e = 0; e < kKeys / 32; ++e)
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
#pragma unroll
      for (int d = 0; d < X::kBlocks; ++d) o[d] *= f;
    }
    const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < kKeys / 32; ++e) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        s[e][x] = __builtin_amdgcn_exp2f(fmaf(s[e][x], a.c, -from));
        l += s[e][x];
      }
      add_columns<T, kD>(o, vt, 32 * e, s[e], lane);
    }
  }
  l = sum_halves(l);
  const int64_t row = (int64_t)bk * a.rows + r;
  if (kSplit) {
    const int64_t at = (int64_t)split * a.B * a.KV * a.rows + row;
    if (there && lane < 32) a.part_ml[at] = make_float2(sees ? m : -INFINITY, sees ? l : 0.f);
    store_row<float, kD>(a.part_o + at * a.h, o, 1.f, sees, there, a.h, lane);
    return;
  }
  const bool some = sees && l != 0.f;  // (NaN too)
  if (there && lane < 32 && a.lse) a.lse[row] = some ? m + __builtin_amdgcn_logf(l) : INFINITY;
  T* out = static_cast<T*>(a.o) +
           ((int64_t)(b * (int64_t)a.T + t) * a.KV * a.rep + (int64_t)kv * a.rep + g) * a.h;
  store_row<T, kD>(out, o, 1.f / l, some, there, a.h, lane);
}

// The splits of a row joined: one wave a row.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a, int parts) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)a.B * a.KV * a.rows;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  float m = -INFINITY;
  for (int p = 0; p < parts; ++p) m = fmaxf(m, a.part_ml[p * n + row].x);
  const float from = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[4] = {};
  for (int p = 0; p < parts; ++p) {
    const float2 x = a.part_ml[p * n + row];
    const float f = __builtin_amdgcn_exp2f(x.x - from);
    l += x.y * f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 64 * e < a.h) o[e] += a.part_o[(p * n + row) * a.h + lane + 64 * e] * f;
  }
  const bool some = l != 0.f;
  const int64_t bk = row / a.rows, r = row - bk * a.rows, b = bk / a.KV, kv = bk - b * a.KV,
                t = r / a.rep, g = r - t * a.rep;
  if (a.lse && lane == 0) a.lse[row] = some ? m + __builtin_amdgcn_logf(l) : INFINITY;
  T* out = static_cast<T*>(a.o) + ((b * a.T + t) * a.KV * a.rep + kv * a.rep + g) * a.h;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 64 * e < a.h) {
      const float x = some ? o[e] / l : 0.f;
      if constexpr (sizeof(T) == 2)
        out[lane + 64 * e] = f32_to_bf16_bits(x);
      else
        out[lane + 64 * e] = x;
    }
}

// ---------------------------------------------------------------------------
// dq and D: rows fixed, keys walked.
// ---------------------------------------------------------------------------

template <typename T, int kD>
__global__ void __launch_bounds__(256, (Tile<T, kD>::kRow <= 256 ? 2 : 1))
    attn_dq_kernel(AttnArgs a) {
  typedef Tile<T, kD> X;
  constexpr int kKeys = ForwardShape<T, kD>::kKeys, kWaves = 4, kBytes = kKeys * X::kRow;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bk, tile;
  place_of(blockIdx.x, a.B * a.KV * a.tiles, a.tiles, &bk, &tile);
  tile = a.tiles - 1 - tile;
  const int b = bk / a.KV, kv = bk - b * a.KV;
  const Sight sight(a, b);
  const int64_t t0 = (int64_t)tile * kRowsWave * kWaves,
                t1 = min(t0 + kRowsWave * kWaves, a.rows);
  const int64_t w0 = t0 + w * kRowsWave, w1 = min(w0 + kRowsWave, t1);
  const RowRange all(a, sight, t0, t1), mine(a, sight, w0, w1 > w0 ? w1 : w0);
  const int64_t r = w0 + (lane & 31);
  const int t = (int)(min(r, a.rows - 1) / a.rep), g = (int)(r - (int64_t)t * a.rep);
  const bool there = r < a.rows, sees = there && t >= mine.t_first && t <= mine.t_last;
  const int lo = sees ? sight.lo(t) : 0, hi = sees ? sight.hi(t) : -1;
  const int64_t head = (int64_t)kv * a.rep + g, row = (int64_t)bk * a.rows + r;
  const int64_t flat = ((int64_t)(b * (int64_t)a.T + t) * a.KV * a.rep + head) * a.h;
  RowFrags<T, kD> q, dout;
  load_row<T, kD>(q, static_cast<const T*>(a.q) + b * a.pq.b + t * a.pq.t + head * a.pq.head, sees,
                  a.h, lane);
  load_row<T, kD>(dout, static_cast<const T*>(a.dout) + b * a.pdo.b + t * a.pdo.t +
                            head * a.pdo.head, sees, a.h, lane);
  float D = 0.f;
#pragma unroll
  for (int i = 0; i < X::kPairs; ++i) {
    const int at = (2 * i + (lane >> 5)) * X::kEach;
    const u32x4_t x = sees && at < a.h
        ? *reinterpret_cast<const u32x4_t*>(static_cast<const T*>(a.out) + flat + at) : u32x4_t{};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 2) {
        D += bf16_bits_to_f32((uint16_t)x[e]) * bf16_bits_to_f32((uint16_t)dout.v[i][e]);
        D += bf16_bits_to_f32((uint16_t)(x[e] >> 16)) *
             bf16_bits_to_f32((uint16_t)(dout.v[i][e] >> 16));
      } else {
        D += __uint_as_float(x[e]) * __uint_as_float(dout.v[i][e]);
      }
    }
  }
  D = sum_halves(D);
  if (there && lane < 32) a.delta[row] = D;
  const float lse = sees ? a.lse[row] : INFINITY;

  const T* kbase = static_cast<const T*>(a.k) + b * a.pk.b + kv * a.pk.head;
  const T* vbase = static_cast<const T*>(a.v) + b * a.pv.b + kv * a.pv.head;
  const int kstride = (int)(a.pk.t * sizeof(T)), vstride = (int)(a.pv.t * sizeof(T));
  Loader<T, kD, kKeys, kWaves> loader;
  loader.init(a.h, w, lane);
  const uint32_t lds0 = lds_addr(lds_dyn);
  f32x16_t dq[X::kBlocks] = {};
  const int first = all.lo / kKeys, n = all.none() ? 0 : all.hi / kKeys - first + 1;
  const int limit = min(sight.len, all.hi + 1);
  auto fetch = [&](int i) __attribute__((always_inline)) {
    const int j0 = (first + i) * kKeys;
    const uint32_t at = lds0 + (i & 1) * 2 * kBytes;
    loader.rows(kbase + (int64_t)j0 * a.pk.t, kstride, limit - j0, at, w);
    loader.rows(vbase + (int64_t)j0 * a.pv.t, vstride, limit - j0, at + kBytes, w);
  };
  if (n > 0) fetch(0);
  for (int i = 0; i < n; ++i) {
    transfers_done();
    __syncthreads();
    if (i + 1 < n) fetch(i + 1);
    const int j0 = (first + i) * kKeys;
    if (mine.none() || j0 > mine.hi || j0 + kKeys <= mine.lo) continue;
    const bool whole = j0 >= mine.lo_all && j0 + kKeys - 1 <= mine.hi_all;
    const uint8_t* kt = lds_dyn + (i & 1) * 2 * kBytes;
    const uint8_t* vt = kt + kBytes;
#pragma unroll
    for (int e = 0; e < kKeys / 32; ++e) {
      f32x16_t s = times_rows<T, kD>(kt, 32 * e, q, lane);
      const f32x16_t dp = times_rows<T, kD>(vt, 32 * e, dout, lane);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[x], a.c, -lse));
        s[x] = p * (dp[x] - D);
      }
      if (!whole) {
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int j = j0 + 32 * e + 8 * (x >> 2) + 4 * (lane >> 5) + (x & 3);
          if (j < lo || j > hi) s[x] = 0.f;
        }
      }
      add_columns<T, kD>(dq, kt, 32 * e, s, lane);
    }
  }
  store_row<T, kD>(static_cast<T*>(a.dq) + flat, dq, a.scale, sees, there, a.h, lane);
}

// ---------------------------------------------------------------------------
// dk and dv: keys fixed, rows walked.
// ---------------------------------------------------------------------------

template <typename T, int kD>
struct KeysShape {
  static constexpr int kRow = Tile<T, kD>::kRow;
  static constexpr int kRows = kRow <= 512 ? 64 : 32;  // of queries, a tile
  static constexpr int kBytes = kRows * kRow;
  static constexpr int kLds = 4 * kBytes + 2 * 2 * 256;  // two stages; each 64 of lse and D
  // Keys and values of a lane in registers, beside their gradients' 2 kD / 2 accumulators.
  static constexpr bool kHold = kRow <= 512;
};

template <typename T, int kD>
__global__ void __launch_bounds__(256, 1) attn_dkv_kernel(AttnArgs a) {
  typedef Tile<T, kD> X;
  typedef KeysShape<T, kD> Sh;
  constexpr int kRows = Sh::kRows, kWaves = 4, kBytes = Sh::kBytes;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bk, tile;  // the first keys are seen by most rows
  place_of(blockIdx.x, a.B * a.KV * a.tiles, a.tiles, &bk, &tile);
  const int b = bk / a.KV, kv = bk - b * a.KV;
  const Sight sight(a, b);
  const int j0 = tile * kRowsWave * kWaves, jw = j0 + w * kRowsWave;
  const int key = jw + (lane & 31);
  const bool there = key < a.S, seen = key < sight.len;
  const T* krow = static_cast<const T*>(a.k) + b * a.pk.b + kv * a.pk.head + key * a.pk.t;
  const T* vrow = static_cast<const T*>(a.v) + b * a.pv.b + kv * a.pv.head + key * a.pv.t;
  RowFrags<T, kD> k, v;
  if constexpr (Sh::kHold) {
    load_row<T, kD>(k, krow, seen, a.h, lane);
    load_row<T, kD>(v, vrow, seen, a.h, lane);
  }
  f32x16_t dk[X::kBlocks] = {}, dv[X::kBlocks] = {};

  // The tokens that may see one of these keys.
  int ta = sight.first(0), tb = sight.last(a.T - 1);
  const int j1 = min(j0 + kRowsWave * kWaves, sight.len) - 1;
  if (sight.causal) {
    ta = max(ta, j0 - sight.start);
    if (sight.window) tb = min(tb, j1 + sight.window - 1 - sight.start);
  }
  if (j0 > j1) tb = ta - 1;
  const int64_t r0 = (int64_t)ta * a.rep, r1 = (int64_t)(tb + 1) * a.rep;
  const int n = tb < ta ? 0 : (int)((r1 - r0 + kRows - 1) / kRows);

  const float inv = 1.f / (float)a.rep;
  const T* qbase = static_cast<const T*>(a.q) + b * a.pq.b + (int64_t)kv * a.rep * a.pq.head;
  const T* dbase = static_cast<const T*>(a.dout) + b * a.pdo.b + (int64_t)kv * a.rep * a.pdo.head;
  const int qt = (int)(a.pq.t * sizeof(T)), qh = (int)(a.pq.head * sizeof(T)),
            dt = (int)(a.pdo.t * sizeof(T)), dh = (int)(a.pdo.head * sizeof(T));
  Loader<T, kD, kRows, kWaves> loader;
  loader.init(a.h, w, lane);
  const uint32_t lds0 = lds_addr(lds_dyn);
  const float* lse = a.lse + (int64_t)bk * a.rows;
  const float* delta = a.delta + (int64_t)bk * a.rows;
  auto fetch = [&](int i) __attribute__((always_inline)) {
    const int64_t r = r0 + (int64_t)i * kRows;
    const int t = (int)(r / a.rep), g0 = (int)(r - (int64_t)t * a.rep);
    const int limit = (int)min((int64_t)kRows, r1 - r);
    const uint32_t at = lds0 + (i & 1) * 2 * kBytes;
    loader.shared(qbase + (int64_t)t * a.pq.t, g0, a.rep, inv, qt, qh, limit, at, w);
    loader.shared(dbase + (int64_t)t * a.pdo.t, g0, a.rep, inv, dt, dh, limit, at + kBytes, w);
    // (Rows past the last are zeros in all four: p = 1, and nothing comes of it.)
    if (w < 2)
      dma4(wave_buffer((w ? delta : lse) + r, limit * 4), __builtin_amdgcn_readfirstlane(lds0 + 4 * kBytes + (i & 1) * 512 + w * 256),
           lane * 4, 0);
  };
  if (n > 0) fetch(0);
  for (int i = 0; i < n; ++i) {
    transfers_done();
    __syncthreads();
    if (i + 1 < n) fetch(i + 1);
    const int64_t r = r0 + (int64_t)i * kRows;
    const int ti = (int)(r / a.rep), tj = min(tb, (int)((r + kRows - 1) / a.rep));
    if (jw > sight.hi(tj) || jw + kRowsWave <= sight.lo(ti) || jw >= sight.len) continue;
    const bool whole = jw >= sight.lo(tj) && jw + kRowsWave - 1 <= sight.hi(ti) &&
                       jw + kRowsWave <= sight.len;
    const uint8_t* qt_ = lds_dyn + (i & 1) * 2 * kBytes;
    const uint8_t* dt_ = qt_ + kBytes;
    const float* st = reinterpret_cast<const float*>(lds_dyn + 4 * kBytes + (i & 1) * 512);
#pragma unroll
    for (int e = 0; e < kRows / 32; ++e) {
      if constexpr (!Sh::kHold) load_row<T, kD>(k, krow, seen, a.h, lane);
      f32x16_t s = times_rows<T, kD>(qt_, 32 * e, k, lane);
      f32x4_t ls[4], dl[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int at = 32 * e + 8 * x + 4 * (lane >> 5);
        ls[x] = *reinterpret_cast<const f32x4_t*>(st + at);
        dl[x] = *reinterpret_cast<const f32x4_t*>(st + 64 + at);
      }
#pragma unroll
      for (int x = 0; x < 16; ++x)
        s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], a.c, -ls[x >> 2][x & 3]));
      if (!whole) {
        const int g0 = (int)(r - (int64_t)ti * a.rep);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int at = g0 + 32 * e + 8 * (x >> 2) + 4 * (lane >> 5) + (x & 3);
          int t = (int)((float)at * inv);
          t -= t * a.rep > at;
          t += (t + 1) * a.rep <= at;
          t += ti;
          if (key < sight.lo(t) || key > sight.hi(t)) s[x] = 0.f;
        }
      }
      add_columns<T, kD>(dv, dt_, 32 * e, s, lane);
      if constexpr (!Sh::kHold) load_row<T, kD>(v, vrow, seen, a.h, lane);
      const f32x16_t dp = times_rows<T, kD>(dt_, 32 * e, v, lane);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float ds = s[x] * (dp[x] - dl[x >> 2][x & 3]);
        s[x] = s[x] == 0.f ? 0.f : ds;
      }
      add_columns<T, kD>(dk, qt_, 32 * e, s, lane);
    }
  }
  const int64_t flat = ((int64_t)(b * (int64_t)a.S + key) * a.KV + kv) * a.h;
  store_row<T, kD>(static_cast<T*>(a.dk) + flat, dk, a.scale, seen, there, a.h, lane);
  store_row<T, kD>(static_cast<T*>(a.dv) + flat, dv, 1.f, seen, there, a.h, lane);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

constexpr int kUnits = 256;

template <typename T, int kD>
struct Launch {
  static constexpr int kSplitWaves = ForwardShape<T, kD>::kSplitWaves;
  static int allow(const void* f, int bytes) {
    if (bytes > 65536)
      DPC_HIP_CHECK(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return DPC_OK;
  }
  static int forward(AttnArgs& a, hipStream_t s) {
    typedef ForwardShape<T, kD> Sh;
    if (a.splits > 0) {
      a.tiles = (int)((a.rows + kRowsWave - 1) / kRowsWave);
      const int rc = allow((const void*)attn_forward_kernel<T, kD, true>, Sh::kSplitLds);
      if (rc) return rc;
      hipLaunchKernelGGL((attn_forward_kernel<T, kD, true>),
                         dim3((unsigned)((int64_t)a.B * a.KV * a.tiles * a.splits)),
                         dim3(64 * Sh::kSplitWaves), Sh::kSplitLds, s, a);
      DPC_HIP_CHECK(hipGetLastError());
      const int64_t rows = (int64_t)a.B * a.KV * a.rows;
      hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s,
                         a, a.splits * Sh::kSplitWaves);
      DPC_HIP_CHECK(hipGetLastError());
      return DPC_OK;
    }
    a.tiles = (int)((a.rows + 127) / 128);
    const int rc = allow((const void*)attn_forward_kernel<T, kD, false>, Sh::kLds);
    if (rc) return rc;
    hipLaunchKernelGGL((attn_forward_kernel<T, kD, false>),
                       dim3((unsigned)((int64_t)a.B * a.KV * a.tiles)), dim3(256), Sh::kLds, s, a);
    DPC_HIP_CHECK(hipGetLastError());
    return DPC_OK;
  }
  static int backward(AttnArgs& a, hipStream_t s) {
    if (a.rows > 0) {
      a.tiles = (int)((a.rows + 127) / 128);
      constexpr int kLds = ForwardShape<T, kD>::kLds;
      const int rc = allow((const void*)attn_dq_kernel<T, kD>, kLds);
      if (rc) return rc;
      hipLaunchKernelGGL((attn_dq_kernel<T, kD>),
                         dim3((unsigned)((int64_t)a.B * a.KV * a.tiles)), dim3(256), kLds, s, a);
      DPC_HIP_CHECK(hipGetLastError());
    }
    if (a.S > 0 && a.dk) {
      a.tiles = (a.S + 127) / 128;
      constexpr int kLds = KeysShape<T, kD>::kLds;
      const int rc = allow((const void*)attn_dkv_kernel<T, kD>, kLds);
      if (rc) return rc;
      hipLaunchKernelGGL((attn_dkv_kernel<T, kD>),
                         dim3((unsigned)((int64_t)a.B * a.KV * a.tiles)), dim3(256), kLds, s, a);
      DPC_HIP_CHECK(hipGetLastError());
    }
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
  return B * KV <= most / ((rows + 31) / 32 + 1) && B * KV <= most / ((S + 127) / 128 + 1);
}

// Splits of the keys (0: none): where whole row tiles would leave compute units idle,
// enough workgroups of 32 rows for two rounds, none with fewer than four tiles of 32 keys a wave.
int splits_of(int64_t B, int64_t T, int64_t S, int H, int KV, int h, int dtype) {
  const int64_t rows = T * (H / KV), heads = B * KV;
  if (heads * ((rows + 127) / 128) >= kUnits) return 0;
  const int64_t groups = heads * ((rows + 31) / 32);
  int64_t n = (2 * kUnits + groups - 1) / groups;
  const int64_t most = S / (32 * 4 * (h * (dtype == DPC_F32 ? 4 : 2) <= 256 ? 4 : 1));
  if (n > most) n = most;
  return n < 1 ? 1 : (n > 64 ? 64 : (int)n);
}

}  // namespace

namespace {

int tensor_places(const int64_t* s, int bytes, int rep, Places* p) {
  *p = Places{s[0], s[1], s[2]};
  const int64_t most = (int64_t)kOutOfRange - (1 << 20);
  if (s[1] < 0 || s[2] < 0 || s[1] > most || s[2] > most) return DPC_ENOTSUP;
  // A tile's 64 rows (of shared key heads: 65 tokens at most) in one buffer.
  if ((65 * s[1] + rep * s[2]) * bytes > most) return DPC_ENOTSUP;
  return (s[0] * bytes | s[1] * bytes | s[2] * bytes) & 15 ? DPC_EINVAL : DPC_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" size_t dpc_attention_workspace_bytes(int64_t B, int64_t T, int64_t S, int H, int KV,
                                                int h, int dtype) {
  if (!valid_sizes(B, T, S, H, KV, h, dtype) || B == 0 || T == 0) return 0;
  const int64_t parts = (int64_t)splits_of(B, T, S, H, KV, h, dtype) * split_waves(dtype, h);
  return (size_t)(parts * B * T * H * (h * 4 + 8));
}

extern "C" int dpc_attention(const void* q, const void* k, const void* v, const int64_t* strides,
                             int64_t B, int64_t T, int64_t S, int H, int KV, int h, int dtype,
                             const int64_t* lengths, const int64_t* starts, int causal, int window,
                             double scale, void* out, float* lse, void* ws, size_t ws_bytes,
                             void* stream) {
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
  if (const int rc = tensor_places(strides, bytes, a.rep, &a.pq)) return rc;
  if (const int rc = tensor_places(strides + 3, bytes, 1, &a.pk)) return rc;
  if (const int rc = tensor_places(strides + 6, bytes, 1, &a.pv)) return rc;
  const size_t need = dpc_attention_workspace_bytes(B, T, S, H, KV, h, dtype);
  if (ws_bytes < need) return DPC_ENOSPC;
  if (need && (!ws || ((uintptr_t)ws & 255))) return DPC_EINVAL;
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = out;
  a.lse = lse;
  a.B = (int)B;
  a.T = (int)T;
  a.S = (int)S;
  a.KV = KV;
  a.h = h;
  a.rows = T * a.rep;
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
                                  int window, double scale, const float* lse, void* dq, void* dk,
                                  void* dv, void* ws, size_t ws_bytes, void* stream) {
  if (!valid_sizes(B, T, S, H, KV, h, dtype) || !strides || window < 0 || (window && !causal) ||
      !((float)scale > 0.f) || !isfinite((float)scale))
    return DPC_EINVAL;
  if (B == 0 || (T == 0 && S == 0)) return DPC_OK;
  if ((T && (!q || !out || !dout || !lse || !dq)) || (S && (!k || !v)) || (!dk != !dv) ||
      !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(dout) ||
      !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return DPC_EINVAL;
  AttnArgs a = {};
  const int bytes = dtype == DPC_F32 ? 4 : 2;
  a.rep = H / KV;
  if (const int rc = tensor_places(strides, bytes, a.rep, &a.pq)) return rc;
  if (const int rc = tensor_places(strides + 3, bytes, 1, &a.pk)) return rc;
  if (const int rc = tensor_places(strides + 6, bytes, 1, &a.pv)) return rc;
  if (const int rc = tensor_places(strides + 9, bytes, a.rep, &a.pdo)) return rc;
  const size_t need = dpc_attention_grad_workspace_bytes(B, T, H);
  if (ws_bytes < need) return DPC_ENOSPC;
  if (need && (!ws || ((uintptr_t)ws & 255))) return DPC_EINVAL;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.dout = dout;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.lse = const_cast<float*>(lse);
  a.delta = static_cast<float*>(ws);
  a.B = (int)B;
  a.T = (int)T;
  a.S = (int)S;
  a.KV = KV;
  a.h = h;
  a.rows = T * a.rep;
  a.lengths = lengths;
  a.starts = starts;
  a.causal = causal != 0;
  a.window = window < kMostTokens ? window : (int)kMostTokens;
  a.scale = (float)scale;
  a.c = (float)(scale * 1.44269504088896340736);
  hipStream_t s = (hipStream_t)stream;
  return by_width(dtype, h, [&](auto l) { return decltype(l)::backward(a, s); });
}
