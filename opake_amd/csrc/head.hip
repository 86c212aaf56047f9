// Losses of a vocabulary head without its logits: softmax cross entropy, and
// distillation from a teacher's top logits, from hidden states H [N, D] and the
// head's weight W [V, D].
//
//   z = inv_tau H W^T,  lse_n = log sum_v exp z_nv,  p = exp(z - lse)
//   cross entropy   loss_n = lse_n - z_n,t
//   distillation    q = softmax of the teacher's entries / tau,
//                   loss_n = tau^2 sum_k q_k (log q_k - z_n,k + lse_n)
//   gradient        dz_nv = g_n coef (p_nv - sum_k q_nk [col_nk = v])
//                   dH = dz W,  dW = dz^T H
//
// Logits, lse and their differences are held in units of log 2 (as exp2 takes them), and
// exponentials are taken of differences that are formed first: exact where a logit is
// its row's largest, however large it is.
//
// Cross entropy is the K = 1, q = 1 case, so both share every kernel.
//
// Rows without a target (the ignored index; no teacher entry above -inf) are left
// out of every product: the rows that have one are numbered on the device, and the
// kernels run over that many.  So such rows cost nothing and whatever they hold
// (padding, NaN) reaches nothing.
//
// Loss: one product whose 256 x 256 tiles never leave the chip; each leaves its
// maximum and sum of exponentials per row and the logits at the entries' columns; a
// join turns them into lse and the loss.
//
// Gradients: a product's tiles also leave exp(z - half a tile's maximum) as fp16
// (float32 inputs: two planes), and a pass turns those into dz (bf16, or planes) once
// the row's lse is known.  So the logits are made once:
//   * the hidden states' alone (a frozen head): the rows in chunks of up to 512 MiB of
//     exponentials, dz for g = 1 in place, and one product with W gives dH for g = 1,
//     kept in float32 until the backward multiplies each row by its g.  Two products.
//   * a trained head whose exponentials fit in 512 MiB: they are kept, and the backward
//     makes dz, dz W and dz^T H of them (float32: dz and dH for g = 1 in the forward;
//     g goes to dH's rows and to a copy of H).  Three products.
//   * beyond that the backward makes the logits again, in pieces of the vocabulary, and
//     turns them into dz in the accumulators.  Four products.
// The products bound it: at 8192 rows, 2048 wide, vocabulary 32000 (bf16) the tiles with
// their exponentials take 850 us, dz 197, dz W 820, a frozen head in all 1.85 ms.  (Two
// products of that size take 1.50 ms in the library, and one writes 524 MB of logits.)
// dz at an entry's column, where p and q may cancel, is formed in float32 by the
// join and put in place of the tile's value.
//
// What is held in fewer than 32 bits, bf16 inputs: exponentials in fp16 (2^-11 of
// them at most, below what follows) and dz in bf16, 2^-8 at most, entries included.
// The products with W and H take dz in their type: in two planes it would cost twice the
// products.  The gradients' own rounding to bf16 is 1.66e-3 of them in the mean square;
// with dz's they are 1.84e-3 from 64 bits for cross entropy and 2.3e-3 for distillation
// from 64 entries, the same as products in 32 bits give from a dz rounded so.  (float32
// inputs: mm_tile.h.)
#include <math.h>

#include <type_traits>

#include "common.h"
#include "mm_planes.h"

namespace {

constexpr double kLog2e64 = 1.44269504088896340736;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

DPC_DEVICE float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
DPC_DEVICE float fast_exp(float x) { return exp2_fast(x * kLog2e); }

constexpr int kLdsBytes = 131072;
__shared__ __attribute__((aligned(16))) uint8_t lds_all[kLdsBytes];

// ---------------------------------------------------------------------------
// Rows, entries and operands as the tiles read them.
// ---------------------------------------------------------------------------

constexpr int kDzShift = 14;  // of exponentials and dz, which are at most 1 (the gradient
                              // is applied later)
constexpr float kDzScale = 1 << kDzShift;

// The rows that have a target, in order: count, active[count], and each row's
// place among them or -1.
struct Rows {
  int32_t* count;
  int32_t* active;
  int32_t* place;
};

// The largest finite magnitudes that the planes' shifts come from, as bits.  Each row
// of H has its own for the logits, so that one row's outlier costs the others nothing;
// dW's sums over rows and W's over the vocabulary take one for the tensor.
struct Tops {
  uint32_t* h;
  uint32_t* w;
  uint32_t* row;  // [rows with a target]
};

// Distillation: whether a row has an entry that counts (or one that is wrong: an
// index outside the vocabulary, a NaN).  One wave a row.
__global__ void __launch_bounds__(256) entries_kernel(const int64_t* __restrict__ index,
                                                      const float* __restrict__ teacher, int64_t N,
                                                      int K, int V, int32_t* __restrict__ flag) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  bool has = false;
  for (int k = lane; k < K; k += 64) {
    const int64_t c = index[n * K + k];
    const float t = teacher[n * K + k];
    has |= c >= V || (c >= 0 && !(t == -INFINITY));
  }
  has = __any(has);
  if (lane == 0) flag[n] = has;
}

// Numbers the rows with a target, and writes the others' losses (0).  Latency bounds it
// (14 us for 16384 rows, two rounds).  One workgroup, 8192 rows a round (8 loads in flight
// a thread): ballots count a wave's 64 rows, and one wave adds up the round's 128 counts.
// `flags` (distillation): rows.place holds entries_kernel's flags.
__global__ void __launch_bounds__(1024) rows_kernel(const int64_t* __restrict__ index,
                                                    int64_t ignore, int flags, int64_t N,
                                                    Rows rows, float* __restrict__ loss,
                                                    Tops tops) {
  __shared__ int total[128], before[129];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int64_t base = 0;
  for (int64_t r0 = 0; r0 < N; r0 += 8192) {
    bool on[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const int64_t n = r0 + t * 1024 + tid;
      on[t] = n < N && (flags ? rows.place[n] != 0 : index[n] != ignore);
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const unsigned long long m = __ballot(on[t]);
      if (lane == 0) total[t * 16 + w] = __popcll(m);
    }
    __syncthreads();
    if (w == 0) {
      const int a = total[2 * lane], b = total[2 * lane + 1];
      int upto = a + b;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
      before[2 * lane] = upto - a - b;
      before[2 * lane + 1] = upto - b;
      if (lane == 63) before[128] = upto;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const int64_t n = r0 + t * 1024 + tid;
      const unsigned long long m = __ballot(on[t]);
      const int64_t at = base + before[t * 16 + w] + __popcll(m & ((1ull << lane) - 1));
      if (n < N) {
        rows.place[n] = on[t] ? (int32_t)at : -1;
        if (on[t])
          rows.active[at] = (int32_t)n;
        else
          loss[n] = 0.f;
      }
    }
    base += before[128];
    __syncthreads();
  }
  if (tid == 0) *rows.count = (int32_t)base;
  if (tid == 0) *tops.h = *tops.w = 0u;
}

// The entries of 256 consecutive numbered rows (one B tile) sorted by the part of a
// tile that they fall into: 256 columns, and of those the wave whose accumulators hold
// the entry (wave w: columns (w & 1) * 128, rows (w >> 1) * 64).  Wave w of tile t finds
// its own at start[8 t + w] .. start[8 t + w + 1] - 1 of the block's list.
struct Entries {
  int32_t* cols;    // [rows, K]: the column; -1: absent, -2: outside the vocabulary
  uint2* list;      // [blocks][256 K]: {row in block * K + k, row in block << 8 | column in tile}
  int32_t* start;   // [blocks][8 tiles + 1]
};

DPC_DEVICE int entry_part(int row, int col) {
  return (col >> 8) * 8 + ((row >> 6) << 1 | ((col >> 7) & 1));
}

// Operands as the tiles read them, in planes of 16-bit rows padded with zeros: the
// rows with a target of `hidden` (bf16 rows of whole 16-byte chunks: only if some
// are left out, else the tiles read the caller's own) and, where it needs planes or
// padding, the weight.  The first `blocks` workgroups make the entries' lists.  Bound by
// memory (float32, 33 MB of H and 262 MB of W into planes: 105 us, 5.6 TB/s) or by the
// lists' counters (8192 rows of 64 entries: 37 us).
struct PrepArgs {
  const void* hidden;
  const void* weight;  // null: read as it is
  int dtype, D, V, K;
  int64_t N, ld;
  Rows rows;
  uint16_t* h;
  uint16_t* w;
  bool pack;
  Tops tops;     // float32
  uint16_t* hg;        // float32, for dW: planes of H times the losses' gradient over gmax
  const int64_t* index;
  bool teacher;
  int blocks, parts;
  Entries entries;
  void* zero;          // the hidden gradient, whose rows without a target are zeroed
  const float* g;      // backward: the losses' gradient,
  float* gmax;         // its largest magnitude that is finite (1 if all are 0), and
  float* g_over;       // [rows]: the gradient over that, by the rows' numbers
};

DPC_DEVICE void pack_chunk(const void* src, int dtype, int64_t row, int D, int c, int64_t ld,
                           int64_t plane, uint16_t* dst, int64_t to, int shift, float times) {
  float x[8];
  u32x4_t o;
  if (dtype == DPC_BF16) {
    const uint16_t* from = static_cast<const uint16_t*>(src) + row * D + c;
    if (c + 8 <= D && D % 8 == 0 && ((uintptr_t)src & 15) == 0) {
      *reinterpret_cast<u32x4_t*>(dst + to * ld + c) = *reinterpret_cast<const u32x4_t*>(from);
      return;
    }
    uint16_t h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      h[e] = c + e < D ? from[e] : (uint16_t)0;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (uint32_t)h[2 * e] | ((uint32_t)h[2 * e + 1] << 16);
    *reinterpret_cast<u32x4_t*>(dst + to * ld + c) = o;
    return;
  }
  const float* from = static_cast<const float*>(src) + row * D + c;
  if (c + 8 <= D && D % 4 == 0 && ((uintptr_t)src & 15) == 0) {
    const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(from),
                  hi = *reinterpret_cast<const f32x4_t*>(from + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < 4 ? lo[e] : hi[e - 4];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = c + e < D ? from[e] : 0.f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = ldexpf(x[e] * times, shift);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = (uint32_t)half_plane(x[2 * e], p) | ((uint32_t)half_plane(x[2 * e + 1], p) << 16);
    *reinterpret_cast<u32x4_t*>(dst + p * plane + to * ld + c) = o;
  }
}

// One read of H and W: 262 MB of W in 70 us (3.7 TB/s).
// blockIdx.y 0: H's rows with a target, one wave a row; 1: W.  (Maxima: any order gives
// the same.)
__global__ void __launch_bounds__(256) tops_kernel(const float* __restrict__ hidden,
                                                   const float* __restrict__ weight, int D, int V,
                                                   Rows rows, Tops tops) {
  __shared__ uint32_t waves[4];
  const int lane = threadIdx.x & 63;
  const bool of_w = blockIdx.y == 1;
  uint32_t top = 0;
  if (of_w) {
    const int64_t n = V * (int64_t)D, t0 = (int64_t)blockIdx.x * 256 + threadIdx.x,
                  step = (int64_t)gridDim.x * 256;
    const int64_t whole = ((uintptr_t)weight & 15) == 0 ? n / 4 : 0;
#pragma unroll 4
    for (int64_t i = t0; i < whole; i += step) {
      const f32x4_t x = reinterpret_cast<const f32x4_t*>(weight)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, finite_bits(x[e]));
    }
#pragma unroll 4
    for (int64_t i = 4 * whole + t0; i < n; i += step) top = max(top, finite_bits(weight[i]));
    top = wave_max_bits(top);
  } else {
    const int64_t count = *rows.count;
    for (int64_t c = blockIdx.x * 4ll + (threadIdx.x >> 6); c < count; c += gridDim.x * 4ll) {
      const float* x = hidden + (int64_t)rows.active[c] * D;
      uint32_t mine = 0;
#pragma unroll 4
      for (int d = lane; d < D; d += 64) mine = max(mine, finite_bits(x[d]));
      mine = wave_max_bits(mine);
      if (lane == 0) tops.row[c] = mine;
      top = max(top, mine);
    }
  }
  // One atomic a workgroup: those of a word go one after the other (2048 of them took
  // 40 us).
  if (lane == 0) waves[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    top = max(max(waves[0], waves[1]), max(waves[2], waves[3]));
    if (top) atomicMax(of_w ? tops.w : tops.h, top);
  }
}

constexpr int kPrepThreads = 512;
constexpr int kMaxTiles = 1 << 11;  // of the vocabulary (8 counters each in LDS)

// i / K for i < 2^24 (exact in float; the quotient is off by one at most).
DPC_DEVICE int row_of(int i, int K, float inv) {
  int r = (int)((float)i * inv);
  r -= r * K > i;
  r += (r + 1) * K <= i;
  return r;
}

DPC_DEVICE void list_entries(const PrepArgs& a, int block, int64_t count, int* counter) {
  constexpr int kBatch = 8;  // loads in flight a thread
  const int tid = threadIdx.x;
  const int64_t first = (int64_t)block * kMmTile;
  if (first >= count) return;
  const int rows = (int)(count - first < kMmTile ? count - first : kMmTile);
  const int n = rows * a.K;
  const float inv = 1.0f / (float)a.K;
  const int32_t* active = a.rows.active + first;
  int32_t* cols = a.entries.cols + first * a.K;
  for (int t = tid; t <= a.parts; t += kPrepThreads) counter[t] = 0;
  __syncthreads();
  for (int i0 = tid; i0 < n; i0 += kBatch * kPrepThreads) {
    int64_t from[kBatch], x[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kPrepThreads;
      const int r = i < n ? row_of(i, a.K, inv) : 0;
      from[b] = i < n ? (int64_t)active[r] * a.K + (i - r * a.K) : 0;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) x[b] = a.index[from[b]];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kPrepThreads;
      if (i >= n) break;
      const int c = a.teacher && x[b] < 0 ? -1 : (x[b] >= 0 && x[b] < a.V ? (int)x[b] : -2);
      cols[i] = c;
      if (c >= 0) atomicAdd(&counter[entry_part(row_of(i, a.K, inv), c) + 1], 1);
    }
  }
  __syncthreads();
  if (tid < 64) {  // counts -> starts, 64 at a time
    int base = 0;
    for (int t0 = 0; t0 <= a.parts; t0 += 64) {
      const int t = t0 + tid;
      const int mine = t <= a.parts ? counter[t] : 0;
      int upto = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (tid >= d) upto += o;
      }
      if (t <= a.parts) {
        counter[t] = base + upto;
        a.entries.start[(int64_t)block * (a.parts + 1) + t] = base + upto;
      }
      base += __shfl(upto, 63);
    }
  }
  __syncthreads();
  // The order within a part is that of the atomics: each entry has a place
  // of its own in every output, so no result depends on it.
  uint2* list = a.entries.list + first * a.K;
  for (int i0 = tid; i0 < n; i0 += kBatch * kPrepThreads) {
    int c[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kPrepThreads;
      c[b] = i < n ? cols[i] : -1;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kPrepThreads;
      if (c[b] < 0) continue;
      const int r = row_of(i, a.K, inv);
      const int at = atomicAdd(&counter[entry_part(r, c[b])], 1);
      list[at] = make_uint2((uint32_t)i, (uint32_t)(r << 8 | (c[b] & 255)));
    }
  }
}

// The losses' gradient over its largest finite magnitude, by one workgroup.
DPC_DEVICE void over_gmax(const PrepArgs& a, int64_t count) {
  __shared__ float wave_top[kPrepThreads / 64];
  float top = 0.f;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < count; i += kPrepThreads) {
    const float x = fabsf(a.g[a.rows.active[i]]);
    if (x < INFINITY) top = fmaxf(top, x);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = top;
  __syncthreads();
  top = wave_top[0];
  for (int i = 1; i < kPrepThreads / 64; ++i) top = fmaxf(top, wave_top[i]);
  if (!(top > 0.f)) top = 1.f;
  if (threadIdx.x == 0) *a.gmax = top;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < count; i += kPrepThreads)
    a.g_over[i] = a.g[a.rows.active[i]] / top;
}

__global__ void __launch_bounds__(kPrepThreads) gmax_kernel(PrepArgs a) {
  over_gmax(a, *a.rows.count);
}

__global__ void __launch_bounds__(kPrepThreads) prep_kernel(PrepArgs a) {
  extern __shared__ int counter[];
  const int64_t count = *a.rows.count;
  if ((int)blockIdx.x < a.blocks) {
    list_entries(a, blockIdx.x, count, counter);
    return;
  }
  if (a.g && !a.hg && blockIdx.x == 0) over_gmax(a, count);
  const int64_t t0 = (int64_t)(blockIdx.x - a.blocks) * kPrepThreads + threadIdx.x,
                step = (int64_t)(gridDim.x - a.blocks) * kPrepThreads;
  const int64_t chunks = a.ld / 8;
  const bool f32 = a.dtype == DPC_F32;
  const int shift_h = f32 ? half_shift(*a.tops.h) : 0, shift_w = f32 ? half_shift(*a.tops.w) : 0;
  const bool pack_h = a.h && (a.pack || count < a.N);
  if (pack_h || a.hg)
    for (int64_t i = t0; i < count * chunks; i += step) {
      const int64_t c = i / chunks;
      const int at = (int)(i - c * chunks) * 8;
      if (pack_h)
        pack_chunk(a.hidden, a.dtype, a.rows.active[c], a.D, at, a.ld, a.N * a.ld, a.h, c,
                   f32 ? half_shift(a.tops.row[c]) : 0, 1.f);
      if (a.hg)
        pack_chunk(a.hidden, a.dtype, a.rows.active[c], a.D, at, a.ld, a.N * a.ld, a.hg, c,
                   shift_h, a.g_over[c]);
    }
  if (a.weight)
    for (int64_t i = t0; i < a.V * chunks; i += step) {
      const int64_t v = i / chunks;
      pack_chunk(a.weight, a.dtype, v, a.D, (int)(i - v * chunks) * 8, a.ld, (int64_t)a.V * a.ld,
                 a.w, v, shift_w, 1.f);
    }
  if (a.zero && count < a.N)
    for (int64_t i = t0; i < a.N * a.D; i += step)
      if (a.rows.place[i / a.D] < 0) {
        if (a.dtype == DPC_F32)
          static_cast<float*>(a.zero)[i] = 0.f;
        else
          static_cast<uint16_t*>(a.zero)[i] = 0;
      }
}

// The hidden rows that a launch reads: the caller's where every row has a target
// and needs no padding, else the packed ones; `first`, `most`: the launch's chunk.
struct Hidden {
  const uint16_t* own;  // null: always the packed rows
  const uint16_t* packed;
  const int32_t* count;
  int64_t N, ld;
  int first, most;
};

DPC_DEVICE int hidden_rows(const Hidden& h, const uint16_t** p) {
  const int count = __builtin_amdgcn_readfirstlane(*h.count);
  *p = (h.own && count == h.N ? h.own : h.packed) + h.first * h.ld;
  return max(0, min(count - h.first, h.most));
}

// ---------------------------------------------------------------------------
// Loss: the tile's statistics and the entries' logits.
// ---------------------------------------------------------------------------

// A workgroup a compute unit goes through tiles, the next one's first step on its way
// while a tile's epilogue runs.  2048 rows, 4096 wide, vocabulary 131072: 1.58 ms a call
// (1.39 PFLOP/s; the K loop's bound, mm_tile.h); 8192 x 2048 x 32000 with exponentials
// written: 850 us (1.26 PFLOP/s).  Nothing hides the epilogues' exponentials and stores.
// (A frozen head's call of twice that: 3.83 ms with a workgroup a tile, 3.77 so.)
// A tile is two halves of 128 columns (one a wave): statistics are per half, so the
// waves finish their halves without waiting for each other or using LDS, while the
// workgroup's next tile is on its way into it.
struct StatsArgs {
  MmArgs mm;  // A = W (vocabulary), B = H (rows with a target)
  Hidden h;
  int V, K;
  float inv_tau;  // times log2 e
  Tops tops;
  Entries entries;
  float* picked;   // [rows, K]: z at the entries' columns
  f32x2_t* part;   // [2 tiles_a][N]: maximum and sum of exponentials of each half
  int64_t N;
  uint16_t* e;     // the chunk's exp(z - the half's maximum) times 2^kDzShift as fp16
                   // (float32 inputs: in two planes), native order: 2^-11 of them is
                   // lost at most (2^-23), or 2^-39 of the maximum
  int64_t lde, plane;  // blocks of a row of them, elements
};

// What a row's products are to be multiplied by (the planes' shifts undone).
DPC_DEVICE float logit_factor(float inv_tau, uint32_t top_h, uint32_t top_w) {
  const int n = -(half_shift(top_h) + half_shift(top_w));
  return ldexpf(inv_tau, max(-126, min(126, n)));
}

// The lane, of unknown value to the compiler: what an epilogue computes from it would
// otherwise be kept in registers through the product's loop, which has none to spare.
DPC_DEVICE int epilogue_lane() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// Loaded values that have to be there: a later wait for them would also wait for the
// next tile's transfers, which the compiler does not count.
template <typename T>
DPC_DEVICE void arrived(T& x) {
  asm volatile("" : "+v"(x));
}

// x over lanes l, l ^ 16, l ^ 32, l ^ 48 (the lanes that share a column of the
// accumulators), in each of them.
template <typename Op>
DPC_DEVICE float column_all(float x, Op op) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const uint32_t v = __float_as_uint(x);
  const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return op(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// OR of x over the wave, uniform.
DPC_DEVICE uint32_t wave_or(uint32_t x) {
  auto step = [&](auto ctrl) __attribute__((always_inline)) {
    x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, false);
  };
  step(std::integral_constant<int, 0xB1>());   // quad_perm [1, 0, 3, 2]
  step(std::integral_constant<int, 0x4E>());   // quad_perm [2, 3, 0, 1]
  step(std::integral_constant<int, 0x141>());  // row_half_mirror
  step(std::integral_constant<int, 0x140>());  // row_mirror
  return __builtin_amdgcn_readlane(x, 0) | __builtin_amdgcn_readlane(x, 16) |
         __builtin_amdgcn_readlane(x, 32) | __builtin_amdgcn_readlane(x, 48);
}

// Entry y (row in block << 8 | column in tile) is value r of block i, j of the wave's
// accumulators in lane from: the values of up to 64 entries, one a lane, by a lane
// move of each block that holds one.
DPC_DEVICE float entry_values(const MmAcc<false>& acc, uint32_t y, bool on) {
  const int block = (int)(((y >> 4) & 7) << 2 | ((y >> 12) & 3));
  const int from = (int)(((y >> 8) & 15) | ((y >> 2) & 3) << 4) * 4;
  const uint32_t hit = wave_or(on ? 1u << block : 0u);
  float v = 0.f;
#pragma unroll
  for (int n = 0; n < 32; ++n)
    if ((hit >> n) & 1) {
      float b[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float a = acc.v[n >> 2][n & 3][r];
        b[r] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(a)));
      }
      const float x = y & 2 ? (y & 1 ? b[3] : b[2]) : (y & 1 ? b[1] : b[0]);
      v = block == n ? x : v;
    }
  return v;
}

template <bool kEmit, bool kHalf>
DPC_DEVICE void stats_epilogue(const StatsArgs& s, MmAcc<false>& acc, const f32x4_t& factor,
                               int N, int ta, int tb, int w, int64_t g0, const uint2* list,
                               int e0, int e1, uint2 first) {
#pragma clang fp contract(off)  // the difference is of the rounded logit and its maximum
  const int lane = epilogue_lane(), wm = w & 1, wn = w >> 1;
  const int v0 = ta * kMmTile, n0 = tb * kMmTile;
  const int vl = wm * 128 + 4 * (lane >> 4);  // + 16 i + r
  const int tl = wn * 64 + (lane & 15);       // + 16 j
  const int vleft = s.V - v0 - vl;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc.v[i][j] *= kHalf ? factor[j] : s.inv_tau;
  for (int e = e0; e < e1; e += 64) {
    const uint2 x = e == e0 ? first : list[min(e + lane, e1 - 1)];
    const bool on = e + lane < e1;
    const float v = entry_values(acc, x.y, on);
    if (on) s.picked[g0 * s.K + x.x] = v;
  }
  if (v0 + kMmTile > s.V) {  // past the vocabulary
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * i + r >= vleft) acc.v[i][j][r] = -INFINITY;
  }
  f32x2_t* part = s.part + (int64_t)(2 * ta + wm) * s.N + g0 + tl;
  uint16_t* out = s.e + (tb * s.lde + 4 * ta + 2 * wm) * kMmBlock + wn * 2048 + lane * 8;
  float tops[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, acc.v[i][j][r]);
    tops[j] = column_all(m, [](float a, float b) { return fmaxf(a, b); });
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float m = tops[j], base = m == -INFINITY ? 0.f : m;
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = exp2_fast(acc.v[i][j][r] - base);
        acc.v[i][j][r] = e;
        sums[r] += e;
      }
    if constexpr (kEmit) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {  // 32 columns: half p % 2 of block p / 2
        typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
        uint16_t* at = out + (p >> 1) * kMmBlock + (p & 1) * 8192 + j * 512;
        half8_t h;
        if constexpr (kHalf) {
#pragma unroll
          for (int pl = 0; pl < 2; ++pl) {
#pragma unroll
            for (int r = 0; r < 8; ++r)
              h[r] = __builtin_bit_cast(
                  _Float16, half_plane(acc.v[2 * p + (r >> 2)][j][r & 3] * kDzScale, pl));
            *reinterpret_cast<half8_t*>(at + pl * s.plane) = h;
          }
        } else {
#pragma unroll
          for (int r = 0; r < 8; ++r)
            h[r] = (_Float16)(acc.v[2 * p + (r >> 2)][j][r & 3] * kDzScale);
          *reinterpret_cast<half8_t*>(at) = h;
        }
      }
    }
    const float sum = column_all((sums[0] + sums[1]) + (sums[2] + sums[3]),
                                 [](float a, float b) { return a + b; });
    if (lane < 16 && n0 + tl + 16 * j < N) part[16 * j] = f32x2_t{m, sum};
  }
}

// A wave's entries of a tile, in a list by row block, tile and wave: [e0, e1), the first
// 64 of them.
struct WaveEntries {
  const uint2* list;
  int e0, e1;
  uint2 first;
  DPC_DEVICE WaveEntries(const Entries& e, int K, int tiles_v, int vt, int64_t block, int w,
                         int lane) {
    const int32_t* start = e.start + block * (8 * tiles_v + 1) + 8 * vt + w;
    list = e.list + block * kMmTile * K;
    e0 = start[0];
    e1 = start[1];
    first = e0 < e1 ? list[min(e0 + lane, e1 - 1)] : make_uint2(0u, 0u);
  }
};

// What the products of the lane's rows are to be multiplied by (float32).
DPC_DEVICE f32x4_t row_factors(const StatsArgs& s, int N, int tb, int w, uint32_t top_w) {
  const int lane = epilogue_lane();
  f32x4_t f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = tb * kMmTile + (w >> 1) * 64 + 16 * j + (lane & 15);
    f[j] = logit_factor(s.inv_tau, n < N ? s.tops.row[s.h.first + n] : 0u, top_w);
  }
  return f;
}

template <bool kEmit, bool kHalf>
__global__ void __launch_bounds__(kMmThreads, 1) head_stats_kernel(StatsArgs s) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int N = hidden_rows(s.h, &s.mm.b.p);
  s.mm.b.rows = N;
  s.mm.tiles_b = tiles_of(N);
  MmTile<true, true, false, false, kHalf> tile(s.mm, lds_all);
  MmAcc<false> acc;
  const uint32_t top_w = kHalf ? *s.tops.w : 0u;
  int split, ta, tb, ta2, tb2, id = blockIdx.x;
  bool more = mm_tile_of(s.mm, id, &split, &ta2, &tb2);
  if (more) tile.begin(ta2, tb2, 0);
  while (more) {
    ta = ta2;
    tb = tb2;
    const int64_t g0 = s.h.first + (int64_t)tb * kMmTile;  // the first row's number
    WaveEntries own(s.entries, s.K, s.mm.tiles_a, ta, g0 / kMmTile, w, lane);
    tile.run(acc);
    f32x4_t factor = {};
    if constexpr (kHalf) {
      factor = row_factors(s, N, tb, w, top_w);
      arrived(factor);
    }
    arrived(own.first.x);
    arrived(own.first.y);
    id += gridDim.x;
    more = mm_tile_of(s.mm, id, &split, &ta2, &tb2);
    if (more) tile.begin(ta2, tb2, 0);
    stats_epilogue<kEmit, kHalf>(s, acc, factor, N, ta, tb, w, g0, own.list, own.e0, own.e1,
                                 own.first);
  }
}

// Few tiles (few rows, or a small vocabulary): the products' K steps in slices, each
// slice's accumulators left as they are held ([slice][tile][wave][block][lane]), then
// the same epilogues on their sums.  A workgroup adds up one wave's part of a tile: its
// four waves every fourth slice each, 16 loads a lane in flight, then the first one theirs,
// all in a fixed order.  Rows past the last are not written, and zeros; waves that have no
// others have nothing to do, and `waves` leaves out those that never have any.
struct LogitsArgs {
  MmArgs mm;
  Hidden h;
  f32x4_t* z;
  int tiles;  // of a slice
};

DPC_DEVICE int64_t logits_at(int64_t tile, int w) { return (tile * 8 + w) * 32 * 64; }

template <bool kHalf>
__global__ void __launch_bounds__(kMmThreads, 1) head_logits_kernel(LogitsArgs s) {
  const int N = hidden_rows(s.h, &s.mm.b.p);
  s.mm.b.rows = N;
  s.mm.tiles_b = tiles_of(N);
  int split, ta, tb;
  if (!mm_tile_of(s.mm, blockIdx.x, &split, &ta, &tb)) return;
  MmTile<true, true, false, false, kHalf> tile(s.mm, lds_all);
  MmAcc<false> acc;
  tile.begin(ta, tb, split);
  tile.run(acc);
  const int lane = epilogue_lane(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x4_t* z = s.z + logits_at((int64_t)split * s.tiles + tb * s.mm.tiles_a + ta, w) + lane;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (tb * kMmTile + (w >> 1) * 64 + 16 * j < N)
#pragma unroll
      for (int i = 0; i < 8; ++i) z[(j * 8 + i) * 64] = acc.v[i][j];
}

constexpr int kAddWaves = 4;

// The sums, in the first wave; false in the others.
DPC_DEVICE bool add_logits(const f32x4_t* z, int slices, int tiles, int64_t tile, int w, int row0,
                           int N, MmAcc<false>& acc) {
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
  f32x4_t* lds = reinterpret_cast<f32x4_t*>(lds_all);  // [kAddWaves - 1][32][64]
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc.v[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int s = q; s < slices; s += kAddWaves) {
    const f32x4_t* from = z + logits_at((int64_t)s * tiles + tile, w) + lane;
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      f32x4_t x[2][8];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = from[((j + k) * 8 + i) * 64];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc.v[i][j + k] += x[k][i];
    }
  }
  if (q > 0)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) lds[((q - 1) * 32 + j * 8 + i) * 64 + lane] = acc.v[i][j];
  __syncthreads();
  if (q > 0) return false;
  for (int k = 0; k < kAddWaves - 1; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc.v[i][j] += lds[(k * 32 + j * 8 + i) * 64 + lane];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (row0 + 16 * j >= N)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc.v[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  return true;
}

template <bool kEmit, bool kHalf>
__global__ void __launch_bounds__(64 * kAddWaves)
    head_split_stats_kernel(StatsArgs s, const f32x4_t* z, int slices, int tiles, int waves) {
  const int id = blockIdx.x / waves, w = blockIdx.x - id * waves, tb = id / s.mm.tiles_a,
            ta = id - tb * s.mm.tiles_a;
  const uint16_t* unused;
  const int N = hidden_rows(s.h, &unused);
  if (tb * kMmTile + (w >> 1) * 64 >= N) return;
  const int64_t g0 = s.h.first + (int64_t)tb * kMmTile;
  const WaveEntries own(s.entries, s.K, s.mm.tiles_a, ta, g0 / kMmTile, w, threadIdx.x);
  MmAcc<false> acc;
  if (!add_logits(z, slices, tiles, id, w, tb * kMmTile + (w >> 1) * 64, N, acc)) return;
  f32x4_t factor = {};
  if constexpr (kHalf) factor = row_factors(s, N, tb, w, *s.tops.w);
  stats_epilogue<kEmit, kHalf>(s, acc, factor, N, ta, tb, w, g0, own.list, own.e0, own.e1,
                               own.first);
}

DPC_DEVICE float wave_max(float v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}
DPC_DEVICE float wave_sum(float v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

struct JoinArgs {
  Rows rows;
  int64_t N;
  int K, parts;
  float inv_tau, loss_scale;
  const int32_t* cols;
  const float* picked;
  const float* teacher;  // [N, K] or null (cross entropy)
  const f32x2_t* part;
  float* loss;  // at the row's own place; the others by the row's number
  float* lse;   // NaN: an entry outside the vocabulary or NaN
  float* corr;  // [rows, K]: p - sum of the q of all entries of the column
  int first;
};

// Row n by one wave, from its lse.
DPC_DEVICE void join_row(const JoinArgs& a, int64_t n, float lse, int lane) {
  const int64_t own = a.rows.active[n];
  const int32_t* cols = a.cols + n * a.K;
  const float* picked = a.picked + n * a.K;
  float* corr = a.corr + n * a.K;
  if (!a.teacher) {
    const int c = cols[0];
    if (c < 0) lse = NAN;
    const float z = c >= 0 ? picked[0] : 0.f;
    if (lane == 0) {
      a.loss[own] = (lse - z) * kLn2 * a.loss_scale;
      a.lse[n] = lse;
      corr[0] = exp2_fast(z - lse) - 1.0f;
    }
    return;
  }
  const float* teacher = a.teacher + own * a.K;
  float tm = -INFINITY;
  bool bad = false;
  for (int k = lane; k < a.K; k += 64) {
    const int c = cols[k];
    bad |= c == -2;
    if (c >= 0) {
      bad |= isnan(teacher[k]);
      tm = fmaxf(tm, teacher[k]);
    }
  }
  bad = __any(bad);
  tm = wave_max(tm);
  // Differences first: entries of any size, the type's lowest value among them, neither
  // overflow nor leave a rounding of their own.
  auto scaled = [&](int k) __attribute__((always_inline)) { return (teacher[k] - tm) * a.inv_tau; };
  float es = 0.f;
  for (int k = lane; k < a.K; k += 64)
    if (cols[k] >= 0) es += fast_exp(scaled(k));
  es = wave_sum(es);
  const float logs = logf(es);
  float loss = 0.f;
  for (int k0 = 0; k0 < a.K; k0 += 64) {
    const int k = k0 + lane;
    const int c = k < a.K ? cols[k] : -1;
    const float lq = c >= 0 ? scaled(k) - logs : -INFINITY;
    const float q = fast_exp(lq), z = c >= 0 ? picked[k] : 0.f;
    if (c >= 0 && q != 0.f) loss += q * (lq - (z - lse) * kLn2);
    // q of every entry of this column: the other entries, 64 at a time.
    float qs = 0.f;
    for (int i0 = 0; i0 < a.K; i0 += 64) {
      const int i = i0 + lane;
      const int ci = i < a.K ? cols[i] : -1;
      const float qi = ci >= 0 ? fast_exp(scaled(i) - logs) : 0.f;
      const int left = min(64, a.K - i0);
      for (int o = 0; o < left; ++o) {
        const int co = __builtin_amdgcn_readlane(ci, o);
        const float qo = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, qi), o));
        if (co == c) qs += qo;
      }
    }
    if (k < a.K) corr[k] = c >= 0 ? exp2_fast(z - lse) - qs : 0.f;
  }
  loss = wave_sum(loss);
  if (bad) lse = NAN;
  if (lane == 0) {
    a.loss[own] = bad ? NAN : loss * a.loss_scale;
    a.lse[n] = lse;
  }
}

// 16 rows a workgroup of 8 waves: their lse from the halves' statistics (16 lanes side
// by side read 16 rows), then their losses (a wave two rows).  10 us for 8192 rows of 250
// halves (1.6 TB/s; latency); 25 us with 64 entries a row, whose equal columns are found
// in K^2 / 64 steps a row.
constexpr int kJoinRows = 16, kJoinThreads = 512;

__global__ void __launch_bounds__(kJoinThreads) head_join_kernel(JoinArgs a) {
  __shared__ f32x2_t stats[kJoinThreads];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t n0 = a.first + (int64_t)blockIdx.x * kJoinRows, count = *a.rows.count;
  if (n0 >= count) return;
  const int rows = (int)(count - n0 < kJoinRows ? count - n0 : kJoinRows);
  const f32x2_t* part = a.part + n0 + min(tid & 15, rows - 1);
  float m = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int i = tid >> 4; i < a.parts; i += kJoinThreads / 16) {
    const f32x2_t x = part[i * a.N];
    const float nm = fmaxf(m, x.x), base = nm == -INFINITY ? 0.f : nm;
    sum = sum * exp2_fast(m - base) + x.y * exp2_fast(x.x - base);
    m = nm;
  }
  stats[tid] = f32x2_t{m, sum};
  __syncthreads();
  for (int k = w; k < rows; k += kJoinThreads / 64) {
    const f32x2_t x = lane < 32 ? stats[lane * 16 + k] : f32x2_t{-INFINITY, 0.f};
    const float top = wave_max(x.x), base = top == -INFINITY ? 0.f : top;
    join_row(a, n0 + k, top + log2f(wave_sum(x.y * exp2_fast(x.x - base))), lane);
  }
}

// exp(z - half's maximum) times exp(half's maximum - lse), and p - q at the entries'
// columns.  Memory bounds it: 8192 x 32000 in place, 1.05 GB, 197 us (5.3 TB/s).  16 rows
// x 8 tiles a workgroup.  The 16 rows are 1 KiB of every
// 32 columns; a wave takes one of each tile's eight, all its loads in flight at once.
constexpr int kFixTiles = 8;

struct FixArgs {
  const int32_t* count;
  int64_t N;
  int K, tiles, first;
  const int32_t* cols;
  const f32x2_t* part;
  const float* lse;
  const float* corr;
  const float* g;  // [rows] to be multiplied by, or null
  const uint16_t* e;
  uint16_t* out;   // may be e
  int64_t lde, plane;
};

template <bool kHalf>
__global__ void __launch_bounds__(kJoinThreads) head_fix_kernel(FixArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int local = blockIdx.x * kJoinRows;  // first row in the chunk
  const int64_t n0 = a.first + local, count = *a.count;
  // Rows past the last are zeros as far as a K step of dW reads.
  if (n0 >= (count + kMmStep - 1) / kMmStep * kMmStep) return;
  const int rows = max(0, (int)(count - n0 < kJoinRows ? count - n0 : kJoinRows));
  const int t0 = blockIdx.y * kFixTiles, tiles = min(kFixTiles, a.tiles - t0);
  typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
  const int64_t block = (local >> 8) * a.lde * kMmBlock + ((local & 255) >> 4) * 512;
  const int64_t at = block + (4 * t0 + (w >> 1)) * kMmBlock + (w & 1) * 8192 + lane * 8;
  const bool live = (lane & 15) < rows;
  const int64_t n = n0 + min(lane & 15, rows - 1);
  const f32x2_t* top = a.part + (2 * t0 + (w >> 2)) * a.N + n;
  const float lse = a.lse[n], g = a.g ? a.g[n] : 1.f;
  constexpr int kPlanes = kHalf ? 2 : 1;
  half8_t h[kFixTiles][kPlanes];
  float f[kFixTiles];
#pragma unroll
  for (int t = 0; t < kFixTiles; ++t)
    if (t < tiles) {
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl)
        h[t][pl] = *reinterpret_cast<const half8_t*>(a.e + at + pl * a.plane + 4 * t * kMmBlock);
      f[t] = top[2 * t * a.N].x;
    }
#pragma unroll
  for (int t = 0; t < kFixTiles; ++t)
    if (t < tiles) {
      const float x = exp2_fast(f[t] - lse) * (kHalf ? g : g / kDzScale);
      uint16_t* to = a.out + at + 4 * t * kMmBlock;
      if constexpr (kHalf) {
        half8_t o[2];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = live ? ((float)h[t][1][e] + (float)h[t][0][e]) * x : 0.f;
#pragma unroll
          for (int pl = 0; pl < 2; ++pl) o[pl][e] = __builtin_bit_cast(_Float16, half_plane(y, pl));
        }
        *reinterpret_cast<half8_t*>(to) = o[0];
        *reinterpret_cast<half8_t*>(to + a.plane) = o[1];
      } else {
        u32x4_t o;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[e] = live ? f32x2_to_bf16x2_bits((float)h[t][0][2 * e] * x,
                                             (float)h[t][0][2 * e + 1] * x)
                      : 0u;
        *reinterpret_cast<u32x4_t*>(to) = o;
      }
    }
  __syncthreads();
  for (int i = tid; i < rows * a.K; i += kJoinThreads) {
    const int c = a.cols[n0 * a.K + i];
    if (c >= 0 && (c >> 8) >= t0 && (c >> 8) < t0 + tiles) {
      const int r = i / a.K;
      uint16_t* to = a.out + block + (c >> 6) * kMmBlock + ((c >> 5) & 1) * 8192 +
                     ((c >> 2) & 3) * 128 + r * 8 + ((c >> 4) & 1) * 4 + (c & 3);
      const float x = a.corr[n0 * a.K + i] * (a.g ? a.g[n0 + r] : 1.f);
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl)
        to[pl * a.plane] = kHalf ? half_plane(ldexpf(x, kDzShift), pl) : f32_to_bf16_bits(x);
    }
  }
}

// out row n = unit's row place[n] times g[n] coef; 0 without a target.  16384 x 2048 into
// bf16: 201 MB, 31 us (6.4 TB/s).
__global__ void __launch_bounds__(256) head_scale_kernel(const float* __restrict__ unit, Rows rows,
                                                         const float* __restrict__ g, float coef,
                                                         int64_t N, int D, int out_bf16,
                                                         void* __restrict__ out) {
  const int64_t t0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  if (D % 8 == 0) {
    const int chunks = D / 8;
    for (int64_t i = t0; i < N * chunks; i += step) {
      const int64_t n = i / chunks;
      const int c = (int)(i - n * chunks) * 8;
      const int at = rows.place[n];
      f32x4_t x = {0.f, 0.f, 0.f, 0.f}, y = x;
      if (at >= 0) {
        const float f = g[n] * coef;
        const f32x4_t* u = reinterpret_cast<const f32x4_t*>(unit + (int64_t)at * D + c);
        x = u[0] * f;
        y = u[1] * f;
      }
      if (out_bf16) {
        *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(out) + n * D + c) =
            u32x4_t{f32x2_to_bf16x2_bits(x[0], x[1]), f32x2_to_bf16x2_bits(x[2], x[3]),
                    f32x2_to_bf16x2_bits(y[0], y[1]), f32x2_to_bf16x2_bits(y[2], y[3])};
      } else {
        f32x4_t* o = reinterpret_cast<f32x4_t*>(static_cast<float*>(out) + n * D + c);
        o[0] = x;
        o[1] = y;
      }
    }
  } else {
    for (int64_t i = t0; i < N * D; i += step) {
      const int64_t n = i / D;
      const int at = rows.place[n];
      const float x = at < 0 ? 0.f : unit[at * (int64_t)D + (i - n * D)] * (g[n] * coef);
      if (out_bf16)
        static_cast<uint16_t*>(out)[i] = f32_to_bf16_bits(x);
      else
        static_cast<float*>(out)[i] = x;
    }
  }
}

// ---------------------------------------------------------------------------
// Backward: dz of one piece of the vocabulary.
// ---------------------------------------------------------------------------

// The stats kernel's tiles again, with another epilogue: 16384 rows, 2048 wide, 16000 of
// the vocabulary's columns take 834 us (1.29 PFLOP/s; the K loop's bound).
struct GradArgs {
  MmArgs mm;  // A = W from the piece's first row, B = H
  Hidden h;
  int V, K, tile0, tiles;  // the piece's first tile; tiles of the vocabulary
  float inv_tau;
  Entries entries;
  const float* corr;
  const float* lse;
  const float* g;     // [rows]: the losses' gradient over the largest: bf16's dz is held over
                      // that, so a gradient that is the same for all rows (one over the
                      // tokens) is not rounded with every value.  (float32: dz is held
                      // without a gradient, which dH's rows and dW's H carry.)
  Tops tops;
  uint16_t* dz;       // [planes], native order
  int64_t ld, plane;  // blocks of a row of them, elements
};

// dz at an entry's column.
template <bool kHalf>
DPC_DEVICE float entry_change(const GradArgs& s, int tb, uint2 x) {
  const float c = s.corr[(int64_t)tb * kMmTile * s.K + x.x];
  return kHalf ? ldexpf(c, kDzShift) : c * s.g[tb * kMmTile + (x.y >> 8)];
}

template <bool kHalf>
DPC_DEVICE void grad_epilogue(const GradArgs& s, MmAcc<false>& acc, int ta, int tb, int w,
                              const f32x4_t& lse, const f32x4_t& g, const uint2* list, int e0,
                              int e1, uint2 first, float change) {
#pragma clang fp contract(off)  // the forward's rounded logit
  const int lane = epilogue_lane(), wm = w & 1, wn = w >> 1;
  const int vt = s.tile0 + ta;
  const int vleft = s.V - vt * kMmTile - wm * 128 - 4 * (lane >> 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // g, float32: what the products are to be multiplied by.
    const float c = kHalf ? g[j] : s.inv_tau;
    const float by = kHalf ? ldexpf(1.f, kDzShift) : g[j];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc.v[i][j][r] = exp2_fast(acc.v[i][j][r] * c - lse[j]) * by;
  }
  if ((vt + 1) * kMmTile > s.V) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * i + r >= vleft) acc.v[i][j][r] = 0.f;
  }
  uint16_t* out = s.dz + (tb * s.ld + 4 * ta + 2 * wm) * kMmBlock + wn * 2048 + lane * 8;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      uint16_t* at = out + (p >> 1) * kMmBlock + (p & 1) * 8192 + j * 512;
      const f32x4_t x = acc.v[2 * p][j], y = acc.v[2 * p + 1][j];
      if (!kHalf) {
        *reinterpret_cast<u32x4_t*>(at) =
            u32x4_t{f32x2_to_bf16x2_bits(x[0], x[1]), f32x2_to_bf16x2_bits(x[2], x[3]),
                    f32x2_to_bf16x2_bits(y[0], y[1]), f32x2_to_bf16x2_bits(y[2], y[3])};
      } else {
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) {
          u32x4_t o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x4_t& z = e < 2 ? x : y;
            const float lo = z[2 * (e & 1)], hi = z[2 * (e & 1) + 1];
            o[e] = half_plane(lo, pl) | ((uint32_t)half_plane(hi, pl) << 16);
          }
          *reinterpret_cast<u32x4_t*>(at + pl * s.plane) = o;
        }
      }
    }
  // Entries: put in place by the lane that stored the value.
  for (int e = e0; e < e1; e += 64) {
    uint2 x = first;
    float d = change;
    if (e > e0) {
      x = list[min(e + lane, e1 - 1)];
      d = entry_change<kHalf>(s, tb, x);
    }
    const int here = min(e1 - e, 64);
    for (int i = 0; i < here; ++i) {
      const uint32_t y = __builtin_amdgcn_readlane(x.y, i);
      const float v =
          __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, d), i));
      const int c = y & 127, j = (y >> 12) & 3;
      uint16_t* at = out + (c >> 6) * kMmBlock + ((c >> 5) & 1) * 8192 + j * 512 +
                     ((c >> 4) & 1) * 4 + (c & 3);
      if (lane == (int)(((y >> 8) & 15) | ((y >> 2) & 3) << 4)) {
#pragma unroll
        for (int pl = 0; pl < (kHalf ? 2 : 1); ++pl)
          at[pl * s.plane] = kHalf ? half_plane(v, pl) : f32_to_bf16_bits(v);
      }
    }
  }
}

// What the epilogue needs of the wave's rows.
struct GradRows {
  f32x4_t lse, g;
  template <bool kHalf>
  DPC_DEVICE void load(const GradArgs& s, int N, int tb, int w, uint32_t top_w) {
    const int lane = epilogue_lane();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = tb * kMmTile + (w >> 1) * 64 + 16 * j + (lane & 15);
      lse[j] = n < N ? s.lse[n] : 0.f;
      if constexpr (kHalf)
        g[j] = logit_factor(s.inv_tau, n < N ? s.tops.row[n] : 0u, top_w);
      else
        g[j] = n < N ? s.g[n] : 0.f;
    }
  }
};

template <bool kHalf>
__global__ void __launch_bounds__(kMmThreads, 1) head_grad_kernel(GradArgs s) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int N = hidden_rows(s.h, &s.mm.b.p);
  s.mm.b.rows = N;
  s.mm.tiles_b = tiles_of(N);
  MmTile<true, true, false, false, kHalf> tile(s.mm, lds_all);
  MmAcc<false> acc;
  const uint32_t top_w = kHalf ? *s.tops.w : 0u;
  int split, ta, tb, ta2, tb2, id = blockIdx.x;
  bool more = mm_tile_of(s.mm, id, &split, &ta2, &tb2);
  if (more) tile.begin(ta2, tb2, 0);
  while (more) {
    ta = ta2;
    tb = tb2;
    WaveEntries own(s.entries, s.K, s.tiles, s.tile0 + ta, tb, w, lane);
    tile.run(acc);
    GradRows rows;
    float change = own.e0 < own.e1 ? entry_change<kHalf>(s, tb, own.first) : 0.f;
    rows.load<kHalf>(s, N, tb, w, top_w);
    arrived(own.first.x);
    arrived(own.first.y);
    arrived(rows.lse);
    arrived(rows.g);
    arrived(change);
    id += gridDim.x;
    more = mm_tile_of(s.mm, id, &split, &ta2, &tb2);
    if (more) tile.begin(ta2, tb2, 0);
    grad_epilogue<kHalf>(s, acc, ta, tb, w, rows.lse, rows.g, own.list, own.e0, own.e1, own.first,
                         change);
  }
}

// ---------------------------------------------------------------------------
// The products with dz: out[b][a] = sum_k A(a, k) B(b, k).
// ---------------------------------------------------------------------------

struct ProductArgs {
  MmArgs mm;
  Hidden h;         // dH: the rows of B and of the output; dW: A and its K
  const int32_t* active;  // dH straight to out: the rows' own places, or null
  int rows_b;       // dW: the output's rows
  int rows_a;       // the output's row length
  float* partial;   // [splits][rows][lda] float32, or null: straight to out
  int64_t plane;    // dW: a slice of it, elements
  int64_t steps;    // dH: the K steps that the number of slices goes by, on the device:
                    // the rows that have a target are known there
  bool direct;      // dH: one slice goes straight to out
  int64_t lda;      // rows_a rounded up to 4
  int accumulate;   // add to what partial holds
  // Straight to out: multiplied by *scale (null: 1), by the row's by_row (null: 1; by the
  // rows' numbers) and by coef.
  const float* scale;
  const float* by_row;
  float coef;
  const uint32_t* shift;  // float32: the magnitude that A's planes were shifted by
  void* out;
  int out_bf16;
};

// What undoes the shifts of dz and of a product's other operand.
DPC_DEVICE int product_shift(const uint32_t* top) {
  return top ? -(kDzShift + half_shift(*top)) : 0;
}
template <bool kHidden>
DPC_DEVICE void product_epilogue(const ProductArgs& s, MmAcc<kHidden>& acc, int ta, int tb, int w,
                                 int split, int rows_b, float all, int shift) {
  const int lane = epilogue_lane();
  const int a0 = ta * kMmTile + acc.row0(w) + 4 * (lane >> 4);
  const int b0 = tb * kMmTile + acc.col0(w) + (lane & 15);
  const bool whole = s.rows_a % 4 == 0;
#pragma unroll
  for (int j = 0; j < MmAcc<kHidden>::kB; ++j) {
    const int b = b0 + 16 * j;
    if (b >= rows_b) continue;
    const float f = kHidden && s.by_row ? all * s.by_row[b] : all;
    const int64_t row = kHidden && s.active && !s.partial ? s.active[b] : b;
#pragma unroll
    for (int i = 0; i < MmAcc<kHidden>::kA; ++i) {
      const int a = a0 + 16 * i;
      if (a >= s.rows_a) continue;
      f32x4_t x = acc.v[i][j];
      if (s.partial) {
        f32x4_t* p = reinterpret_cast<f32x4_t*>(s.partial + split * s.plane + row * s.lda + a);
        if (s.accumulate) x += *p;
        *p = x;
      } else {
        store_row4(s.out, row * s.rows_a + a, s.rows_a - a, whole, s.out_bf16,
                   shifted(x, shift) * f);
      }
    }
  }
}

// 8192 rows, 2048 wide, vocabulary 32000: dH 820 us, dW 828 (1.30 PFLOP/s; the K loop's
// bound).  kHidden: dH (A = W, K the vocabulary, B = dz by rows); else dW (A = H, K the rows,
// B = dz by columns).
template <bool kHidden, bool kHalf>
__global__ void __launch_bounds__(kMmThreads, 1) head_product_kernel(ProductArgs s) {
  int split, ta, tb;
  const uint16_t* hp;
  const int count = hidden_rows(s.h, &hp);
  int rows_b = s.rows_b;
  if (kHidden) {
    rows_b = s.mm.b.rows = count;
    s.mm.tiles_b = tiles_of(count);
    if (count == 0) return;
    s.mm.splits = s.partial ? __builtin_amdgcn_readfirstlane(
                                  slices((int64_t)s.mm.tiles_a * s.mm.tiles_b, s.steps))
                            : 1;
    s.plane = count * s.lda;
    if (s.mm.splits == 1 && s.direct) s.partial = nullptr;
  } else {
    s.mm.a.p = hp;
    s.mm.kl = count;
  }
  MmTile<false, kHidden, true, kHidden, kHalf> tile(s.mm, lds_all);
  MmAcc<kHidden> acc;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float all = (s.scale ? *s.scale : 1.f) * s.coef;
  const int shift = kHalf ? product_shift(s.shift) : 0;
  int split2, ta2, tb2, id = blockIdx.x;
  bool more = mm_tile_of(s.mm, id, &split2, &ta2, &tb2);
  if (more) tile.begin(ta2, tb2, split2);
  while (more) {
    split = split2;
    ta = ta2;
    tb = tb2;
    tile.run(acc);
    // dW: tile after tile, as the logits' (2 to 5% of it).  dH's tiles are a round at most
    // but for the longest batches, and its epilogue has loads of its own.
    id += gridDim.x;
    more = !kHidden && mm_tile_of(s.mm, id, &split2, &ta2, &tb2);
    if (more) tile.begin(ta2, tb2, split2);
    product_epilogue<kHidden>(s, acc, ta, tb, w, split, rows_b, all, shift);
  }
}

// The slices of partial added up in order, multiplied as a product's own output: row r
// to out's row active[r] (or r).
struct ReduceArgs {
  const float* partial;
  int splits;
  int64_t plane, rows, lda;
  // dH: clamp(*count - first, 0, rows) rows, and the product's slices of them.
  const int32_t* count;
  int first, tiles_d;
  int64_t steps;
  bool direct;
  const int32_t* active;
  const float* scale;
  const float* by_row;
  float coef;
  const uint32_t* shift;
  int D;
  void* out;
  int out_bf16;
};

__global__ void __launch_bounds__(256) head_reduce_kernel(ReduceArgs a) {
  const int64_t quads = a.lda / 4;
  int64_t rows = a.rows;
  if (a.count) {
    const int64_t left = (int64_t)*a.count - a.first;
    rows = left < 0 ? 0 : (left < rows ? left : rows);
    if (rows == 0) return;
    a.splits = slices((int64_t)a.tiles_d * tiles_of((int)rows), a.steps);
    if (a.splits == 1 && a.direct) return;
    a.plane = rows * a.lda;
  }
  const float all = (a.scale ? *a.scale : 1.f) * a.coef;
  const int shift = product_shift(a.shift);
  const bool whole = a.D % 4 == 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * quads;
       i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / quads;
    const int c = (int)(i - row * quads) * 4;
    f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.partial + row * a.lda + c);
    for (int s = 1; s < a.splits; ++s)
      x += *reinterpret_cast<const f32x4_t*>(a.partial + s * a.plane + row * a.lda + c);
    store_row4(a.out, (a.active ? a.active[row] : row) * (int64_t)a.D + c, a.D - c, whole,
               a.out_bf16, shifted(x, shift) * (a.by_row ? all * a.by_row[row] : all));
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// Held at once: dz of a piece of the vocabulary, or a chunk's exponentials.
constexpr int64_t kPieceBytes = 512ll << 20;

// The logits' K steps in slices where their tiles leave compute units idle.  A step
// takes 1.2 us, the second launch 13 us and 0.6 us a slice of a tile's 256 rows: as many
// slices as make the sum least, if that beats the steps in a row.  (The loss of 675 rows
// with a third of them active, 1536 wide, vocabulary 203, float32: 72 steps of one tile
// take 51 us a call in 12 slices and 114 in one.)
int logit_slices(int64_t tiles, int64_t steps, int64_t N) {
  const int64_t rows = N < kMmTile ? N : kMmTile;
  int64_t s = (int64_t)sqrt(2.0 * (double)steps * kMmTile / (double)rows);
  if (s > kUnits / tiles) s = kUnits / tiles;
  if (s > steps / 4) s = steps / 4;
  return s < 2 || 1.2 * (double)(steps - steps / s) < 13.0 + 0.6 * (double)(s * rows) / kMmTile
             ? 1
             : (int)s;
}

bool valid_head(int64_t N, int D, int V, int K, int dtype) {
  return N >= 0 && N <= 0x7fffff00ll && D >= 1 && D <= (1 << 20) && V >= 1 &&
         V <= kMaxTiles * kMmTile && K >= 1 && K <= (1 << 16) &&
         (dtype == DPC_F32 || dtype == DPC_BF16);
}

// What a call needs and where it lies.
struct Plan {
  int64_t N;
  int D, V, K, dtype, planes;
  bool want_h, want_w, emit;
  int64_t ld;  // of the operands as the tiles read them
  bool pack;
  int tiles_v, tiles_n, tiles_d;
  int64_t lda;
  int chunk;                     // emit: rows of a chunk
  int64_t steps_h;               // of dH's products
  int piece_tiles, pieces;       // backward
  int splits_w, splits_z;
  bool held;  // dz for g = 1 is kept in the state
  // Byte offsets: state (kept for the backward), workspaces.
  int64_t s_rows, s_tops, s_lse, s_corr, s_list, s_start, s_cols, s_part, s_unit, s_e,
      state_bytes;
  int64_t f_rows, f_tops, f_lse, f_corr, f_list, f_start, f_cols, f_h, f_w, f_picked, f_part, f_e,
      f_pc, f_z, fwd_bytes;
  int64_t b_h, b_w, b_hg, b_g, b_dz, b_ph, b_pw, bwd_bytes;
};

// Rows of all slices together of a dH product, whatever number of rows has a target.
int64_t slice_rows(const Plan& p, int64_t rows) {
  const int64_t tiles = (rows + kMmTile - 1) / kMmTile, most = kMostSliced / p.tiles_d;
  return (most < 32 * tiles ? most : 32 * tiles) * kMmTile;
}

Plan head_plan(int64_t N, int D, int V, int K, int dtype, int want_h, int want_w) {
  Plan p = {};
  p.N = N;
  p.D = D;
  p.V = V;
  p.K = K;
  p.dtype = dtype;
  p.planes = dtype == DPC_F32 ? 2 : 1;
  p.want_h = want_h != 0;
  p.want_w = want_w != 0;
  // The logits' tiles read 128 bytes of a row at a time: rows of whole 128-byte lines are
  // read faster, and copies have them.  bf16 of other widths is copied where the tokens are
  // many.  (1000 wide, vocabulary 32000: the logits of 8192 rows take 617 us read as they
  // are and 510 from a copy, of 4096 rows 324 and 275; the copy takes 25, and a trained
  // head makes it twice.  Below 256 wide a row is 4 lines at most: 16384 rows, 264 wide, a
  // frozen head 1450 us and 1409 in all, a trained one 1834 and 1803; 200 wide 1236 and
  // 1249, 1384 and 1366; vocabulary 4000, 200 wide, the loss alone 64 and 71.)
  p.pack = dtype == DPC_F32 || D % 8 != 0 ||
           (D % 64 != 0 && D >= 256 && N >= (want_w ? 8192 : 4096));
  p.ld = up(D, p.pack && D >= 256 ? 64 : 8);
  p.tiles_v = (V + kMmTile - 1) / kMmTile;
  p.tiles_n = (int)((N + kMmTile - 1) / kMmTile);
  p.tiles_d = (D + kMmTile - 1) / kMmTile;
  p.lda = up(D, 4);
  const int64_t row_bytes = p.planes * (int64_t)p.tiles_v * kMmTile * 2;  // of dz
  p.held = p.want_w && p.tiles_n * kMmTile * row_bytes <= kPieceBytes;
  p.emit = (p.held && p.planes == 2) || (p.want_h && !p.want_w);
  const int pairs = p.planes == 1 ? 1 : 3;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  const int64_t rows_b = (2 * N + 1) * 4, lse_b = N * 4, corr_b = N * K * 4, list_b = N * K * 8,
                start_b = (int64_t)p.tiles_n * (8 * p.tiles_v + 1) * 4;
  const bool keep = (p.want_h || p.want_w) && !p.emit;
  if (p.want_h || p.want_w) {
    p.s_rows = take(rows_b);
    p.s_tops = take(8 + N * 4);
  }
  if (keep) {
    p.s_lse = take(lse_b);
    p.s_corr = take(corr_b);
    p.s_list = take(list_b);
    p.s_start = take(start_b);
  }
  if (keep && p.held) {
    p.s_cols = take(N * K * 4);
    p.s_part = take(N * p.tiles_v * 16);
  }
  if (p.emit && p.want_h) p.s_unit = take(N * D * 4);
  if (p.held) p.s_e = take(p.tiles_n * kMmTile * row_bytes);
  p.state_bytes = at;
  at = 0;
  if (!p.want_h && !p.want_w) {
    p.f_rows = take(rows_b);
    p.f_tops = take(8 + N * 4);
  }
  if (!keep) {
    p.f_lse = take(lse_b);
    p.f_corr = take(corr_b);
    p.f_list = take(list_b);
    p.f_start = take(start_b);
  }
  if (!(keep && p.held)) {
    p.f_cols = take(N * K * 4);
    p.f_part = take(N * p.tiles_v * 16);
  }
  p.f_h = take(p.planes * N * p.ld * 2);
  if (p.pack) p.f_w = take(p.planes * (int64_t)V * p.ld * 2);
  p.f_picked = take(N * K * 4);
  if (p.emit) {
    int64_t c = kPieceBytes / row_bytes / kMmTile * kMmTile;
    if (c < kMmTile) c = kMmTile;
    // Chunks of equal size.
    const int64_t rows = up(N, kMmTile);
    if (c > rows) c = rows;
    const int64_t n = (rows + c - 1) / c;
    p.chunk = (int)up((rows + n - 1) / n, kMmTile);
    p.steps_h = pairs * (int64_t)p.tiles_v * 4;
    if (!p.held) p.f_e = take(p.chunk * row_bytes);
    if (p.want_h && slices(p.tiles_d, p.steps_h) > 1)
      p.f_pc = take(slice_rows(p, p.chunk) * p.lda * 4);
  }
  const int64_t z_tiles = (int64_t)p.tiles_v * (p.emit ? p.chunk / kMmTile : p.tiles_n);
  p.splits_z = logit_slices(z_tiles, pairs * up(D, kMmStep) / kMmStep, N);
  if (p.splits_z > 1) p.f_z = take(p.splits_z * z_tiles * kMmTile * kMmTile * 4);
  p.fwd_bytes = at;
  at = 0;
  if (p.held && p.emit) {
    p.b_hg = take(p.planes * N * p.ld * 2);
    p.b_g = take(4 + N * 4);
    p.splits_w = slices((int64_t)p.tiles_d * p.tiles_v, pairs * ((N + 63) / 64));
    if (p.splits_w > 1) p.b_pw = take(p.splits_w * (int64_t)V * p.lda * 4);
  }
  if (keep) {
    p.b_h = take(p.planes * N * p.ld * 2);
    if (p.pack) p.b_w = take(p.planes * (int64_t)V * p.ld * 2);
    if (p.planes == 2 && p.want_w) p.b_hg = take(p.planes * N * p.ld * 2);
    p.b_g = take(4 + N * 4);
    const int64_t rows = (int64_t)p.tiles_n * kMmTile;
    int64_t t = kPieceBytes / (p.planes * rows * kMmTile * 2);
    if (t < 1) t = 1;
    if (t > p.tiles_v) t = p.tiles_v;
    p.pieces = (int)((p.tiles_v + t - 1) / t);
    p.piece_tiles = (p.tiles_v + p.pieces - 1) / p.pieces;
    p.pieces = (p.tiles_v + p.piece_tiles - 1) / p.piece_tiles;
    p.b_dz = take(p.planes * rows * p.piece_tiles * kMmTile * 2);
    if (p.want_h) {
      p.steps_h = pairs * (int64_t)p.piece_tiles * 4;
      const int64_t most = slices(p.tiles_d, p.steps_h) > 1 ? slice_rows(p, N) : 0;
      const int64_t need = p.pieces > 1 && N > most ? N : most;
      if (need) p.b_ph = take(need * p.lda * 4);
    }
    if (p.want_w) {
      p.splits_w = slices((int64_t)p.tiles_d * p.piece_tiles, pairs * ((N + 63) / 64));
      if (p.splits_w > 1)
        p.b_pw = take(p.splits_w * (int64_t)p.piece_tiles * kMmTile * p.lda * 4);
    }
  }
  p.bwd_bytes = at;
  return p;
}

Rows rows_at(uint8_t* base, int64_t N) {
  int32_t* r = reinterpret_cast<int32_t*>(base);
  return Rows{r, r + 1, r + 1 + N};
}

Tops tops_at(uint8_t* base) {
  uint32_t* r = reinterpret_cast<uint32_t*>(base);
  return Tops{r, r + 1, r + 2};
}

// The prep launch, and W and H as the tiles read them.
int operands(const Plan& p, PrepArgs& a, const void* hidden, const void* weight, uint8_t* h,
             uint8_t* w, hipStream_t s, Hidden* ho, MmOperand* wo) {
  a.hidden = hidden;
  a.weight = p.pack ? weight : nullptr;
  a.dtype = p.dtype;
  a.D = p.D;
  a.V = p.V;
  a.K = p.K;
  a.N = p.N;
  a.ld = p.ld;
  a.pack = p.pack;
  a.h = reinterpret_cast<uint16_t*>(h);
  a.w = reinterpret_cast<uint16_t*>(w);
  int64_t items = p.N * p.ld / 8;
  if (p.pack && p.V * p.ld / 8 > items) items = p.V * p.ld / 8;
  int64_t grid = (items + kPrepThreads - 1) / kPrepThreads;
  if (grid > 4096) grid = 4096;
  const size_t lds = a.blocks ? (size_t)(a.parts + 1) * 4 : 0;
  hipLaunchKernelGGL(prep_kernel, dim3((unsigned)(a.blocks + grid)), dim3(kPrepThreads), lds, s, a);
  DPC_HIP_CHECK(hipGetLastError());
  *ho = Hidden{p.pack ? nullptr : static_cast<const uint16_t*>(hidden), a.h, a.rows.count, p.N,
               p.ld, 0, (int)p.N};
  *wo = MmOperand{p.pack ? a.w : static_cast<const uint16_t*>(weight), p.ld, (int64_t)p.V * p.ld,
                  p.V};
  return DPC_OK;
}

int reduce(const ReduceArgs& a, hipStream_t s) {
  int64_t grid = (a.rows * (a.lda / 4) + 255) / 256;
  if (grid > 2048) grid = 2048;  // (most of dH's have nothing to add up)
  hipLaunchKernelGGL(head_reduce_kernel, dim3((unsigned)grid), dim3(256), 0, s, a);
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}

// Workgroups that go through `tiles` tiles, one a compute unit (LDS holds one).
dim3 tile_grid(int64_t tiles) { return dim3((unsigned)(tiles < kUnits ? tiles : kUnits)); }

// Workgroups of a dH product over at most tiles_n row blocks, in slices or not.
dim3 product_tiles(const Plan& p, int tiles_n) {
  int64_t most = (int64_t)p.tiles_d * tiles_n;
  for (int64_t n = p.tiles_d; n <= kUnits && n <= (int64_t)p.tiles_d * tiles_n; n += p.tiles_d) {
    const int64_t sliced = n * slices(n, p.steps_h);
    if (sliced > most) most = sliced;
  }
  return dim3((unsigned)most);
}

// Waves of a tile that may have rows.
int split_waves(const Plan& p) { return 2 * (int)(((p.N < kMmTile ? p.N : kMmTile) + 63) / 64); }

// The statistics of a launch's tiles (`tiles_b` row blocks at most).
template <bool kEmit>
int stats(const Plan& p, const StatsArgs& a, int tiles_b, f32x4_t* z, hipStream_t s) {
  const bool half = p.planes == 2;
  const int64_t tiles = (int64_t)p.tiles_v * tiles_b;
  if (p.splits_z > 1) {
    LogitsArgs l = {a.mm, a.h, z, (int)tiles};
    l.mm.splits = p.splits_z;
    const dim3 grid((unsigned)(tiles * p.splits_z)), waves((unsigned)(tiles * split_waves(p)));
    if (half) {
      hipLaunchKernelGGL((head_logits_kernel<true>), grid, dim3(kMmThreads), 0, s, l);
      DPC_HIP_CHECK(hipGetLastError());
      hipLaunchKernelGGL((head_split_stats_kernel<kEmit, true>), waves, dim3(64 * kAddWaves), 0, s,
                         a, z, p.splits_z, (int)tiles, split_waves(p));
    } else {
      hipLaunchKernelGGL((head_logits_kernel<false>), grid, dim3(kMmThreads), 0, s, l);
      DPC_HIP_CHECK(hipGetLastError());
      hipLaunchKernelGGL((head_split_stats_kernel<kEmit, false>), waves, dim3(64 * kAddWaves), 0, s,
                         a, z, p.splits_z, (int)tiles, split_waves(p));
    }
  } else if (half) {
    hipLaunchKernelGGL((head_stats_kernel<kEmit, true>), tile_grid(tiles), dim3(kMmThreads), 0, s,
                       a);
  } else {
    hipLaunchKernelGGL((head_stats_kernel<kEmit, false>), tile_grid(tiles), dim3(kMmThreads), 0, s,
                       a);
  }
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}

int fix(const Plan& p, const FixArgs& a, int64_t rows, hipStream_t s) {
  const dim3 grid((unsigned)(rows / kJoinRows),
                  (unsigned)((p.tiles_v + kFixTiles - 1) / kFixTiles));
  if (p.planes == 1)
    hipLaunchKernelGGL((head_fix_kernel<false>), grid, dim3(kJoinThreads), 0, s, a);
  else
    hipLaunchKernelGGL((head_fix_kernel<true>), grid, dim3(kJoinThreads), 0, s, a);
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}

// dW's rows of a piece of the vocabulary (`cols` of them, in `tiles`) from its dz, and H.
int weight_product(const Plan& p, const PrepArgs& g, const Hidden& h, const MmOperand& dz,
                   const Tops& tops, int cols, int tiles, float coef, float* partial,
                   void* out, hipStream_t s) {
  const bool half = p.planes == 2;
  ProductArgs m = {};
  m.mm = MmArgs{MmOperand{nullptr, p.ld, p.N * p.ld, 0}, dz, 0, p.tiles_d, tiles, p.splits_w};
  m.h = h;
  m.rows_a = p.D;
  m.rows_b = cols;
  m.lda = p.lda;
  m.plane = (int64_t)cols * p.lda;
  m.scale = g.gmax;
  m.coef = coef;
  m.shift = half ? tops.h : nullptr;
  m.partial = p.splits_w == 1 ? nullptr : partial;
  m.out = out;
  m.out_bf16 = p.dtype == DPC_BF16;
  const dim3 grid = tile_grid((int64_t)p.tiles_d * tiles * p.splits_w);
  if (half)
    hipLaunchKernelGGL((head_product_kernel<false, true>), grid, dim3(kMmThreads), 0, s, m);
  else
    hipLaunchKernelGGL((head_product_kernel<false, false>), grid, dim3(kMmThreads), 0, s, m);
  DPC_HIP_CHECK(hipGetLastError());
  if (!m.partial) return DPC_OK;
  ReduceArgs r = {};
  r.partial = m.partial;
  r.splits = p.splits_w;
  r.plane = m.plane;
  r.rows = cols;
  r.lda = p.lda;
  r.scale = m.scale;
  r.coef = coef;
  r.shift = m.shift;
  r.D = p.D;
  r.out_bf16 = m.out_bf16;
  r.out = out;
  return reduce(r, s);
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// (Its square and its reciprocal are taken in float32.)
bool valid_temperature(double t) { return t > 1e-15 && t < 1e15; }

}  // namespace

extern "C" size_t dpc_head_loss_state_bytes(int64_t N, int D, int V, int K, int dtype,
                                            int want_hidden, int want_weight) {
  if (!valid_head(N, D, V, K, dtype) || N == 0) return 0;
  return (size_t)head_plan(N, D, V, K, dtype, want_hidden, want_weight).state_bytes;
}

extern "C" size_t dpc_head_loss_workspace_bytes(int64_t N, int D, int V, int K, int dtype,
                                                int want_hidden, int want_weight) {
  if (!valid_head(N, D, V, K, dtype) || N == 0) return 0;
  return (size_t)head_plan(N, D, V, K, dtype, want_hidden, want_weight).fwd_bytes;
}

extern "C" size_t dpc_head_loss_grad_workspace_bytes(int64_t N, int D, int V, int K, int dtype,
                                                     int want_hidden, int want_weight) {
  if (!valid_head(N, D, V, K, dtype) || N == 0) return 0;
  return (size_t)head_plan(N, D, V, K, dtype, want_hidden, want_weight).bwd_bytes;
}

extern "C" int dpc_head_loss(const void* hidden, const void* weight, int64_t N, int D, int V,
                             int dtype, const int64_t* index, const float* teacher, int K,
                             int64_t ignore_index, double temperature, int want_hidden,
                             int want_weight, float* loss, void* state, size_t state_bytes,
                             void* ws, size_t ws_bytes, void* stream) {
  if (!valid_head(N, D, V, K, dtype) || !valid_temperature(temperature)) return DPC_EINVAL;
  if (!teacher && K != 1) return DPC_EINVAL;
  if (N == 0) return DPC_OK;
  if (!hidden || !weight || !index || !loss || !ws) return DPC_EINVAL;
  const Plan p = head_plan(N, D, V, K, dtype, want_hidden, want_weight);
  if (!p.pack && (misaligned(hidden) || misaligned(weight))) return DPC_EINVAL;
  if (p.state_bytes && (!state || misaligned(state))) return DPC_EINVAL;
  if (misaligned(ws)) return DPC_EINVAL;
  if (ws_bytes < (size_t)p.fwd_bytes || state_bytes < (size_t)p.state_bytes) return DPC_ENOSPC;
  if ((int64_t)p.tiles_v * p.tiles_n > 0x7fffffffll) return DPC_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  uint8_t* base = static_cast<uint8_t*>(ws);
  uint8_t* kept = static_cast<uint8_t*>(state);
  const bool any = p.want_h || p.want_w, keep = any && !p.emit;
  auto place = [&](bool in_state, int64_t so, int64_t fo) {
    return in_state ? kept + so : base + fo;
  };
  const Rows rows = rows_at(place(any, p.s_rows, p.f_rows), N);
  const Tops tops = tops_at(place(any, p.s_tops, p.f_tops));
  const bool held = keep && p.held;  // bf16: the backward makes dz of the exponentials
  const Entries entries = {reinterpret_cast<int32_t*>(place(held, p.s_cols, p.f_cols)),
                           reinterpret_cast<uint2*>(place(keep, p.s_list, p.f_list)),
                           reinterpret_cast<int32_t*>(place(keep, p.s_start, p.f_start))};
  float* lse = reinterpret_cast<float*>(place(keep, p.s_lse, p.f_lse));
  float* corr = reinterpret_cast<float*>(place(keep, p.s_corr, p.f_corr));
  if (teacher) {
    hipLaunchKernelGGL(entries_kernel, dim3((unsigned)((N + 3) / 4)), dim3(256), 0, s, index,
                       teacher, N, K, V, rows.place);
    DPC_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(1024), 0, s, index, ignore_index,
                     teacher != nullptr, N, rows, loss, tops);
  DPC_HIP_CHECK(hipGetLastError());
  if (dtype == DPC_F32) {
    hipLaunchKernelGGL(tops_kernel, dim3(256, 2), dim3(256), 0, s,
                       static_cast<const float*>(hidden), static_cast<const float*>(weight), D, V,
                       rows, tops);
    DPC_HIP_CHECK(hipGetLastError());
  }
  PrepArgs q = {};
  q.rows = rows;
  q.tops = tops;
  q.index = index;
  q.teacher = teacher != nullptr;
  q.blocks = p.tiles_n;
  q.parts = 8 * p.tiles_v;
  q.entries = entries;
  StatsArgs a = {};
  const int rc = operands(p, q, hidden, weight, base + p.f_h, base + p.f_w, s, &a.h, &a.mm.a);
  if (rc != DPC_OK) return rc;
  const MmOperand w = a.mm.a;
  a.mm.b = MmOperand{nullptr, p.ld, N * p.ld, 0};
  a.mm.kl = (int)p.ld;
  a.mm.tiles_a = p.tiles_v;
  a.mm.splits = 1;
  a.V = V;
  a.K = K;
  a.inv_tau = (float)(kLog2e64 / temperature);
  a.tops = tops;
  a.entries = entries;
  a.picked = reinterpret_cast<float*>(base + p.f_picked);
  a.part = reinterpret_cast<f32x2_t*>(place(held, p.s_part, p.f_part));
  a.N = N;
  JoinArgs j = {};
  j.rows = rows;
  j.N = N;
  j.K = K;
  j.parts = 2 * p.tiles_v;
  j.inv_tau = (float)(1.0 / temperature);
  j.loss_scale = (float)(temperature * temperature);
  j.cols = entries.cols;
  j.picked = a.picked;
  j.teacher = teacher;
  j.part = a.part;
  j.loss = loss;
  j.lse = lse;
  j.corr = corr;
  f32x4_t* z = reinterpret_cast<f32x4_t*>(base + p.f_z);
  const int tiles_c = p.emit ? p.chunk / kMmTile : p.tiles_n;
  a.lde = (int64_t)p.tiles_v * 4;
  a.plane = tiles_c * a.lde * kMmBlock;
  a.e = reinterpret_cast<uint16_t*>(place(p.held, p.s_e, p.f_e));
  a.h.most = tiles_c * kMmTile;
  if (!p.emit) {
    const int rz = held ? stats<true>(p, a, tiles_c, z, s) : stats<false>(p, a, tiles_c, z, s);
    if (rz != DPC_OK) return rz;
    hipLaunchKernelGGL(head_join_kernel, dim3((unsigned)((N + kJoinRows - 1) / kJoinRows)),
                       dim3(kJoinThreads), 0, s, j);
    DPC_HIP_CHECK(hipGetLastError());
    return DPC_OK;
  }
  float* unit = reinterpret_cast<float*>(kept + p.s_unit);
  for (int64_t first = 0; first < N; first += p.chunk) {
    a.h.first = j.first = (int)first;
    const int rz = stats<true>(p, a, tiles_c, z, s);
    if (rz != DPC_OK) return rz;
    hipLaunchKernelGGL(head_join_kernel, dim3((unsigned)(p.chunk / kJoinRows)),
                       dim3(kJoinThreads), 0, s, j);
    DPC_HIP_CHECK(hipGetLastError());
    const FixArgs x = {rows.count, N, K, p.tiles_v, (int)first, entries.cols, a.part, lse, corr,
                       nullptr, a.e, a.e, a.lde, a.plane};
    const int rx = fix(p, x, p.chunk, s);
    if (rx != DPC_OK) return rx;
    if (!p.want_h) continue;
    ProductArgs m = {};
    m.mm = MmArgs{w, MmOperand{a.e, a.lde, a.plane, 0}, V, p.tiles_d, tiles_c, 1};
    m.steps = p.steps_h;
    m.direct = true;
    m.coef = 1.f;
    m.shift = p.planes == 2 ? tops.w : nullptr;
    m.h = a.h;
    m.rows_a = D;
    m.lda = p.lda;
    m.partial = p.f_pc ? reinterpret_cast<float*>(base + p.f_pc) : nullptr;
    m.out = unit + first * D;
    const dim3 product_grid = product_tiles(p, tiles_c);
    if (p.planes == 1)
      hipLaunchKernelGGL((head_product_kernel<true, false>), product_grid, dim3(kMmThreads), 0, s,
                         m);
    else
      hipLaunchKernelGGL((head_product_kernel<true, true>), product_grid, dim3(kMmThreads), 0, s,
                         m);
    DPC_HIP_CHECK(hipGetLastError());
    if (m.partial) {
      ReduceArgs r = {};
      r.partial = m.partial;
      r.tiles_d = p.tiles_d;
      r.steps = m.steps;
      r.direct = m.direct;
      r.rows = p.chunk;
      r.lda = p.lda;
      r.count = rows.count;
      r.first = (int)first;
      r.coef = 1.f;
      r.shift = m.shift;
      r.D = D;
      r.out = m.out;
      const int rr = reduce(r, s);
      if (rr != DPC_OK) return rr;
    }
  }
  return DPC_OK;
}

extern "C" int dpc_head_loss_grad(const void* hidden, const void* weight, int64_t N, int D, int V,
                                  int dtype, int K, double temperature, int want_hidden,
                                  int want_weight, const void* state, size_t state_bytes,
                                  const float* grad_loss, void* hidden_grad, void* weight_grad,
                                  void* ws, size_t ws_bytes, void* stream) {
  if (!valid_head(N, D, V, K, dtype) || !valid_temperature(temperature)) return DPC_EINVAL;
  if (N == 0) return DPC_OK;
  if (!hidden_grad && !weight_grad) return DPC_EINVAL;
  if ((hidden_grad && !want_hidden) || (weight_grad && !want_weight)) return DPC_EINVAL;
  if (!hidden || !weight || !state || !grad_loss) return DPC_EINVAL;
  const Plan p = head_plan(N, D, V, K, dtype, want_hidden, want_weight);
  if (!p.pack && (misaligned(hidden) || misaligned(weight))) return DPC_EINVAL;
  if (misaligned(hidden_grad) || misaligned(weight_grad) || misaligned(state)) return DPC_EINVAL;
  if (p.bwd_bytes && (!ws || misaligned(ws))) return DPC_EINVAL;
  if (ws_bytes < (size_t)p.bwd_bytes || state_bytes < (size_t)p.state_bytes) return DPC_ENOSPC;
  hipStream_t s = (hipStream_t)stream;
  uint8_t* base = static_cast<uint8_t*>(ws);
  uint8_t* kept = static_cast<uint8_t*>(const_cast<void*>(state));
  const Rows rows = rows_at(kept + p.s_rows, N);
  if (p.emit && hidden_grad) {
    const int64_t items = D % 8 == 0 ? N * D / 8 : N * D;
    int64_t grid = (items + 255) / 256;
    if (grid > 8192) grid = 8192;
    hipLaunchKernelGGL(head_scale_kernel, dim3((unsigned)grid), dim3(256), 0, s,
                       reinterpret_cast<const float*>(kept + p.s_unit), rows, grad_loss,
                       (float)temperature, N, D, dtype == DPC_BF16, hidden_grad);
    DPC_HIP_CHECK(hipGetLastError());
  }
  if (p.emit && !weight_grad) return DPC_OK;
  if ((int64_t)p.piece_tiles * p.tiles_n > 0x7fffffffll) return DPC_EINVAL;
  PrepArgs pa = {};
  pa.rows = rows;
  pa.g = grad_loss;
  pa.gmax = reinterpret_cast<float*>(base + p.b_g);
  pa.g_over = pa.gmax + 1;
  const Tops tops = tops_at(kept + p.s_tops);
  pa.tops = tops;
  const bool half = p.planes == 2;
  if (half) {
    hipLaunchKernelGGL(gmax_kernel, dim3(1), dim3(kPrepThreads), 0, s, pa);
    DPC_HIP_CHECK(hipGetLastError());
    pa.g = nullptr;
    if (weight_grad) pa.hg = reinterpret_cast<uint16_t*>(base + p.b_hg);
  }
  const int64_t esz = dtype == DPC_BF16 ? 2 : 4;
  if (p.emit) {
    pa.hidden = hidden;
    pa.dtype = dtype;
    pa.D = D;
    pa.N = N;
    pa.ld = p.ld;
    int64_t grid = (N * p.ld / 8 + kPrepThreads - 1) / kPrepThreads;
    if (grid > 4096) grid = 4096;
    hipLaunchKernelGGL(prep_kernel, dim3((unsigned)grid), dim3(kPrepThreads), 0, s, pa);
    DPC_HIP_CHECK(hipGetLastError());
    const int64_t ldz = (int64_t)p.tiles_v * 4;
    const MmOperand zop = {reinterpret_cast<const uint16_t*>(kept + p.s_e), ldz,
                           p.tiles_n * ldz * kMmBlock, 0};
    const Hidden h = {nullptr, pa.hg, rows.count, N, p.ld, 0, (int)N};
    return weight_product(p, pa, h, zop, tops, V, p.tiles_v, (float)temperature,
                          reinterpret_cast<float*>(base + p.b_pw), weight_grad, s);
  }
  pa.zero = hidden_grad;
  Hidden h;
  MmOperand w;
  const int rc = operands(p, pa, hidden, weight, base + p.b_h, base + p.b_w, s, &h, &w);
  if (rc != DPC_OK) return rc;
  const MmOperand hop = {nullptr, p.ld, N * p.ld, 0};
  const int out_bf16 = dtype == DPC_BF16;
  const int64_t ldz = (int64_t)p.piece_tiles * 4;
  const int64_t plane = p.tiles_n * ldz * kMmBlock;
  uint16_t* dz = reinterpret_cast<uint16_t*>(base + p.b_dz);
  for (int i = 0; i < p.pieces; ++i) {
    const int tile0 = i * p.piece_tiles, first = tile0 * kMmTile;
    const int tiles = p.tiles_v - tile0 < p.piece_tiles ? p.tiles_v - tile0 : p.piece_tiles;
    const int cols_here = V - first < tiles * kMmTile ? V - first : tiles * kMmTile;
    MmOperand wpiece = w;
    wpiece.p = w.p + (int64_t)first * w.ld;
    wpiece.rows = cols_here;
    GradArgs a = {};
    a.mm = MmArgs{wpiece, hop, (int)p.ld, tiles, p.tiles_n, 1};
    a.h = h;
    a.V = V;
    a.K = K;
    a.tile0 = tile0;
    a.tiles = p.tiles_v;
    a.inv_tau = (float)(kLog2e64 / temperature);
    a.entries = Entries{nullptr, reinterpret_cast<uint2*>(kept + p.s_list),
                        reinterpret_cast<int32_t*>(kept + p.s_start)};
    a.corr = reinterpret_cast<const float*>(kept + p.s_corr);
    a.lse = reinterpret_cast<const float*>(kept + p.s_lse);
    a.g = pa.g_over;
    a.tops = tops;
    a.dz = dz;
    a.ld = ldz;
    a.plane = plane;
    if (p.held) {
      const FixArgs x = {rows.count, N, K, p.tiles_v, 0,
                         reinterpret_cast<const int32_t*>(kept + p.s_cols),
                         reinterpret_cast<const f32x2_t*>(kept + p.s_part), a.lse, a.corr, a.g,
                         reinterpret_cast<const uint16_t*>(kept + p.s_e), dz, ldz, plane};
      const int rx = fix(p, x, (int64_t)p.tiles_n * kMmTile, s);
      if (rx != DPC_OK) return rx;
    } else {
      const dim3 grid = tile_grid((int64_t)tiles * p.tiles_n);
      if (half)
        hipLaunchKernelGGL((head_grad_kernel<true>), grid, dim3(kMmThreads), 0, s, a);
      else
        hipLaunchKernelGGL((head_grad_kernel<false>), grid, dim3(kMmThreads), 0, s, a);
      DPC_HIP_CHECK(hipGetLastError());
    }
    const MmOperand zop = {dz, ldz, plane, 0};
    ProductArgs q = {};
    q.h = h;
    q.rows_a = D;
    q.lda = p.lda;
    q.scale = pa.gmax;
    q.coef = (float)temperature;
    q.out_bf16 = out_bf16;
    ReduceArgs r = {};
    r.lda = p.lda;
    r.scale = pa.gmax;
    r.coef = q.coef;
    r.D = D;
    r.out_bf16 = out_bf16;
    if (hidden_grad) {
      // A = W (D, K-slow: a row holds one vocabulary entry), B = dz by rows.  dz is zero
      // past the vocabulary, and W's rows there read as zeros.
      ProductArgs m = q;
      m.mm = MmArgs{wpiece, zop, cols_here, p.tiles_d, p.tiles_n, 1};
      m.active = rows.active;
      m.steps = p.steps_h;
      m.direct = p.pieces == 1;
      m.partial = p.b_ph ? reinterpret_cast<float*>(base + p.b_ph) : nullptr;
      m.accumulate = i > 0;
      m.out = hidden_grad;
      m.by_row = half ? pa.g_over : nullptr;
      m.shift = half ? tops.w : nullptr;
      const dim3 product_grid = product_tiles(p, p.tiles_n);
      if (half)
        hipLaunchKernelGGL((head_product_kernel<true, true>), product_grid, dim3(kMmThreads), 0, s,
                           m);
      else
        hipLaunchKernelGGL((head_product_kernel<true, false>), product_grid, dim3(kMmThreads), 0,
                           s, m);
      DPC_HIP_CHECK(hipGetLastError());
      if (m.partial && i + 1 == p.pieces) {
        r.partial = m.partial;
        r.tiles_d = p.tiles_d;
        r.steps = m.steps;
        r.direct = m.direct;
        r.rows = N;
        r.count = rows.count;
        r.active = rows.active;
        r.by_row = m.by_row;
        r.shift = m.shift;
        r.out = hidden_grad;
        const int rr = reduce(r, s);
        if (rr != DPC_OK) return rr;
      }
    }
    if (weight_grad) {
      Hidden hw = h;
      if (half) hw.packed = pa.hg;
      const int rw = weight_product(p, pa, hw, zop, tops, cols_here, tiles,
                                    (float)temperature, reinterpret_cast<float*>(base + p.b_pw),
                                    static_cast<uint8_t*>(weight_grad) + (int64_t)first * D * esz,
                                    s);
      if (rw != DPC_OK) return rw;
    }
  }
  return DPC_OK;
}
