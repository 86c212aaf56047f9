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
// Cross entropy is the K = 1, q = 1 case, so both share every kernel.
//
// Rows without a target (the ignored index; no teacher entry above -inf) are left
// out of every product: the rows that have one are numbered on the device, and the
// kernels run over that many.  So such rows cost nothing and whatever they hold
// (padding, NaN) reaches nothing.
//
// Forward: one product whose 256 x 256 tiles never leave the chip; each leaves
// its maximum and sum of exponentials per token and the logits at the entries'
// columns; a join turns them into lse and the loss.  Backward, in pieces of the
// vocabulary: the logits' tiles again, turned into dz in the accumulators and
// written as bf16 (float32 inputs: as three bf16 planes, exact), then the two
// products dz W (added up over the pieces in float32) and dz^T H.  dz at an
// entry's column, where p and q may cancel, is formed in float32 by the join and
// put in place of the tile's value.
#include <math.h>

#include "common.h"
#include "mm_tile.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

DPC_DEVICE float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

constexpr int kLdsBytes = 131072;
__shared__ __attribute__((aligned(16))) uint8_t lds_all[kLdsBytes];

// ---------------------------------------------------------------------------
// Operands as the tiles read them.
// ---------------------------------------------------------------------------

// Plane p (0..2) of x: x0 = bf16(x), x1 = bf16(x - x0), x2 = x - x0 - x1, which
// sum to x exactly (8 + 8 + 8 bits; parts below the normal range are flushed by
// the matrix cores).  A value that rounds past the largest bf16 is truncated
// instead.  Not finite: plane 0 alone carries it.
DPC_DEVICE uint16_t split_plane(float x, int p) {
  if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) return p ? 0 : f32_to_bf16_bits(x);
  uint16_t b = 0;
  for (int i = 0; i <= p; ++i) {
    b = f32_to_bf16_bits(x);
    if ((b & 0x7f80u) == 0x7f80u) b = (uint16_t)(__float_as_uint(x) >> 16);
    x -= bf16_bits_to_f32(b);
  }
  return b;
}

// The rows that have a target, in order: count, active[count], and each row's
// place among them or -1.
struct Rows {
  int32_t* count;
  int32_t* active;
  int32_t* place;
};

Rows rows_of(int32_t* rows, int64_t N) { return Rows{rows, rows + 1, rows + 1 + N}; }

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
  if (__any(has) && lane == 0) flag[n] = 1;
  else if (!__any(has) && lane == 0) flag[n] = 0;
}

// Numbers the rows with a target, and writes the others' losses (0).  One
// workgroup; a thread takes 32 consecutive rows a round, whose flags are the bits
// of a word.  `flag` (distillation) is rows.place before it is overwritten.
__global__ void __launch_bounds__(1024) rows_kernel(const int64_t* __restrict__ index,
                                                    int64_t ignore, int flags, int64_t N,
                                                    Rows rows, float* __restrict__ loss) {
  __shared__ int wave_total[16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int64_t base = 0;
  for (int64_t r0 = 0; r0 < N; r0 += 32 * 1024) {
    const int64_t left = N - r0;
    const int per = (int)(left >= 32 * 1024 ? 32 : (left + 1023) / 1024);
    const int64_t first = r0 + (int64_t)tid * per;
    uint32_t bits = 0;
    for (int i = 0; i < per; ++i)
      if (first + i < N && (flags ? rows.place[first + i] != 0 : index[first + i] != ignore))
        bits |= 1u << i;
    const int mine = __popc(bits);
    int upto = mine;  // inclusive sum over the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 63) wave_total[w] = upto;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < 16; ++i) {
      before += i < w ? wave_total[i] : 0;
      all += wave_total[i];
    }
    int64_t at = base + before + upto - mine;
    for (int i = 0; i < per; ++i) {
      const int64_t n = first + i;
      if (n >= N) break;
      const bool on = (bits >> i) & 1;
      rows.place[n] = on ? (int32_t)at : -1;
      if (on)
        rows.active[at++] = (int32_t)n;
      else
        loss[n] = 0.f;
    }
    base += all;
    __syncthreads();
  }
  if (tid == 0) *rows.count = (int32_t)base;
}

// Operands as the tiles read them, in planes of bf16 rows padded with zeros:
// the rows with a target of `hidden` (bf16 rows of whole 16-byte chunks: only if
// some are left out, else the tiles read the caller's own) and, where the weight
// needs planes or padding, the weight.  With `index` also the entries' columns in
// 32 bits (-1: absent, -2: outside the vocabulary); with `zero` also the zero
// rows of the hidden gradient.
struct PrepArgs {
  const void* hidden;
  const void* weight;  // null: read as it is
  int dtype, D, V, K;
  int64_t N, ld;
  Rows rows;
  uint16_t* h;
  uint16_t* w;
  bool pack;
  const int64_t* index;
  bool teacher;
  int32_t* cols;
  void* zero;
};

DPC_DEVICE void pack_chunk(const void* src, int dtype, int64_t row, int D, int c, int64_t ld,
                           int64_t plane, uint16_t* dst, int64_t to) {
  const int planes = dtype == DPC_F32 ? 3 : 1;
  float x[8];
  uint16_t h[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = 0.f;
    h[e] = 0;
    if (c + e < D) {
      if (dtype == DPC_F32)
        x[e] = static_cast<const float*>(src)[row * D + c + e];
      else
        h[e] = static_cast<const uint16_t*>(src)[row * D + c + e];
    }
  }
  for (int p = 0; p < planes; ++p) {
    u32x4_t o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint16_t a = planes == 1 ? h[2 * e] : split_plane(x[2 * e], p);
      const uint16_t b = planes == 1 ? h[2 * e + 1] : split_plane(x[2 * e + 1], p);
      o[e] = (uint32_t)a | ((uint32_t)b << 16);
    }
    *reinterpret_cast<u32x4_t*>(dst + p * plane + to * ld + c) = o;
  }
}

__global__ void __launch_bounds__(256) prep_kernel(PrepArgs a) {
  const int64_t count = *a.rows.count;
  const int64_t t0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  if (a.index) {
    for (int64_t i = t0; i < count * a.K; i += step) {
      const int64_t c = i / a.K;
      const int64_t t = a.index[(int64_t)a.rows.active[c] * a.K + (i - c * a.K)];
      a.cols[i] = a.teacher && t < 0 ? -1 : (t >= 0 && t < a.V ? (int32_t)t : -2);
    }
  }
  const int64_t chunks = a.ld / 8;
  if (a.h && (a.pack || count < a.N))
    for (int64_t i = t0; i < count * chunks; i += step) {
      const int64_t c = i / chunks;
      pack_chunk(a.hidden, a.dtype, a.rows.active[c], a.D, (int)(i - c * chunks) * 8, a.ld,
                 a.N * a.ld, a.h, c);
    }
  if (a.weight)
    for (int64_t i = t0; i < a.V * chunks; i += step) {
      const int64_t v = i / chunks;
      pack_chunk(a.weight, a.dtype, v, a.D, (int)(i - v * chunks) * 8, a.ld, (int64_t)a.V * a.ld,
                 a.w, v);
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
// and needs no padding, else the packed ones; and how many.
struct Hidden {
  const uint16_t* own;  // null: always the packed rows
  const uint16_t* packed;
  const int32_t* count;
  int64_t N;
};

DPC_DEVICE int hidden_rows(const Hidden& h, const uint16_t** p) {
  const int count = __builtin_amdgcn_readfirstlane(*h.count);
  *p = h.own && count == h.N ? h.own : h.packed;
  return count;
}

DPC_DEVICE int tiles_of(int rows) { return (rows + kMmTile - 1) / kMmTile; }

// ---------------------------------------------------------------------------
// Forward: the tile's statistics and the entries' logits.
// ---------------------------------------------------------------------------

struct StatsArgs {
  MmArgs mm;  // A = W (vocabulary), B = H (rows with a target)
  Hidden h;
  int V, K;
  float inv_tau;
  const int32_t* cols;  // [rows, K]
  float* picked;        // [rows, K]: z at the entries' columns
  f32x2_t* part;        // [rows, tiles_a]: maximum and sum of exponentials of each tile
};

__global__ void __launch_bounds__(kMmThreads, 1) head_stats_kernel(StatsArgs s) {
  int split, ta, tb;
  const int N = hidden_rows(s.h, &s.mm.b.p);
  s.mm.b.rows = N;
  s.mm.tiles_b = tiles_of(N);
  if (!mm_tile_of(s.mm, &split, &ta, &tb)) return;
  MmAcc acc;
  mm_loop<true, true>(s.mm, ta, tb, 0, lds_all, acc);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wm = w & 1, wn = w >> 1;
  const int v0 = ta * kMmTile, n0 = tb * kMmTile;
  const int vl = wm * 128 + 4 * (lane >> 4);  // + 16 i + r
  const int tl = wn * 64 + (lane & 15);       // + 16 j
  const int vleft = s.V - v0 - vl;
  f32x2_t* st = reinterpret_cast<f32x2_t*>(lds_all);  // [2][256]
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float z = acc.v[i][j][r] * s.inv_tau;
        acc.v[i][j][r] = z;
        if (16 * i + r < vleft) m = fmaxf(m, z);
      }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    float sum = 0.f;
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * i + r < vleft) sum += fast_exp(acc.v[i][j][r] - base);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (lane < 16) st[wm * 256 + tl + 16 * j] = f32x2_t{m, sum};
  }
  __syncthreads();
  if (tid < kMmTile && n0 + tid < N) {
    const f32x2_t a = st[tid], b = st[256 + tid];
    const float m = fmaxf(a.x, b.x), base = m == -INFINITY ? 0.f : m;
    s.part[(int64_t)(n0 + tid) * s.mm.tiles_a + ta] =
        f32x2_t{m, a.y * fast_exp(a.x - base) + b.y * fast_exp(b.x - base)};
  }
  // Entries: the tile in float32, 128 tokens at a time, rows of 1 KiB whose
  // 16-byte chunks are XOR-swizzled by the token.
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    __syncthreads();
    if ((wn >> 1) == p) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int t = (tl + 16 * j) & 127, v = vl + 16 * i;
          *reinterpret_cast<f32x4_t*>(lds_all + t * 1024 + (((v >> 2) ^ (t & 15)) << 4)) =
              acc.v[i][j];
        }
    }
    __syncthreads();
    const int64_t first = n0 + 128 * p;
    const int64_t left = N - first;
    if (left > 0) {
      const int64_t base = first * s.K;
      const int count = (int)(left < 128 ? left : 128) * s.K;
      for (int e = tid; e < count; e += kMmThreads) {
        const int c = s.cols[base + e] - v0;
        if ((unsigned)c < (unsigned)kMmTile) {
          const int t = e / s.K;
          s.picked[base + e] = *reinterpret_cast<const float*>(
              lds_all + t * 1024 + (((c >> 2) ^ (t & 15)) << 4) + (c & 3) * 4);
        }
      }
    }
  }
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
  int K, parts;
  float inv_tau, loss_scale;
  const int32_t* cols;
  const float* picked;
  const float* teacher;  // [N, K] or null (cross entropy)
  const f32x2_t* part;
  float* loss;  // at the row's own place; the others by the row's number
  float* lse;   // NaN: an entry outside the vocabulary or NaN
  float* corr;  // [rows, K]: p - sum of the q of all entries of the column
};

// One wave a row.
__global__ void __launch_bounds__(256) head_join_kernel(JoinArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= *a.rows.count) return;
  const int64_t own = a.rows.active[n];
  const f32x2_t* part = a.part + n * a.parts;
  float m = -INFINITY, sum = 0.f;
  for (int i = lane; i < a.parts; i += 64) {
    const f32x2_t x = part[i];
    const float nm = fmaxf(m, x.x), base = nm == -INFINITY ? 0.f : nm;
    sum = sum * fast_exp(m - base) + x.y * fast_exp(x.x - base);
    m = nm;
  }
  const float top = wave_max(m), tb = top == -INFINITY ? 0.f : top;
  sum = wave_sum(sum * fast_exp(m - tb));
  float lse = top + logf(sum);
  const int32_t* cols = a.cols + n * a.K;
  const float* picked = a.picked + n * a.K;
  float* corr = a.corr + n * a.K;
  if (!a.teacher) {
    if (lane == 0) {
      const int c = cols[0];
      if (c < 0) lse = NAN;
      const float z = c >= 0 ? picked[0] : 0.f;
      a.loss[own] = (lse - z) * a.loss_scale;
      a.lse[n] = lse;
      corr[0] = fast_exp(z - lse) - 1.0f;
    }
    return;
  }
  const float* teacher = a.teacher + own * a.K;
  float tm = -INFINITY;
  bool bad = false, nan = false;
  for (int k = lane; k < a.K; k += 64) {
    const int c = cols[k];
    bad |= c == -2;
    if (c >= 0) {
      nan |= isnan(teacher[k]);
      tm = fmaxf(tm, teacher[k] * a.inv_tau);
    }
  }
  bad = __any(bad || nan);
  tm = wave_max(tm);
  float es = 0.f;
  for (int k = lane; k < a.K; k += 64)
    if (cols[k] >= 0) es += fast_exp(teacher[k] * a.inv_tau - tm);
  es = wave_sum(es);
  const float logs = logf(es);
  float loss = 0.f;
  for (int k = lane; k < a.K; k += 64) {
    const int c = cols[k];
    float out = 0.f;
    if (c >= 0) {
      const float lq = teacher[k] * a.inv_tau - tm - logs, q = fast_exp(lq);
      const float z = picked[k];
      if (q != 0.f) loss += q * (lq - (z - lse));
      float qs = 0.f;
      for (int i = 0; i < a.K; ++i)
        if (cols[i] == c) qs += fast_exp(teacher[i] * a.inv_tau - tm - logs);
      out = fast_exp(z - lse) - qs;
    }
    corr[k] = out;
  }
  loss = wave_sum(loss);
  if (lane == 0) {
    a.loss[own] = bad ? NAN : loss * a.loss_scale;
    a.lse[n] = bad ? NAN : lse;
  }
}

// ---------------------------------------------------------------------------
// Backward: dz of one piece of the vocabulary.
// ---------------------------------------------------------------------------

struct GradArgs {
  MmArgs mm;  // A = W from the piece's first row, B = H
  Hidden h;
  const int32_t* active;
  int V, K, first;  // the piece's first column
  float inv_tau, coef;
  const int32_t* cols;
  const float* corr;
  const float* lse;
  const float* g;  // [N]: the losses' gradient, at the rows' own places
  uint16_t* dz;    // [planes][rows][ld]
  int64_t ld, plane;
};

template <int kPlanes>
__global__ void __launch_bounds__(kMmThreads, 1) head_grad_kernel(GradArgs s) {
  int split, ta, tb;
  const int N = hidden_rows(s.h, &s.mm.b.p);
  s.mm.b.rows = N;
  s.mm.tiles_b = tiles_of(N);
  if (!mm_tile_of(s.mm, &split, &ta, &tb)) return;
  MmAcc acc;
  mm_loop<true, true>(s.mm, ta, tb, 0, lds_all, acc);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wm = w & 1, wn = w >> 1;
  const int p0 = ta * kMmTile, v0 = s.first + p0;
  const int64_t n0 = (int64_t)tb * kMmTile;
  const int vl = wm * 128 + 4 * (lane >> 4);
  const int tl = wn * 64 + (lane & 15);
  const int vleft = s.V - v0 - vl;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t n = n0 + tl + 16 * j;
    const float lse = n < N ? s.lse[n] : 0.f;
    const float g = n < N ? s.g[s.active[n]] * s.coef : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float z = acc.v[i][j][r] * s.inv_tau;
        acc.v[i][j][r] = 16 * i + r < vleft ? fast_exp(z - lse) * g : 0.f;
      }
  }
  const int64_t left = N - n0;
  const int rows = (int)(left < kMmTile ? left : kMmTile);
  const int64_t base = n0 * s.K;
  const int count = rows * s.K;
  // One plane at a time through LDS: 256 tokens of 512 bytes, 16-byte chunks
  // XOR-swizzled by the token.
#pragma unroll 1
  for (int pl = 0; pl < kPlanes; ++pl) {
    if (pl) __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = tl + 16 * j, v = vl + 16 * i;
        const f32x4_t x = acc.v[i][j];
        uint32_t lo, hi;
        if (kPlanes == 1) {
          lo = f32x2_to_bf16x2_bits(x[0], x[1]);
          hi = f32x2_to_bf16x2_bits(x[2], x[3]);
        } else {
          lo = split_plane(x[0], pl) | ((uint32_t)split_plane(x[1], pl) << 16);
          hi = split_plane(x[2], pl) | ((uint32_t)split_plane(x[3], pl) << 16);
        }
        *reinterpret_cast<uint2*>(lds_all + t * 512 + (((v >> 3) ^ (t & 15)) << 4) + (v & 4) * 2) =
            make_uint2(lo, hi);
      }
    __syncthreads();
    for (int e = tid; e < count; e += kMmThreads) {
      const int c = s.cols[base + e] - v0;
      if ((unsigned)c < (unsigned)kMmTile) {
        const int t = e / s.K;
        const float x = s.corr[base + e] * (s.g[s.active[n0 + t]] * s.coef);
        *reinterpret_cast<uint16_t*>(lds_all + t * 512 + (((c >> 3) ^ (t & 15)) << 4) +
                                     (c & 7) * 2) =
            kPlanes == 1 ? f32_to_bf16_bits(x) : split_plane(x, pl);
      }
    }
    __syncthreads();
    for (int i = tid; i < rows * 32; i += kMmThreads) {
      const int t = i >> 5, c = i & 31;
      *reinterpret_cast<u32x4_t*>(s.dz + pl * s.plane + (n0 + t) * s.ld + p0 + 8 * c) =
          *reinterpret_cast<const u32x4_t*>(lds_all + t * 512 + ((c ^ (t & 15)) << 4));
    }
  }
}

// ---------------------------------------------------------------------------
// The products with dz: out[b][a] = sum_k A(a, k) B(b, k).
// ---------------------------------------------------------------------------

struct ProductArgs {
  MmArgs mm;
  Hidden h;         // dH: the rows of B and of the output; dW: A and its K
  const int32_t* active;  // dH, straight to out: the rows' own places
  int rows_b;       // dW: the output's rows
  int rows_a;       // the output's row length
  float* partial;   // [splits][plane] float32 rows of lda, or null: straight to out
  int64_t plane;
  int64_t lda;      // rows_a rounded up to 4
  int accumulate;   // add to what partial holds
  void* out;
  int out_bf16;
};

DPC_DEVICE void store_row4(void* out, int64_t at, int left, int bf16, f32x4_t x) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r < left) {
      if (bf16)
        static_cast<uint16_t*>(out)[at + r] = f32_to_bf16_bits(x[r]);
      else
        static_cast<float*>(out)[at + r] = x[r];
    }
}

// kHidden: dH (A = W, K the piece's columns, B = dz by rows); else dW (A = H, K the
// rows, B = dz by columns).
template <bool kHidden>
__global__ void __launch_bounds__(kMmThreads, 1) head_product_kernel(ProductArgs s) {
  int split, ta, tb;
  const uint16_t* hp;
  const int count = hidden_rows(s.h, &hp);
  int rows_b = s.rows_b;
  if (kHidden) {
    rows_b = s.mm.b.rows = count;
    s.mm.tiles_b = tiles_of(count);
  } else {
    s.mm.a.p = hp;
    s.mm.kl = count;
  }
  if (!mm_tile_of(s.mm, &split, &ta, &tb)) return;
  MmAcc acc;
  mm_loop<false, kHidden>(s.mm, ta, tb, split, lds_all, acc);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wm = w & 1, wn = w >> 1;
  const int a0 = ta * kMmTile + wm * 128 + 4 * (lane >> 4);
  const int b0 = tb * kMmTile + wn * 64 + (lane & 15);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int b = b0 + 16 * j;
    if (b >= rows_b) continue;
    const int64_t row = kHidden && !s.partial ? s.active[b] : b;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int a = a0 + 16 * i;
      if (a >= s.rows_a) continue;
      f32x4_t x = acc.v[i][j];
      if (s.partial) {
        f32x4_t* p = reinterpret_cast<f32x4_t*>(s.partial + split * s.plane + row * s.lda + a);
        if (s.accumulate) x += *p;
        *p = x;
      } else {
        store_row4(s.out, row * s.rows_a + a, s.rows_a - a, s.out_bf16, x);
      }
    }
  }
}

// The slices of partial added up in order: row r to out's row active[r] (or r).
__global__ void __launch_bounds__(256) head_reduce_kernel(const float* __restrict__ partial,
                                                          int splits, int64_t plane, int64_t rows,
                                                          const int32_t* __restrict__ count,
                                                          const int32_t* __restrict__ active,
                                                          int D, int64_t lda,
                                                          void* __restrict__ out, int out_bf16) {
  const int64_t quads = lda / 4, total = (count ? *count : rows) * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / quads;
    const int c = (int)(i - row * quads) * 4;
    f32x4_t x = *reinterpret_cast<const f32x4_t*>(partial + row * lda + c);
    for (int s = 1; s < splits; ++s)
      x += *reinterpret_cast<const f32x4_t*>(partial + s * plane + row * lda + c);
    store_row4(out, (active ? active[row] : row) * (int64_t)D + c, D - c, out_bf16, x);
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

constexpr int64_t kDzBytes = 256ll << 20;  // dz of one piece

int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
int64_t up_bytes(int64_t x) { return up(x, 256); }

struct Plan {
  int64_t N;
  int D, V, K, planes;
  int64_t ld;  // of the operands as the tiles read them
  bool pack;
  int tiles_v, tiles_n, tiles_d;
  int piece_tiles, pieces;
  int splits_h, splits_w;
  int64_t lda;
  // Byte offsets in the workspace.
  int64_t h, w, picked, part, dz, ph, pw, bytes;
};

// Slices of `steps` K steps for `tiles` tiles: about one workgroup a compute
// unit, no slice under 8 steps.
int slices(int64_t tiles, int64_t steps) {
  int64_t s = 256 / tiles;
  if (s > steps / 8) s = steps / 8;
  if (s > 32) s = 32;
  return s < 1 ? 1 : (int)s;
}

bool valid_head(int64_t N, int D, int V, int K, int dtype) {
  return N >= 0 && N <= 0x7fffff00ll && D >= 1 && D <= (1 << 20) && V >= 1 && V <= (1 << 30) &&
         K >= 1 && K <= (1 << 16) && (dtype == DPC_F32 || dtype == DPC_BF16);
}

Plan head_plan(int64_t N, int D, int V, int K, int dtype, bool backward, bool dh, bool dw) {
  Plan p = {};
  p.N = N;
  p.D = D;
  p.V = V;
  p.K = K;
  p.planes = dtype == DPC_F32 ? 3 : 1;
  p.ld = up(D, 8);
  p.pack = dtype == DPC_F32 || D % 8 != 0;
  p.tiles_v = (V + kMmTile - 1) / kMmTile;
  p.tiles_n = (int)((N + kMmTile - 1) / kMmTile);
  p.tiles_d = (D + kMmTile - 1) / kMmTile;
  p.lda = up(D, 4);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up_bytes(bytes);
    return o;
  };
  p.h = take(p.planes * N * p.ld * 2);
  if (p.pack) p.w = take(p.planes * (int64_t)V * p.ld * 2);
  if (!backward) {
    p.picked = take(N * K * 4);
    p.part = take(N * p.tiles_v * 8);
  } else {
    int64_t t = kDzBytes / (p.planes * N * kMmTile * 2);
    if (t < 1) t = 1;
    if (t > p.tiles_v) t = p.tiles_v;
    p.pieces = (int)((p.tiles_v + t - 1) / t);
    p.piece_tiles = (p.tiles_v + p.pieces - 1) / p.pieces;
    const int pairs = p.planes == 1 ? 1 : 6;
    p.dz = take(p.planes * N * p.piece_tiles * kMmTile * 2);
    if (dh) {
      p.splits_h = slices((int64_t)p.tiles_d * p.tiles_n, (int64_t)pairs * p.piece_tiles * 4);
      if (p.pieces > 1 || p.splits_h > 1) p.ph = take(p.splits_h * N * p.lda * 4);
    }
    if (dw) {
      p.splits_w = slices((int64_t)p.tiles_d * p.piece_tiles, pairs * ((N + 63) / 64));
      if (p.splits_w > 1)
        p.pw = take(p.splits_w * (int64_t)p.piece_tiles * kMmTile * p.lda * 4);
    }
  }
  p.bytes = at;
  return p;
}

unsigned grid_for(int64_t items) {
  int64_t g = (items + 255) / 256;
  return (unsigned)(g > 16384 ? 16384 : (g < 1 ? 1 : g));
}

// Numbers of rows and operands: the prep launch, and W and H as the tiles read them.
int operands(const Plan& p, PrepArgs& a, uint8_t* ws, hipStream_t s, Hidden* h, MmOperand* w) {
  a.ld = p.ld;
  a.pack = p.pack;
  a.h = reinterpret_cast<uint16_t*>(ws + p.h);
  a.w = reinterpret_cast<uint16_t*>(ws + p.w);
  const void* weight = a.weight;
  if (!p.pack) a.weight = nullptr;
  int64_t items = p.N * p.ld / 8;
  if (p.pack && p.V * p.ld / 8 > items) items = p.V * p.ld / 8;
  hipLaunchKernelGGL(prep_kernel, dim3(grid_for(items)), dim3(256), 0, s, a);
  DPC_HIP_CHECK(hipGetLastError());
  *h = Hidden{p.pack ? nullptr : static_cast<const uint16_t*>(a.hidden), a.h, a.rows.count, p.N};
  *w = MmOperand{p.pack ? a.w : static_cast<const uint16_t*>(weight), p.ld, (int64_t)p.V * p.ld,
                 p.V};
  return DPC_OK;
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace

extern "C" size_t dpc_head_loss_workspace_bytes(int64_t N, int D, int V, int K, int dtype) {
  if (!valid_head(N, D, V, K, dtype) || N == 0) return 0;
  return (size_t)head_plan(N, D, V, K, dtype, false, false, false).bytes;
}

extern "C" size_t dpc_head_loss_grad_workspace_bytes(int64_t N, int D, int V, int K, int dtype,
                                                     int want_hidden, int want_weight) {
  if (!valid_head(N, D, V, K, dtype) || N == 0) return 0;
  return (size_t)head_plan(N, D, V, K, dtype, true, want_hidden != 0, want_weight != 0).bytes;
}

extern "C" int dpc_head_loss(const void* hidden, const void* weight, int64_t N, int D, int V,
                             int dtype, const int64_t* index, const float* teacher, int K,
                             int64_t ignore_index, double temperature, float* loss, int32_t* rows,
                             float* lse, int32_t* cols, float* corr, void* ws, size_t ws_bytes,
                             void* stream) {
  if (!valid_head(N, D, V, K, dtype) || !(temperature > 0.0) || !(temperature < 1e30))
    return DPC_EINVAL;
  if (!teacher && K != 1) return DPC_EINVAL;
  if (N == 0) return DPC_OK;
  if (!hidden || !weight || !index || !loss || !rows || !lse || !cols || !corr || !ws) return DPC_EINVAL;
  const Plan p = head_plan(N, D, V, K, dtype, false, false, false);
  if (!p.pack && (misaligned(hidden) || misaligned(weight))) return DPC_EINVAL;
  if (misaligned(ws)) return DPC_EINVAL;
  if (ws_bytes < (size_t)p.bytes) return DPC_ENOSPC;
  if ((int64_t)p.tiles_v * p.tiles_n > 0x7fffffffll) return DPC_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  uint8_t* base = static_cast<uint8_t*>(ws);
  const Rows r = rows_of(rows, N);
  if (teacher) {
    hipLaunchKernelGGL(entries_kernel, dim3((unsigned)((N + 3) / 4)), dim3(256), 0, s, index,
                       teacher, N, K, V, r.place);
    DPC_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(1024), 0, s, index, ignore_index,
                     teacher != nullptr, N, r, loss);
  DPC_HIP_CHECK(hipGetLastError());
  PrepArgs q = {};
  q.hidden = hidden;
  q.weight = weight;
  q.dtype = dtype;
  q.D = D;
  q.V = V;
  q.K = K;
  q.N = N;
  q.rows = r;
  q.index = index;
  q.teacher = teacher != nullptr;
  q.cols = cols;
  StatsArgs a = {};
  const int rc = operands(p, q, base, s, &a.h, &a.mm.a);
  if (rc != DPC_OK) return rc;
  a.mm.b = MmOperand{nullptr, p.ld, N * p.ld, 0};
  a.mm.kl = (int)p.ld;
  a.mm.planes = p.planes;
  a.mm.tiles_a = p.tiles_v;
  a.mm.tiles_b = p.tiles_n;
  a.mm.splits = 1;
  a.V = V;
  a.K = K;
  a.inv_tau = (float)(1.0 / temperature);
  a.cols = cols;
  a.picked = reinterpret_cast<float*>(base + p.picked);
  a.part = reinterpret_cast<f32x2_t*>(base + p.part);
  hipLaunchKernelGGL(head_stats_kernel, dim3((unsigned)p.tiles_v * (unsigned)p.tiles_n),
                     dim3(kMmThreads), 0, s, a);
  DPC_HIP_CHECK(hipGetLastError());
  JoinArgs j = {r,         K,       p.tiles_v, a.inv_tau, (float)(temperature * temperature),
                cols,      a.picked, teacher,   a.part,    loss,
                lse,       corr};
  hipLaunchKernelGGL(head_join_kernel, dim3((unsigned)((N + 3) / 4)), dim3(256), 0, s, j);
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}

extern "C" int dpc_head_loss_grad(const void* hidden, const void* weight, int64_t N, int D, int V,
                                  int dtype, int32_t* rows, const int32_t* cols,
                                  const float* corr, int K, const float* lse, const float* grad_loss, double temperature,
                                  void* hidden_grad, void* weight_grad, void* ws, size_t ws_bytes,
                                  void* stream) {
  if (!valid_head(N, D, V, K, dtype) || !(temperature > 0.0) || !(temperature < 1e30))
    return DPC_EINVAL;
  if (N == 0) return DPC_OK;
  if (!hidden_grad && !weight_grad) return DPC_EINVAL;
  if (!hidden || !weight || !rows || !cols || !corr || !lse || !grad_loss || !ws) return DPC_EINVAL;
  const Plan p = head_plan(N, D, V, K, dtype, true, hidden_grad != nullptr, weight_grad != nullptr);
  if (!p.pack && (misaligned(hidden) || misaligned(weight))) return DPC_EINVAL;
  if (misaligned(ws)) return DPC_EINVAL;
  if (ws_bytes < (size_t)p.bytes) return DPC_ENOSPC;
  if ((int64_t)p.piece_tiles * p.tiles_n > 0x7fffffffll) return DPC_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  uint8_t* base = static_cast<uint8_t*>(ws);
  const Rows r = rows_of(rows, N);
  PrepArgs pa = {};
  pa.hidden = hidden;
  pa.weight = weight;
  pa.dtype = dtype;
  pa.D = D;
  pa.V = V;
  pa.K = K;
  pa.N = N;
  pa.rows = r;
  pa.zero = hidden_grad;
  Hidden h;
  MmOperand w;
  const int rc = operands(p, pa, base, s, &h, &w);
  if (rc != DPC_OK) return rc;
  const MmOperand hop = {nullptr, p.ld, N * p.ld, 0};
  const int out_bf16 = dtype == DPC_BF16;
  const int64_t esz = out_bf16 ? 2 : 4;
  const int64_t ldz = (int64_t)p.piece_tiles * kMmTile;
  uint16_t* dz = reinterpret_cast<uint16_t*>(base + p.dz);
  for (int i = 0; i < p.pieces; ++i) {
    const int first = i * p.piece_tiles * kMmTile;
    const int tiles = p.tiles_v - i * p.piece_tiles < p.piece_tiles
                          ? p.tiles_v - i * p.piece_tiles
                          : p.piece_tiles;
    if (tiles <= 0) break;
    const int cols_here = V - first < tiles * kMmTile ? V - first : tiles * kMmTile;
    MmOperand wpiece = w;
    wpiece.p = w.p + (int64_t)first * w.ld;
    wpiece.rows = cols_here;
    GradArgs a = {};
    a.mm = MmArgs{wpiece, hop, (int)p.ld, p.planes, tiles, p.tiles_n, 1};
    a.h = h;
    a.active = r.active;
    a.V = V;
    a.K = K;
    a.first = first;
    a.inv_tau = (float)(1.0 / temperature);
    a.coef = (float)temperature;
    a.cols = cols;
    a.corr = corr;
    a.lse = lse;
    a.g = grad_loss;
    a.dz = dz;
    a.ld = ldz;
    a.plane = N * ldz;
    const dim3 grid((unsigned)tiles * (unsigned)p.tiles_n);
    if (p.planes == 1)
      hipLaunchKernelGGL((head_grad_kernel<1>), grid, dim3(kMmThreads), 0, s, a);
    else
      hipLaunchKernelGGL((head_grad_kernel<3>), grid, dim3(kMmThreads), 0, s, a);
    DPC_HIP_CHECK(hipGetLastError());
    const MmOperand zop = {dz, ldz, N * ldz, 0};
    if (hidden_grad) {
      // A = W (D, K-slow: a row holds one vocabulary entry), B = dz (tokens).
      // dz is zero past the vocabulary; W's rows there read as zeros.
      ProductArgs q = {};
      q.mm = MmArgs{wpiece, zop, cols_here, p.planes, p.tiles_d, p.tiles_n, p.splits_h};
      q.h = h;
      q.active = r.active;
      q.rows_a = D;
      q.lda = p.lda;
      q.plane = N * p.lda;
      const bool direct = p.pieces == 1 && p.splits_h == 1;
      q.partial = direct ? nullptr : reinterpret_cast<float*>(base + p.ph);
      q.accumulate = i > 0;
      q.out = hidden_grad;
      q.out_bf16 = out_bf16;
      hipLaunchKernelGGL((head_product_kernel<true>),
                         dim3((unsigned)(p.tiles_d * p.tiles_n * p.splits_h)), dim3(kMmThreads), 0,
                         s, q);
      DPC_HIP_CHECK(hipGetLastError());
      if (!direct && i + 1 == p.pieces) {
        hipLaunchKernelGGL(head_reduce_kernel, dim3(grid_for(N * p.lda / 4)), dim3(256), 0, s,
                           q.partial, p.splits_h, q.plane, N, r.count, r.active, D, p.lda,
                           hidden_grad, out_bf16);
        DPC_HIP_CHECK(hipGetLastError());
      }
    }
    if (weight_grad) {
      ProductArgs q = {};
      q.mm = MmArgs{hop, zop, 0, p.planes, p.tiles_d, tiles, p.splits_w};
      q.h = h;
      q.rows_b = cols_here;
      q.rows_a = D;
      q.lda = p.lda;
      q.plane = (int64_t)cols_here * p.lda;
      q.partial = p.splits_w == 1 ? nullptr : reinterpret_cast<float*>(base + p.pw);
      q.out = static_cast<uint8_t*>(weight_grad) + (int64_t)first * D * esz;
      q.out_bf16 = out_bf16;
      hipLaunchKernelGGL((head_product_kernel<false>),
                         dim3((unsigned)(p.tiles_d * tiles * p.splits_w)), dim3(kMmThreads), 0, s,
                         q);
      DPC_HIP_CHECK(hipGetLastError());
      if (q.partial) {
        hipLaunchKernelGGL(head_reduce_kernel, dim3(grid_for((int64_t)cols_here * p.lda / 4)),
                           dim3(256), 0, s, q.partial, p.splits_w, q.plane, (int64_t)cols_here,
                           (const int32_t*)nullptr, (const int32_t*)nullptr, D, p.lda, q.out,
                           out_bf16);
        DPC_HIP_CHECK(hipGetLastError());
      }
    }
  }
  return DPC_OK;
}
