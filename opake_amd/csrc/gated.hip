// A gated feed-forward layer's projections, activation and product, from x [N, D] and
// w [2 F, D] (gate rows, then up rows), and their gradients:
//
//   z = x w^T = [g, u],  h = act(g) u;  act(g) = g s(g) with s the logistic function
//   (SiLU) or the normal distribution's (GELU)
//   dz = [dh u act'(g), dh act(g)],  dx = dz w,  dw = dz^T x
//
// Forward: one product whose 256 x 256 tiles hold the gate and the up projection of 128
// columns, so that h is formed in the accumulators (mm_tile.h, kPaired); z is written
// too where a gradient will be asked for.  Few tiles: the K steps go out in slices, whose
// float32 sums are added up, in order, by a second launch that forms h.  Few tokens:
// a kernel of their own, which reads the weights as they are.
// Backward: dz in one pass over z and dh, and two products.
//
// float32 operands are multiplied as two fp16 planes (mm_tile.h).  Rows of x and of dz
// have a shift each in the products that do not sum over them, w one for the tensor; in dw
// the shift of a row of dz is undone in its row of x before that is shifted as a whole.
//
// Held in fewer than 32 bits, bf16 inputs: dz, which the products take as their operand
// (2^-8 of itself at most, the size of the gradients' own rounding).  z is kept with 8 bits
// more than bf16 has (`rest`, 2^-16): of a z in bf16 the gradients would be 3.0e-3 from
// 64 bits in the mean square, so 2.4e-3.  h is formed from the float32 accumulators.
#include <math.h>

#include "common.h"
#include "mm_planes.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

__shared__ __attribute__((aligned(16))) uint8_t lds_all[131072];

// s(g), and act'(g) where asked for: act' = s + g s'.  kExact: float32's results.
// GELU: with a = |g| / sqrt 2 the normal distribution's tail is erfc(a) / 2, and erfc(a) =
// exp(-a^2) t P(t), t = 1 / (1 + 0.4 a), P a polynomial fitted to exp(a^2) erfc(a) / t
// at Chebyshev's points of t for a from 0 to 35 (1.0e-7 of it at most).
template <bool kExact>
DPC_DEVICE float gate_of(float g, int act, float* slope) {
  auto exp_of = [](float x) { return kExact ? expf(x) : __builtin_amdgcn_exp2f(x * kLog2e); };
  auto over = [](float x) { return kExact ? 1.0f / x : __builtin_amdgcn_rcpf(x); };
  if (act == DPC_ACT_SILU) {
    const float s = over(1.0f + exp_of(-g));
    if (slope) *slope = s * (1.0f + g * (1.0f - s));
    return s;
  }
  const float t = over(fmaf(fabsf(g), 0.4f * 0.70710678118654752f, 1.0f));
  const float e = exp_of(-0.5f * g * g);
  float p = 0.0469222845f;
  p = fmaf(p, t, -0.167397184f);
  p = fmaf(p, t, 0.138786424f);
  p = fmaf(p, t, 0.0267844172f);
  p = fmaf(p, t, 0.120832299f);
  p = fmaf(p, t, 0.17646823f);
  p = fmaf(p, t, 0.206053677f);
  p = fmaf(p, t, 0.225884548f);
  p = fmaf(p, t, 0.225665403f);
  const float tail = 0.5f * p * t * e;
  const float s = g > 0.0f ? 1.0f - tail : tail;
  if (slope) *slope = fmaf(g * 0.39894228040143267794f, e, s);
  return s;
}

// ---------------------------------------------------------------------------
// float32 operands: shifts and planes.  bf16 ones of odd widths: padded copies.  Bound by memory
// and launches (D = 1000, F = 2731, 1773 tokens: 12 us the magnitudes, 19 the planes, each way).
// ---------------------------------------------------------------------------

// Magnitudes that shifts come from, as the bits of the float: each row's largest finite
// one, and the largest of a tensor.
struct Tops {
  const float* src;
  int64_t rows;
  int cols;
  uint32_t* row;  // [rows], or null
  uint32_t* all;  // one word, or null (zero before the launch)
};

// One wave a row; blockIdx.y: the tensor.  Few and large workgroups, since each ends in an
// atomic on one word (1366 of them: 23 us of 22 MB; 256 with wide loads: 12).
constexpr int kTopsWaves = 16;

struct TopsArgs {
  Tops t[2];
};

__global__ void __launch_bounds__(64 * kTopsWaves) gated_tops_kernel(TopsArgs args) {
  __shared__ uint32_t waves[kTopsWaves];
  const Tops a = args.t[blockIdx.y];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t top = 0;
  for (int64_t r = blockIdx.x * (int64_t)kTopsWaves + w; r < a.rows;
       r += gridDim.x * (int64_t)kTopsWaves) {
    const float* x = a.src + r * a.cols;
    uint32_t mine = 0;
    // Up to the first 16-byte boundary, from there in whole quads, and what is left.
    const int head = min((int)(-((uintptr_t)x >> 2) & 3), a.cols), quads = (a.cols - head) / 4;
    const f32x4_t* q = reinterpret_cast<const f32x4_t*>(x + head);
#pragma unroll 4
    for (int c = lane; c < quads; c += 64) {
      const f32x4_t v = q[c];
      mine = max(max(mine, max(finite_bits(v[0]), finite_bits(v[1]))),
                 max(finite_bits(v[2]), finite_bits(v[3])));
    }
    if (lane < head) mine = max(mine, finite_bits(x[lane]));
    if (head + 4 * quads + lane < a.cols) mine = max(mine, finite_bits(x[head + 4 * quads + lane]));
    mine = wave_max_bits(mine);
    if (a.row && lane == 0) a.row[r] = mine;
    top = max(top, mine);
  }
  if (!a.all) return;
  if (lane == 0) waves[w] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kTopsWaves; ++i) top = max(top, waves[i]);
    if (top) atomicMax(a.all, top);
  }
}

__global__ void __launch_bounds__(64) gated_clear_kernel(uint32_t* words, int n) {
  if ((int)threadIdx.x < n) words[threadIdx.x] = 0u;
}

// The largest exponent of a row of x over the power of two that its row of dz is shifted
// by, over the rows whose dz is not zero, plus kExponentBias (0: there is none).  (A
// maximum: any order gives the same.)
constexpr int kExponentBias = 1024;

DPC_DEVICE int exponent_of(uint32_t top) {
  const int e = (int)(top >> 23) & 255;
  return e ? e : 1;
}

__global__ void __launch_bounds__(256) gated_exponent_kernel(const uint32_t* __restrict__ x,
                                                             const uint32_t* __restrict__ dz,
                                                             int64_t N, uint32_t* out) {
  uint32_t top = 0;
  for (int64_t n = blockIdx.x * 256ll + threadIdx.x; n < N; n += gridDim.x * 256ll)
    if (x[n] && dz[n])
      top = max(top, (uint32_t)(exponent_of(x[n]) - half_shift(dz[n]) + kExponentBias));
  top = wave_max_bits(top);
  if ((threadIdx.x & 63) == 0 && top) atomicMax(out, top);
}

// dw's shift of x: 14 less than the largest exponent reaches 2^14 .. 2^15.
DPC_DEVICE int mixed_shift(uint32_t largest) {
  return largest ? 14 + 127 + kExponentBias - (int)largest : 0;
}

// Rows of `cols` elements into planes of 16-bit rows of ld, padded with zeros (`rows_out`
// rows: what lies past the last is zero too).
struct Pack {
  const void* src;
  uint16_t* dst;
  int64_t rows, rows_out, ld;
  int cols;
  const uint32_t* row;    // shifts: by each row's, by the tensor's, or (mixed) for dw by
  const uint32_t* all;    // the exponents' largest and against dz's row's
  int mixed;
};

struct PackArgs {
  Pack p[2];
};

template <bool kHalf>
__global__ void __launch_bounds__(256) gated_pack_kernel(PackArgs args) {
  const Pack a = args.p[blockIdx.y];
  const int64_t chunks = a.ld / 8, items = a.rows_out * chunks, plane = a.rows_out * a.ld;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < items; i += gridDim.x * 256ll) {
    const int64_t r = i / chunks;
    const int c = (int)(i - r * chunks) * 8;
    const bool in = r < a.rows;
    u32x4_t o = {};
    uint16_t* to = a.dst + r * a.ld + c;
    if constexpr (!kHalf) {
      const uint16_t* from = static_cast<const uint16_t*>(a.src) + r * a.cols + c;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (in && c + e < a.cols) o[e >> 1] |= (uint32_t)from[e] << (16 * (e & 1));
      *reinterpret_cast<u32x4_t*>(to) = o;
    } else {
      const float* from = static_cast<const float*>(a.src) + r * a.cols + c;
      int shift = 0;
      bool none = false;  // a row of dz that is zero: so are its products
      if (in && a.mixed) {
        none = a.row[r] == 0;
        shift = mixed_shift(*a.all) - half_shift(a.row[r]);
      } else if (in) {
        shift = half_shift(a.row ? a.row[r] : *a.all);
      }
      float x[8];
      if (in && c + 8 <= a.cols && a.cols % 4 == 0) {
        const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(from),
                      hi = *reinterpret_cast<const f32x4_t*>(from + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e < 4 ? lo[e] : hi[e - 4];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = in && c + e < a.cols ? from[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = none && fabsf(x[e]) < INFINITY ? 0.f : ldexpf(x[e], shift);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[e] = (uint32_t)half_plane(x[2 * e], p) | ((uint32_t)half_plane(x[2 * e + 1], p) << 16);
        *reinterpret_cast<u32x4_t*>(to + p * plane) = o;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The products.  Bound by the K loop (mm_tile.h), the forward also by what it writes.  16384
// tokens, D = 2048, F = 8192, bf16: forward 1062 us (1.04 PFLOP/s; 1.07 GB of h, z and rest),
// dx 848 (1.30), dw 815 (1.35).  1773 tokens, D = 1000, F = 2731, float32: forward 105, dx 64,
// 154 and 28 tiles of 256, so that units are left idle or the sum is cut in slices; 8192 tokens
// of it 372, 235 and dw 271.
// ---------------------------------------------------------------------------

enum Kind { kForward, kHidden, kWeight };

struct ProductArgs {
  MmArgs mm;
  int rows_b;        // forward, dx: tokens; dw: 2 F
  int rows_a;        // forward: F; else D
  float* partial;    // [splits][rows_b][lda] float32, or null: straight to out
  int64_t plane, lda;
  const uint32_t* row;  // float32: the shifts of B's rows (or null),
  const uint32_t* all;  // and the tensor's, or dw's
  int act;
  void* out;         // h, dx or dw
  void* z;           // forward: [N, 2 F], or null,
  int8_t* rest;      // and bf16: what rounding took from it
  int bf16;
};

template <int kKind>
DPC_DEVICE int tensor_shift(const uint32_t* all) {
  return -(kKind == kWeight ? mixed_shift(*all) : half_shift(*all));
}

// Quads of two neighbouring 16-column blocks, as the matrix cores leave them (lane l: columns
// 4 (l / 16) .. of either), to 8 columns a lane, and those as bf16: first block 8 (l / 32) ..
// for even l / 16, second for odd.  64 bytes of a row a store instead of 32.
struct Eight {
  u32x4_t hi;
  uint2 rest;
};
DPC_DEVICE Eight eight_columns(f32x4_t a, f32x4_t b, bool want_rest) {
  uint32_t p[4] = {f32x2_to_bf16x2_bits(a[0], a[1]), f32x2_to_bf16x2_bits(a[2], a[3]),
                   f32x2_to_bf16x2_bits(b[0], b[1]), f32x2_to_bf16x2_bits(b[2], b[3])};
  const auto lo = __builtin_amdgcn_permlane16_swap(p[0], p[2], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(p[1], p[3], false, false);
  Eight r;
  r.hi = u32x4_t{lo[0], hi[0], lo[1], hi[1]};
  r.rest = make_uint2(0, 0);
  if (want_rest) {
    uint32_t q[2] = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t wa = p[e >> 1] >> (16 * (e & 1)) & 0xffffu,
                     wb = p[2 + (e >> 1)] >> (16 * (e & 1)) & 0xffffu;
      q[0] |= (uint32_t)(rest_of(a[e], wa) & 255) << (8 * e);
      q[1] |= (uint32_t)(rest_of(b[e], wb) & 255) << (8 * e);
    }
    const auto t = __builtin_amdgcn_permlane16_swap(q[0], q[1], false, false);
    r.rest = make_uint2(t[0], t[1]);
  }
  return r;
}

// Four columns f .. f + 3 of row n's g and u: z and h.
template <bool kHalf>
DPC_DEVICE void gated_out(const ProductArgs& s, int64_t n, int f, bool whole, f32x4_t g,
                          f32x4_t u) {
  const int F = s.rows_a, left = F - f;
  if (s.z) {
    store_row4(s.z, n * 2 * F + f, left, whole, s.bf16, g);
    store_row4(s.z, n * 2 * F + F + f, left, whole, s.bf16, u);
    if (!kHalf) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < left) {
          s.rest[n * 2 * F + f + r] = (int8_t)rest_of(g[r], f32_to_bf16_bits(g[r]));
          s.rest[n * 2 * F + F + f + r] = (int8_t)rest_of(u[r], f32_to_bf16_bits(u[r]));
        }
    }
  }
  f32x4_t h;
#pragma unroll
  for (int r = 0; r < 4; ++r) h[r] = g[r] * gate_of<kHalf>(g[r], s.act, nullptr) * u[r];
  store_row4(s.out, n * F + f, left, whole, s.bf16, h);
}

// The same, bf16, of two neighbouring blocks of 16 columns: eight from f on of row n.
DPC_DEVICE void gated_out8(const ProductArgs& s, int64_t n, int f, f32x4_t g0, f32x4_t g1,
                           f32x4_t u0, f32x4_t u1) {
  const int F = s.rows_a;
  f32x4_t h0, h1;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    h0[r] = g0[r] * gate_of<false>(g0[r], s.act, nullptr) * u0[r];
    h1[r] = g1[r] * gate_of<false>(g1[r], s.act, nullptr) * u1[r];
  }
  const Eight h = eight_columns(h0, h1, false);
  const bool in = f < F;
  if (in) *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(s.out) + n * F + f) = h.hi;
  if (!s.z) return;
  const Eight g = eight_columns(g0, g1, true), u = eight_columns(u0, u1, true);
  if (!in) return;
  const int64_t at = n * 2 * F + f;
  *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(s.z) + at) = g.hi;
  *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(s.z) + at + F) = u.hi;
  *reinterpret_cast<uint2*>(s.rest + at) = g.rest;
  *reinterpret_cast<uint2*>(s.rest + at + F) = u.rest;
}

template <int kKind, bool kHalf>
DPC_DEVICE void product_epilogue(const ProductArgs& s, MmAcc<kKind == kHidden>& acc, int ta,
                                 int tb, int w, int split, int all) {
  const int lane = threadIdx.x & 63;
  constexpr bool kPairs = kKind == kForward;
  const int a0 = (kPairs ? ta * (kMmTile / 2) + acc.row0(w) / 2 : ta * kMmTile + acc.row0(w)) +
                 4 * (lane >> 4);
  const int b0 = tb * kMmTile + acc.col0(w) + (lane & 15);
  const bool whole = s.rows_a % 4 == 0;
  constexpr int kBlocks = kPairs ? 4 : MmAcc<kKind == kHidden>::kA;
#pragma unroll
  for (int j = 0; j < MmAcc<kKind == kHidden>::kB; ++j) {
    const int b = b0 + 16 * j;
    if (b >= s.rows_b) continue;
    const int shift = kHalf ? all - (s.row ? half_shift(s.row[b]) : 0) : 0;
    if constexpr (kPairs && !kHalf) {
      if (!s.partial && s.rows_a % 8 == 0) {
        const int f = a0 - 4 * (lane >> 4) + 16 * ((lane >> 4) & 1) + 8 * (lane >> 5);
        gated_out8(s, b, f, acc.v[0][j], acc.v[1][j], acc.v[4][j], acc.v[5][j]);
        gated_out8(s, b, f + 32, acc.v[2][j], acc.v[3][j], acc.v[6][j], acc.v[7][j]);
        continue;
      }
    }
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const int a = a0 + 16 * i;
      if (a >= s.rows_a) continue;
      f32x4_t x = acc.v[i][j];
      if (s.partial) {
        float* p = s.partial + split * s.plane + b * s.lda + a;
        *reinterpret_cast<f32x4_t*>(p) = x;
        if constexpr (kPairs) *reinterpret_cast<f32x4_t*>(p + s.lda / 2) = acc.v[i + 4][j];
        continue;
      }
      x = shifted(x, shift);
      if constexpr (kPairs)
        gated_out<kHalf>(s, b, a, whole, x, shifted(acc.v[i + 4][j], shift));
      else
        store_row4(s.out, (int64_t)b * s.rows_a + a, s.rows_a - a, whole, s.bf16, x);
    }
  }
}

// A workgroup a compute unit goes through the tiles, the next one's first step on its way
// while a tile's epilogue runs.
template <int kKind, bool kHalf>
__global__ void __launch_bounds__(kMmThreads, 1) gated_product_kernel(ProductArgs s) {
  constexpr bool kKc = kKind == kForward, kWide = kKind == kHidden;
  MmTile<kKc, kKind != kWeight, false, kWide, kHalf, kKc, kWide> tile(s.mm, lds_all);
  MmAcc<kWide> acc;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int all = kHalf ? tensor_shift<kKind>(s.all) : 0;
  int split2, ta2, tb2, id = blockIdx.x;
  bool more = mm_tile_of(s.mm, id, &split2, &ta2, &tb2);
  if (more) tile.begin(ta2, tb2, split2);
  while (more) {
    const int split = split2, ta = ta2, tb = tb2;
    tile.run(acc);
    id += gridDim.x;
    more = mm_tile_of(s.mm, id, &split2, &ta2, &tb2);
    if (more) tile.begin(ta2, tb2, split2);
    product_epilogue<kKind, kHalf>(s, acc, ta, tb, w, split, all);
  }
}

// The slices added up in order; forward: then h (and z) of them.
template <int kKind, bool kHalf>
__global__ void __launch_bounds__(256) gated_reduce_kernel(ProductArgs s) {
  const int64_t width = kKind == kForward ? s.lda / 2 : s.lda, quads = width / 4;
  const int all = kHalf ? tensor_shift<kKind>(s.all) : 0;
  const bool whole = s.rows_a % 4 == 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < s.rows_b * quads;
       i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / quads;
    const int c = (int)(i - row * quads) * 4;
    const float* p = s.partial + row * s.lda + c;
    f32x4_t x = *reinterpret_cast<const f32x4_t*>(p), u = {};
    if (kKind == kForward) u = *reinterpret_cast<const f32x4_t*>(p + width);
    for (int k = 1; k < s.mm.splits; ++k) {
      p += s.plane;
      x += *reinterpret_cast<const f32x4_t*>(p);
      if (kKind == kForward) u += *reinterpret_cast<const f32x4_t*>(p + width);
    }
    const int shift = kHalf ? all - (s.row ? half_shift(s.row[row]) : 0) : 0;
    x = shifted(x, shift);
    if (kKind == kForward)
      gated_out<kHalf>(s, row, c, whole, x, shifted(u, shift));
    else
      store_row4(s.out, row * s.rows_a + c, s.rows_a - c, whole, s.bf16, x);
  }
}

// ---------------------------------------------------------------------------
// Few tokens: the weights' way from memory is all there is.
// ---------------------------------------------------------------------------

// h (and z) of up to 16 kBlocks tokens: a workgroup takes 16 gate rows of w and their up
// rows, each wave the products of every eighth run of four fragments along D (256 bytes of a row, so
// that whole lines are asked for), and the waves' sums are added up in order.  The next
// run's loads are on their way while one is multiplied.  Rows and tokens past the last are
// read as the last one's, and left out when h is written; behind D there are zeros.
// Bound by memory: 16 tokens of D = 4096, F = 14336 in bf16 take 50 us, 4.7 TB/s of weights,
// one 44 (5.3 TB/s); called again at once, with part of the weights still in the cache, the 16
// take 46.  Beyond 16 by the tokens' reads from L2, as long as the weights'.
// float32: each lane's 16 bytes are four k of its row, one for each of four products (the
// k of a product may be any, if both operands have the same), so nothing is split or shifted.
template <bool kHalf, int kBlocks>
__global__ void __launch_bounds__(512) gated_few_kernel(const void* __restrict__ x,
                                                        const void* __restrict__ wt, int D,
                                                        ProductArgs s) {
  constexpr int kSize = kHalf ? 4 : 2, kLane = 16 / kSize, kStep = 4 * kLane, kRun = 4 * kStep;
  constexpr int kWaves = 8;
  __shared__ f32x4_t sums[kWaves * 2 * kBlocks * 64];  // [wave][gate, up][token block][lane]
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int F = s.rows_a, N = s.rows_b, f0 = blockIdx.x * 16;
  const int at = kLane * (lane >> 4);
  const int64_t row = min(f0 + (lane & 15), F - 1);
  const uint8_t* pw[2] = {static_cast<const uint8_t*>(wt) + (row * D + at) * kSize,
                          static_cast<const uint8_t*>(wt) + ((row + F) * D + at) * kSize};
  const uint8_t* px[kBlocks];
#pragma unroll
  for (int j = 0; j < kBlocks; ++j)
    px[j] = static_cast<const uint8_t*>(x) +
            ((int64_t)min(16 * j + (lane & 15), N - 1) * D + at) * kSize;
  struct Run {
    u32x4_t w[4][2], x[4][kBlocks];
  };
  f32x4_t acc[2][kBlocks] = {};
  auto load = [&](Run& r, int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = (k0 + i * kStep) * kSize;
#pragma unroll
      for (int p = 0; p < 2; ++p) r.w[i][p] = *reinterpret_cast<const u32x4_t*>(pw[p] + k);
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) r.x[i][j] = *reinterpret_cast<const u32x4_t*>(px[j] + k);
    }
  };
  auto multiply = [&](const Run& r) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kBlocks; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          if constexpr (kHalf) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[p][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  __uint_as_float(r.w[i][p][e]), __uint_as_float(r.x[i][j][e]), acc[p][j], 0, 0, 0);
          } else {
            acc[p][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, r.w[i][p]), __builtin_bit_cast(bf16x8_t, r.x[i][j]),
                acc[p][j], 0, 0, 0);
          }
        }
  };
  const int runs = D / kRun;
  Run a, b;
  int r = w;
  if (r < runs) load(a, r * kRun);
  while (r < runs) {
    if (r + kWaves < runs) load(b, (r + kWaves) * kRun);
    multiply(a);
    r += kWaves;
    if (r >= runs) break;
    if (r + kWaves < runs) load(a, (r + kWaves) * kRun);
    multiply(b);
    r += kWaves;
  }
  if (r == runs && runs * kRun < D) {  // what is left: the next wave in turn
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = (runs * kRun + i * kStep) * kSize;
      const bool in = runs * kRun + i * kStep + at < D;
#pragma unroll
      for (int p = 0; p < 2; ++p)
        a.w[i][p] = in ? *reinterpret_cast<const u32x4_t*>(pw[p] + k) : u32x4_t{};
#pragma unroll
      for (int j = 0; j < kBlocks; ++j)
        a.x[i][j] = in ? *reinterpret_cast<const u32x4_t*>(px[j] + k) : u32x4_t{};
    }
    multiply(a);
  }
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) sums[((w * 2 + p) * kBlocks + j) * 64 + lane] = acc[p][j];
  __syncthreads();
  if (w >= kBlocks) return;
  f32x4_t g = {}, u = {};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    g += sums[(2 * i * kBlocks + w) * 64 + lane];
    u += sums[((2 * i + 1) * kBlocks + w) * 64 + lane];
  }
  const int n = 16 * w + (lane & 15), f = f0 + 4 * (lane >> 4);
  if (n < N && f < F) gated_out<kHalf>(s, n, f, F % 4 == 0, g, u);
}

// ---------------------------------------------------------------------------
// dz from z and dh: one pass, bound by memory (16384 tokens, F = 8192, bf16: 331 us, 4.9 TB/s).
// ---------------------------------------------------------------------------

// kVec columns a thread; rows need not start at a vector (the loads' own alignment is the
// element's), the last vector of a row may be short.
template <typename T, int kVec>
__global__ void __launch_bounds__(256) gated_act_grad_kernel(const T* __restrict__ z,
                                                             const int8_t* __restrict__ rest,
                                                             const T* __restrict__ dh, int64_t N,
                                                             int F, int act, T* __restrict__ dz) {
  typedef int8_t bytes_t __attribute__((ext_vector_type(kVec)));
  struct __attribute__((packed, aligned(1))) loose_bytes_t {
    bytes_t v;
  };
  typedef T vec_t __attribute__((ext_vector_type(kVec)));
  struct __attribute__((packed, aligned(sizeof(T)))) loose_t {
    vec_t v;
  };
  const int chunks = (F + kVec - 1) / kVec;
  const int64_t items = N * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items;
       i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / chunks;
    const int f = (int)(i - n * chunks) * kVec;
    const T *pg = z + n * 2 * F + f, *pu = pg + F, *pd = dh + n * F + f;
    T *qg = dz + n * 2 * F + f, *qu = qg + F;
    vec_t g, u, d, og, ou;
    bytes_t rg = {}, ru = {};
    const int8_t *prg = rest + n * 2 * F + f, *pru = prg + F;
    const bool all = f + kVec <= F;
    if (all) {
      g = reinterpret_cast<const loose_t*>(pg)->v;
      u = reinterpret_cast<const loose_t*>(pu)->v;
      d = reinterpret_cast<const loose_t*>(pd)->v;
      if constexpr (sizeof(T) == 2) {
        rg = reinterpret_cast<const loose_bytes_t*>(prg)->v;
        ru = reinterpret_cast<const loose_bytes_t*>(pru)->v;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const bool in = f + e < F;
        g[e] = in ? pg[e] : T(0);
        u[e] = in ? pu[e] : T(0);
        d[e] = in ? pd[e] : T(0);
        if constexpr (sizeof(T) == 2) {
          rg[e] = in ? prg[e] : 0;
          ru[e] = in ? pru[e] : 0;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      constexpr bool kExact = sizeof(T) == 4;
      float gf, uf, df;
      if constexpr (kExact) {
        gf = g[e];
        uf = u[e];
        df = d[e];
      } else {
        gf = with_rest(g[e], rg[e]);
        uf = with_rest(u[e], ru[e]);
        df = bf16_bits_to_f32(d[e]);
      }
      float slope;
      const float s = gate_of<kExact>(gf, act, &slope);
      const float dg = df * uf * slope, du = df * (gf * s);
      if constexpr (kExact) {
        og[e] = dg;
        ou[e] = du;
      } else {
        og[e] = f32_to_bf16_bits(dg);
        ou[e] = f32_to_bf16_bits(du);
      }
    }
    if (all) {
      reinterpret_cast<loose_t*>(qg)->v = og;
      reinterpret_cast<loose_t*>(qu)->v = ou;
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (f + e < F) {
          qg[e] = og[e];
          qu[e] = ou[e];
        }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

bool valid_sizes(int64_t N, int D, int F, int dtype) {
  return N >= 0 && N <= (1ll << 30) && D >= 1 && D <= (1 << 20) && F >= 1 && F <= (1 << 19) &&
         (dtype == DPC_F32 || dtype == DPC_BF16);
}

int64_t blocks_of(int64_t n) { return (n + kMmTile - 1) / kMmTile; }

// One operand as the products read it.
struct Operand {
  int64_t rows, rows_out, ld;
  int cols;
  bool copied;
  size_t at, bytes;  // in the workspace
};

// So many tokens at most go to gated_few_kernel, rows of whole 16-byte chunks given.  D = 4096,
// F = 14336, from memory, against the tiles: bf16 (tiles 67 us) one token 44 us, 16 50, 32 68,
// 48 87; float32 (tiles 433, with the planes' making) one 91, 16 102, 32 151, 64 248.
// (D = 2048, F = 8192, bf16: 14.6, 15, 21, 27; tiles 28.)
bool few(int64_t N, int D, int dtype) {
  return dtype == DPC_BF16 ? N <= 32 && D % 8 == 0 : N <= 64 && D % 4 == 0;
}

struct Plan {
  int64_t N;
  int D, F;
  bool half;
  Operand x, w, dz;
  size_t tops, row_x, row_dz, partial, total;
  int splits[3];

  size_t take(size_t* at, size_t bytes) {
    *at = total;
    total += (bytes + 255) / 256 * 256;
    return *at;
  }
  void operand(Operand* o, int64_t rows, int cols, int64_t rows_out) {
    o->rows = rows;
    o->cols = cols;
    o->copied = half || cols % 8;
    o->ld = o->copied ? up(cols, 64) : cols;
    o->rows_out = o->copied ? rows_out : rows;
    o->bytes = o->copied ? (size_t)(o->rows_out * o->ld * 2 * (half ? 2 : 1)) : 0;
    take(&o->at, o->bytes);
  }
  // Tiles of A and B, and the sum's length.
  void product(Kind kind, int64_t a, int64_t b, int64_t k, int64_t rows_b, int64_t lda) {
    splits[kind] = slices(a * b, (k + kMmStep - 1) / kMmStep * (half ? kMmPairs : 1));
    const size_t need = splits[kind] > 1 ? (size_t)(splits[kind] * rows_b * lda * 4) : 0;
    if (need > partial_bytes) partial_bytes = need;
  }
  size_t partial_bytes;

  Plan(int64_t n, int d, int f, int dtype, bool forward, bool want_x, bool want_w)
      : N(n), D(d), F(f), half(dtype == DPC_F32), total(0), partial_bytes(0) {
    take(&tops, 256);
    take(&row_x, half ? (size_t)N * 4 : 0);
    take(&row_dz, half && !forward ? (size_t)N * 4 : 0);
    x = w = dz = Operand{};
    for (int& v : splits) v = 1;
    if (forward && few(N, D, dtype)) return;
    if (forward || want_w) operand(&x, N, D, N);
    if (forward || want_x) operand(&w, 2ll * F, D, 2ll * F);
    if (!forward) operand(&dz, N, 2 * F, N);
    if (forward)
      product(kForward, (F + 127) / 128, blocks_of(N), D, N, 2 * up(F, 4));
    if (want_x && !forward) product(kHidden, blocks_of(D), blocks_of(N), 2ll * F, N, up(D, 4));
    if (want_w && !forward) product(kWeight, blocks_of(D), blocks_of(2ll * F), N, 2ll * F, up(D, 4));
    take(&partial, partial_bytes);
  }
};

int tops(const TopsArgs& a, int n, hipStream_t s) {
  int64_t rows = a.t[0].rows;
  if (n > 1 && a.t[1].rows > rows) rows = a.t[1].rows;
  int64_t grid = (rows + kTopsWaves - 1) / kTopsWaves;
  if (grid > kUnits) grid = kUnits;
  hipLaunchKernelGGL(gated_tops_kernel, dim3((unsigned)grid, n), dim3(64 * kTopsWaves), 0, s, a);
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}

int pack(const PackArgs& a, int n, bool half, hipStream_t s) {
  int64_t items = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t k = a.p[i].rows_out * (a.p[i].ld / 8);
    if (k > items) items = k;
  }
  int64_t grid = (items + 255) / 256;
  if (grid > 8192) grid = 8192;
  if (half)
    hipLaunchKernelGGL((gated_pack_kernel<true>), dim3((unsigned)grid, n), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((gated_pack_kernel<false>), dim3((unsigned)grid, n), dim3(256), 0, s, a);
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}

template <int kKind, bool kHalf>
int product(ProductArgs& a, hipStream_t s) {
  const int64_t tiles = (int64_t)a.mm.tiles_a * a.mm.tiles_b * a.mm.splits;
  if (tiles > INT32_MAX) return DPC_ENOTSUP;
  if (a.mm.splits == 1) a.partial = nullptr;
  hipLaunchKernelGGL((gated_product_kernel<kKind, kHalf>),
                     dim3((unsigned)(tiles < kUnits ? tiles : kUnits)), dim3(kMmThreads), 0, s, a);
  DPC_HIP_CHECK(hipGetLastError());
  if (a.partial) {
    int64_t grid = (a.rows_b * (a.lda / 4) + 255) / 256;
    if (grid > 4096) grid = 4096;
    hipLaunchKernelGGL((gated_reduce_kernel<kKind, kHalf>), dim3((unsigned)grid), dim3(256), 0, s,
                       a);
    DPC_HIP_CHECK(hipGetLastError());
  }
  return DPC_OK;
}

template <int kKind>
int product(ProductArgs& a, bool half, hipStream_t s) {
  return half ? product<kKind, true>(a, s) : product<kKind, false>(a, s);
}

MmOperand mm_operand(const Operand& o, const void* src, uint8_t* ws, int64_t rows) {
  return MmOperand{o.copied ? reinterpret_cast<const uint16_t*>(ws + o.at)
                            : static_cast<const uint16_t*>(src),
                   o.ld, o.rows_out * o.ld, (int)rows};
}

Pack pack_of(const Operand& o, const void* src, uint8_t* ws, const uint32_t* row,
             const uint32_t* all, int mixed) {
  return Pack{src, reinterpret_cast<uint16_t*>(ws + o.at), o.rows, o.rows_out, o.ld, o.cols, row,
              all, mixed};
}

template <bool kHalf>
int few_product(const ProductArgs& a, const void* x, const void* w, int D, hipStream_t s) {
  const dim3 grid((unsigned)((a.rows_a + 15) / 16)), block(512);
  if (a.rows_b <= 16)
    hipLaunchKernelGGL((gated_few_kernel<kHalf, 1>), grid, block, 0, s, x, w, D, a);
  else if (a.rows_b <= 32)
    hipLaunchKernelGGL((gated_few_kernel<kHalf, 2>), grid, block, 0, s, x, w, D, a);
  else if constexpr (kHalf)
    hipLaunchKernelGGL((gated_few_kernel<kHalf, 4>), grid, block, 0, s, x, w, D, a);
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" size_t dpc_gated_linear_workspace_bytes(int64_t N, int D, int F, int dtype) {
  if (!valid_sizes(N, D, F, dtype) || N == 0) return 0;
  return Plan(N, D, F, dtype, true, false, false).total;
}

extern "C" int dpc_gated_linear(const void* x, const void* w, int64_t N, int D, int F, int dtype,
                                int activation, void* h, void* z, void* rest, void* ws,
                                size_t ws_bytes, void* stream) {
  if (!valid_sizes(N, D, F, dtype) ||
      (activation != DPC_ACT_SILU && activation != DPC_ACT_GELU))
    return DPC_EINVAL;
  if (N == 0) return DPC_OK;
  if (!x || !w || !h || !ws || !aligned16(x) || !aligned16(w) || !aligned16(h) || !aligned16(z) ||
      !aligned16(rest) || (z && dtype == DPC_BF16 && !rest) || ((uintptr_t)ws & 255))
    return DPC_EINVAL;
  const Plan p(N, D, F, dtype, true, false, false);
  if (ws_bytes < p.total) return DPC_ENOSPC;
  hipStream_t s = (hipStream_t)stream;
  uint8_t* base = static_cast<uint8_t*>(ws);
  ProductArgs a = {};
  a.rows_b = (int)N;
  a.rows_a = F;
  a.act = activation;
  a.out = h;
  a.z = z;
  a.rest = static_cast<int8_t*>(rest);
  a.bf16 = !p.half;
  if (few(N, D, dtype))
    return p.half ? few_product<true>(a, x, w, D, s) : few_product<false>(a, x, w, D, s);
  uint32_t* words = reinterpret_cast<uint32_t*>(base + p.tops);
  uint32_t* row_x = reinterpret_cast<uint32_t*>(base + p.row_x);
  if (p.half) {
    hipLaunchKernelGGL(gated_clear_kernel, dim3(1), dim3(64), 0, s, words, 1);
    DPC_HIP_CHECK(hipGetLastError());
    const TopsArgs t = {{{static_cast<const float*>(x), N, D, row_x, nullptr},
                         {static_cast<const float*>(w), 2ll * F, D, nullptr, words}}};
    if (const int rc = tops(t, 2, s)) return rc;
  }
  if (p.x.copied) {
    const PackArgs k = {{pack_of(p.x, x, base, row_x, nullptr, 0),
                         pack_of(p.w, w, base, nullptr, words, 0)}};
    if (const int rc = pack(k, 2, p.half, s)) return rc;
  }
  a.mm = MmArgs{mm_operand(p.w, w, base, F), mm_operand(p.x, x, base, N), (int)up(D, 8),
                (F + 127) / 128, (int)blocks_of(N), p.splits[kForward]};
  a.partial = reinterpret_cast<float*>(base + p.partial);
  a.lda = 2 * up(F, 4);
  a.plane = N * a.lda;
  a.row = row_x;
  a.all = words;
  return product<kForward>(a, p.half, s);
}

extern "C" int dpc_gated_linear_act_grad(const void* z, const void* rest, const void* dh,
                                         int64_t N, int F, int dtype, int activation, void* dz,
                                         void* stream) {
  if (!valid_sizes(N, 1, F, dtype) ||
      (activation != DPC_ACT_SILU && activation != DPC_ACT_GELU))
    return DPC_EINVAL;
  if (N == 0) return DPC_OK;
  if (!z || !dh || !dz || !aligned16(z) || !aligned16(dh) || !aligned16(dz) ||
      (dtype == DPC_BF16 && !rest))
    return DPC_EINVAL;
  const int vec = dtype == DPC_BF16 ? 8 : 4;
  int64_t grid = (N * ceil_div(F, vec) + 255) / 256;
  if (grid > 65536) grid = 65536;
  if (dtype == DPC_BF16)
    hipLaunchKernelGGL((gated_act_grad_kernel<uint16_t, 8>), dim3((unsigned)grid), dim3(256), 0,
                       (hipStream_t)stream, static_cast<const uint16_t*>(z),
                       static_cast<const int8_t*>(rest),
                       static_cast<const uint16_t*>(dh), N, F, activation,
                       static_cast<uint16_t*>(dz));
  else
    hipLaunchKernelGGL((gated_act_grad_kernel<float, 4>), dim3((unsigned)grid), dim3(256), 0,
                       (hipStream_t)stream, static_cast<const float*>(z), nullptr,
                       static_cast<const float*>(dh), N, F, activation, static_cast<float*>(dz));
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}

extern "C" size_t dpc_gated_linear_grad_workspace_bytes(int64_t N, int D, int F, int dtype,
                                                        int want_x, int want_w) {
  if (!valid_sizes(N, D, F, dtype) || N == 0) return 0;
  return Plan(N, D, F, dtype, false, want_x, want_w).total;
}

extern "C" int dpc_gated_linear_grad(const void* x, const void* w, const void* dz, int64_t N,
                                     int D, int F, int dtype, void* dx, void* dw, void* ws,
                                     size_t ws_bytes, void* stream) {
  if (!valid_sizes(N, D, F, dtype)) return DPC_EINVAL;
  if (N == 0 || (!dx && !dw)) return DPC_OK;
  if (!dz || !ws || (dx && !w) || (dw && !x) || !aligned16(x) || !aligned16(w) || !aligned16(dz) ||
      !aligned16(dx) || !aligned16(dw) || ((uintptr_t)ws & 255))
    return DPC_EINVAL;
  const Plan p(N, D, F, dtype, false, dx != nullptr, dw != nullptr);
  if (ws_bytes < p.total) return DPC_ENOSPC;
  hipStream_t s = (hipStream_t)stream;
  uint8_t* base = static_cast<uint8_t*>(ws);
  uint32_t* words = reinterpret_cast<uint32_t*>(base + p.tops);  // w's largest, dw's exponent
  uint32_t* row_x = reinterpret_cast<uint32_t*>(base + p.row_x);
  uint32_t* row_dz = reinterpret_cast<uint32_t*>(base + p.row_dz);
  if (p.half) {
    hipLaunchKernelGGL(gated_clear_kernel, dim3(1), dim3(64), 0, s, words, 2);
    DPC_HIP_CHECK(hipGetLastError());
    TopsArgs t = {{{static_cast<const float*>(dz), N, 2 * F, row_dz, nullptr}, {}}};
    if (dx) t.t[1] = Tops{static_cast<const float*>(w), 2ll * F, D, nullptr, words};
    if (const int rc = tops(t, dx ? 2 : 1, s)) return rc;
    if (dw) {
      const TopsArgs u = {{{static_cast<const float*>(x), N, D, row_x, nullptr}, {}}};
      if (const int rc = tops(u, 1, s)) return rc;
      int64_t grid = (N + 255) / 256;
      if (grid > 64) grid = 64;
      hipLaunchKernelGGL(gated_exponent_kernel, dim3((unsigned)grid), dim3(256), 0, s, row_x,
                         row_dz, N, words + 1);
      DPC_HIP_CHECK(hipGetLastError());
    }
  }
  PackArgs a = {};
  int n = 0;
  if (p.dz.copied) a.p[n++] = pack_of(p.dz, dz, base, row_dz, nullptr, 0);
  if (dx && p.w.copied) a.p[n++] = pack_of(p.w, w, base, nullptr, words, 0);
  if (n)
    if (const int rc = pack(a, n, p.half, s)) return rc;
  if (dw && p.x.copied) {
    const PackArgs b = {{pack_of(p.x, x, base, row_dz, words + 1, 1), {}}};
    if (const int rc = pack(b, 1, p.half, s)) return rc;
  }
  const MmOperand z = mm_operand(p.dz, dz, base, N);
  if (dx) {
    ProductArgs g = {};
    g.mm = MmArgs{mm_operand(p.w, w, base, 2ll * F), z, (int)up(2ll * F, 8), (int)blocks_of(D),
                  (int)blocks_of(N), p.splits[kHidden]};
    g.rows_b = (int)N;
    g.rows_a = D;
    g.partial = reinterpret_cast<float*>(base + p.partial);
    g.lda = up(D, 4);
    g.plane = N * g.lda;
    g.row = row_dz;
    g.all = words;
    g.out = dx;
    g.bf16 = !p.half;
    if (const int rc = product<kHidden>(g, p.half, s)) return rc;
  }
  if (dw) {
    ProductArgs g = {};
    g.mm = MmArgs{mm_operand(p.x, x, base, D), mm_operand(p.dz, dz, base, 2ll * F), (int)N,
                  (int)blocks_of(D), (int)blocks_of(2ll * F), p.splits[kWeight]};
    g.rows_b = 2 * F;
    g.rows_a = D;
    g.partial = reinterpret_cast<float*>(base + p.partial);
    g.lda = up(D, 4);
    g.plane = 2ll * F * g.lda;
    g.all = words + 1;
    g.out = dw;
    g.bf16 = !p.half;
    return product<kWeight>(g, p.half, s);
  }
  return DPC_OK;
}
