// Routing of tokens to experts: scores of router logits z [N, E], the k experts
// with the largest keys, their weights, and the gradient of z.
//
//   s_e = softmax(z)_e or 1 / (1 + exp(-z_e));  key_e = s_e + bias_e, or z_e without a
//   bias (the same order, no rounding)
//   groups: E / groups consecutive experts each; only the top_groups groups whose
//   largest keys are largest take part, or (by_two) those whose two largest s_e + bias_e
//   have the largest sum (of one expert that is left: that one's)
//   w_j = scale s_j, or scale s_j / sum over the chosen s
//
// Ties go to the lower index.  An expert whose logit or key is -inf or NaN is never
// chosen; a slot for which none is left gets expert -1 and weight 0.  A NaN logit
// makes its row's weights NaN.
//
// A row lives in kLanes lanes of a wave (64 / kLanes rows a wave), kVals experts a
// lane, as order-preserving 32-bit keys; a round finds the largest key and then the
// lowest index that has it, by lane moves within the row's lanes.  Rounds: one a
// group kept, one an expert chosen.
//
// Few tokens: a launch's latency (16 tokens of 256 experts: 6 us).  Many: the rounds'
// operations (65536 tokens, 256 experts in 8 groups of which 4, the best 8: 47 us, 67 MB
// of logits at 1.4 TB/s; 63 us with the index found in every round; groups by two: 8 us
// more, 9 where a group is not whole lanes).
#include <float.h>
#include <math.h>

#include "common.h"

namespace {

struct RouteArgs {
  const void* logits;
  int64_t N;
  int E, dtype;
  const float* bias;  // [E] or null
  int k, sigmoid, groups, top_groups, renormalize;
  float scale;
  float* weights;    // [N, k]
  int64_t* experts;  // [N, k]
};

DPC_DEVICE float load_logit(const void* p, int64_t i, int dtype) {
  if (dtype == DPC_BF16) return bf16_bits_to_f32(global_ptr<const uint16_t>(p)[i]);
  if (dtype == DPC_F16) return (float)global_ptr<const _Float16>(p)[i];
  return global_ptr<const float>(p)[i];
}

// Unsigned order of the float order; 0 for -inf and NaN.  -0 counts as +0.
DPC_DEVICE uint32_t order_key(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

DPC_DEVICE float key_value(uint32_t key) {
  return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key);
}

template <int kCtrl>
DPC_DEVICE uint32_t lane_move(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, kCtrl, 0xf, 0xf, false);
}

// op over the row's lanes, in every one of them.
template <int kLanes, typename Op>
DPC_DEVICE uint32_t row_all(uint32_t x, Op op) {
  if (kLanes >= 2) x = op(x, lane_move<0xB1>(x));   // quad_perm [1, 0, 3, 2]
  if (kLanes >= 4) x = op(x, lane_move<0x4E>(x));   // quad_perm [2, 3, 0, 1]
  if (kLanes >= 8) x = op(x, lane_move<0x141>(x));  // row_half_mirror
  if (kLanes >= 16) x = op(x, lane_move<0x140>(x));  // row_mirror
  if (kLanes >= 64) {
    const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16),
                   c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
    x = op(op(a, b), op(c, d));
  }
  return x;
}

struct MaxU {
  DPC_DEVICE uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};
struct MinU {
  DPC_DEVICE uint32_t operator()(uint32_t a, uint32_t b) const { return a < b ? a : b; }
};
struct OrU {
  DPC_DEVICE uint32_t operator()(uint32_t a, uint32_t b) const { return a | b; }
};
struct AddU {
  DPC_DEVICE uint32_t operator()(uint32_t a, uint32_t b) const { return a + b; }
};
struct MaxF {
  DPC_DEVICE uint32_t operator()(uint32_t a, uint32_t b) const {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
};
struct AddF {
  DPC_DEVICE uint32_t operator()(uint32_t a, uint32_t b) const {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }
};
template <int kLanes>
DPC_DEVICE float row_max(float x) {
  return __uint_as_float(row_all<kLanes>(__float_as_uint(x), MaxF()));
}
template <int kLanes>
DPC_DEVICE float row_sum(float x) {
  return __uint_as_float(row_all<kLanes>(__float_as_uint(x), AddF()));
}

// exp2's argument is rounded once, which makes |x| 2^-24 of the result: a score is held in
// 32 bits and within 2^-20 (1 + |x|) of itself, as the choice and the weights need it.
constexpr float kLog2e = 1.44269504088896340736f;
DPC_DEVICE float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
// (The hardware's reciprocal, 1 ulp; of infinity 0.)
DPC_DEVICE float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-z)); }

// The two largest keys of each lane (a >= b) to those of the row's lanes, in every one
// of them.
template <int kLanes>
DPC_DEVICE void row_two(uint32_t& a, uint32_t& b) {
  auto join = [&](uint32_t oa, uint32_t ob) __attribute__((always_inline)) {
    b = MaxU()(MinU()(a, oa), MaxU()(b, ob));
    a = MaxU()(a, oa);
  };
  if (kLanes >= 2) join(lane_move<0xB1>(a), lane_move<0xB1>(b));
  if (kLanes >= 4) join(lane_move<0x4E>(a), lane_move<0x4E>(b));
  if (kLanes >= 8) join(lane_move<0x141>(a), lane_move<0x141>(b));
  if (kLanes >= 16) join(lane_move<0x140>(a), lane_move<0x140>(b));
  if (kLanes >= 64) {
    const uint32_t x = a, y = b;
    a = __builtin_amdgcn_readlane(x, 0);
    b = __builtin_amdgcn_readlane(y, 0);
#pragma unroll
    for (int l = 16; l < 64; l += 16)
      join(__builtin_amdgcn_readlane(x, l), __builtin_amdgcn_readlane(y, l));
  }
}

// The key of a group's two largest keys' sum; 0 where it has none.  (Sums that overflow
// downwards still count as there.)
DPC_DEVICE uint32_t sum_key(uint32_t a, uint32_t b) {
  if (a == 0) return 0;
  return MaxU()(order_key(b ? key_value(a) + key_value(b) : key_value(a)), 1u);
}

// The largest key among key[] and its lowest index (none: 0).
template <int kLanes, int kVals>
DPC_DEVICE uint32_t row_first(const uint32_t (&key)[kVals], int lane, int* index) {
  uint32_t m = key[0];
#pragma unroll
  for (int v = 1; v < kVals; ++v) m = MaxU()(m, key[v]);
  m = row_all<kLanes>(m, MaxU());
  uint32_t at = 0xffffffffu;
#pragma unroll
  for (int v = kVals - 1; v >= 0; --v)
    if (key[v] == m) at = lane + v * kLanes;
  *index = (int)row_all<kLanes>(at, MinU());
  return m;
}

// The k largest keys in order: lane j's `mine` is the j-th's expert.  Three operations
// a key and round: whatever equals the round's largest is taken out at once, and its
// index is the lowest of them.  False where a row has equal keys among its largest
// (more were taken out than rounds found one): then every round has to take one alone.
template <int kLanes, int kVals>
DPC_DEVICE bool choose_distinct(uint32_t (&key)[kVals], int lane, int k, int* mine) {
  int taken = 0, rounds = 0;
#pragma unroll
  for (int v = 0; v < kVals; ++v) taken += key[v] != 0;
  for (int j = 0; j < k; ++j) {
    uint32_t m = key[0];
#pragma unroll
    for (int v = 1; v < kVals; ++v) m = MaxU()(m, key[v]);
    m = row_all<kLanes>(m, MaxU());
    uint32_t at = 0xffffffffu;
    const uint32_t some = m ? m : 1u;
#pragma unroll
    for (int v = kVals - 1; v >= 0; --v) {
      const bool hit = key[v] == some;
      at = hit ? (uint32_t)(lane + v * kLanes) : at;
      key[v] = hit ? 0u : key[v];
    }
    rounds += m != 0;
    at = row_all<kLanes>(at, MinU());
    if (lane == j && m) *mine = (int)at;
  }
#pragma unroll
  for (int v = 0; v < kVals; ++v) taken -= key[v] != 0;
  return (int)row_all<kLanes>((uint32_t)taken, AddU()) == rounds;
}

template <int kLanes, int kVals>
DPC_DEVICE void choose_any(uint32_t (&key)[kVals], int lane, int k, int* mine) {
  for (int j = 0; j < k; ++j) {
    int at;
    const uint32_t m = row_first<kLanes, kVals>(key, lane, &at);
    if (lane == j && m) *mine = at;
#pragma unroll
    for (int v = 0; v < kVals; ++v)
      if (lane + v * kLanes == at) key[v] = 0;
  }
}

// Groups of kSlots * kLanes experts: group g is by[kSlots g ..] of all the row's
// lanes, so their best (kByTwo: the sums of their two best) are row maxima that every
// lane holds.  Keys outside the top_groups best groups become 0.
template <int kLanes, int kVals, int kSlots, bool kByTwo>
DPC_DEVICE void keep_groups(uint32_t (&key)[kVals], const uint32_t (&by)[kVals], int top_groups) {
  constexpr int kGroups = kVals / kSlots;
  uint32_t best[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    uint32_t m = by[g * kSlots], second = 0;
#pragma unroll
    for (int v = 1; v < kSlots; ++v) {
      const uint32_t x = by[g * kSlots + v];
      if (kByTwo) second = MaxU()(second, MinU()(m, x));
      m = MaxU()(m, x);
    }
    if (kByTwo) {
      row_two<kLanes>(m, second);
      best[g] = sum_key(m, second);
    } else {
      best[g] = row_all<kLanes>(m, MaxU());
    }
  }
  uint32_t kept = 0;
  for (int r = 0; r < top_groups; ++r) {
    uint32_t m = best[0];
#pragma unroll
    for (int g = 1; g < kGroups; ++g) m = MaxU()(m, best[g]);
    int at = -1;
#pragma unroll
    for (int g = kGroups - 1; g >= 0; --g)
      if (best[g] == m) at = g;
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      if (g == at) best[g] = 0;
    kept |= m ? 1u << at : 0u;
  }
#pragma unroll
  for (int v = 0; v < kVals; ++v)
    if (!((kept >> (v / kSlots)) & 1)) key[v] = 0;
}

// Groups of any size: each round keeps the group of the largest key outside the kept
// ones.
template <int kLanes, int kVals>
DPC_DEVICE void keep_any_groups(uint32_t (&key)[kVals], int lane, int size, int top_groups) {
  const uint32_t magic = (1u << 20) / size + 1;  // e / size for e, size <= 1024
  uint32_t open[kVals];
  uint32_t kept = 0;  // bit v: key[v]'s group is kept
#pragma unroll
  for (int v = 0; v < kVals; ++v) open[v] = key[v];
  for (int r = 0; r < top_groups; ++r) {
    int at;
    const uint32_t m = row_first<kLanes, kVals>(open, lane, &at);
    const int g = m ? (int)(((uint32_t)at * magic) >> 20) : -1;
#pragma unroll
    for (int v = 0; v < kVals; ++v)
      if ((int)(((uint32_t)(lane + v * kLanes) * magic) >> 20) == g) {
        open[v] = 0;
        kept |= 1u << v;
      }
  }
#pragma unroll
  for (int v = 0; v < kVals; ++v)
    if (!((kept >> v) & 1)) key[v] = 0;
}

// The same by the sums of their two largest keys: each group's in a pass over the keys,
// lane g % kLanes keeps group g's (there are no more groups than experts), then a round
// for each one kept.
template <int kLanes, int kVals>
DPC_DEVICE void keep_any_groups_by_two(uint32_t (&key)[kVals], const uint32_t (&by)[kVals],
                                       int lane, int size, int groups, int top_groups) {
  const uint32_t magic = (1u << 20) / size + 1;
  uint32_t best[kVals];
  uint32_t kept = 0;
#pragma unroll
  for (int v = 0; v < kVals; ++v) best[v] = 0;
  for (int g = 0; g < groups; ++g) {
    uint32_t m = 0, second = 0;
#pragma unroll
    for (int v = 0; v < kVals; ++v) {
      const int of = (int)(((uint32_t)(lane + v * kLanes) * magic) >> 20);
      const uint32_t x = of == g ? by[v] : 0u;
      second = MaxU()(second, MinU()(m, x));
      m = MaxU()(m, x);
    }
    row_two<kLanes>(m, second);
    const uint32_t sum = sum_key(m, second);
#pragma unroll
    for (int v = 0; v < kVals; ++v)
      if (lane + v * kLanes == g) best[v] = sum;
  }
  for (int r = 0; r < top_groups; ++r) {
    int at;
    const uint32_t m = row_first<kLanes, kVals>(best, lane, &at);
    const int g = m ? at : -1;
#pragma unroll
    for (int v = 0; v < kVals; ++v) {
      if (lane + v * kLanes == g) best[v] = 0;
      if ((int)(((uint32_t)(lane + v * kLanes) * magic) >> 20) == g) kept |= 1u << v;
    }
  }
#pragma unroll
  for (int v = 0; v < kVals; ++v)
    if (!((kept >> v) & 1)) key[v] = 0;
}

template <int kLanes, int kVals, bool kByTwo>
__global__ void __launch_bounds__(256) route_kernel(RouteArgs a) {
  constexpr int kRows = 64 / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int64_t row =
      ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * kRows + (threadIdx.x & 63) / kLanes;
  const bool in = row < a.N;
  const int64_t base = in ? row * a.E : 0;
  float z[kVals];
  uint32_t key[kVals];
  bool nan = false;
#pragma unroll
  for (int v = 0; v < kVals; ++v) {
    const int e = lane + v * kLanes;
    z[v] = in && e < a.E ? load_logit(a.logits, base + e, a.dtype) : -INFINITY;
    nan |= isnan(z[v]);
  }
  nan = row_all<kLanes>(nan ? 1u : 0u, OrU()) != 0;
  float top = -INFINITY, inv = 0.0f;
  if (!a.sigmoid && (a.bias || !a.renormalize || kByTwo)) {
#pragma unroll
    for (int v = 0; v < kVals; ++v) top = fmaxf(top, z[v]);
    top = row_max<kLanes>(top);
    const float b = top > -INFINITY ? top : 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < kVals; ++v) sum += fast_exp(z[v] - b);
    sum = row_sum<kLanes>(sum);
    inv = 1.0f / sum;
    top = b;
  }
#pragma unroll
  for (int v = 0; v < kVals; ++v) {
    const int e = lane + v * kLanes;
    float x = z[v];
    if (a.bias && x > -INFINITY) {
      const float s = a.sigmoid ? sigmoid(x) : fast_exp(x - top) * inv;
      x = s + (e < a.E ? a.bias[e] : 0.0f);
    }
    key[v] = order_key(x);
  }
  if (a.top_groups < a.groups) {
    const int size = a.E / a.groups, slots = size / kLanes;
    uint32_t by[kVals];  // what the groups go by
#pragma unroll
    for (int v = 0; v < kVals; ++v) {
      by[v] = key[v];
      if (kByTwo && !a.bias && key[v])  // scores: the logits add up in another order
        by[v] = order_key(a.sigmoid ? sigmoid(z[v]) : fast_exp(z[v] - top) * inv);
    }
    if (size % kLanes == 0 && kVals >= 2 && slots == 1)
      keep_groups<kLanes, kVals, 1, kByTwo>(key, by, a.top_groups);
    else if (size % kLanes == 0 && kVals >= 4 && slots == 2)
      keep_groups<kLanes, kVals, kVals >= 4 ? 2 : 1, kByTwo>(key, by, a.top_groups);
    else if (size % kLanes == 0 && kVals >= 8 && slots == 4)
      keep_groups<kLanes, kVals, kVals >= 8 ? 4 : 1, kByTwo>(key, by, a.top_groups);
    else if (kByTwo)
      keep_any_groups_by_two<kLanes, kVals>(key, by, lane, size, a.groups, a.top_groups);
    else
      keep_any_groups<kLanes, kVals>(key, lane, size, a.top_groups);
  }
  int mine = -1;  // lane j: slot j's expert
  uint32_t left[kVals];
#pragma unroll
  for (int v = 0; v < kVals; ++v) left[v] = key[v];
  const bool distinct = choose_distinct<kLanes, kVals>(left, lane, a.k, &mine);
  if (__any(!distinct)) {
    mine = -1;
    choose_any<kLanes, kVals>(key, lane, a.k, &mine);
  }
  float s = 0.0f, w = 0.0f;
  const float zj = mine >= 0 ? load_logit(a.logits, base + mine, a.dtype) : -INFINITY;
  if (!a.sigmoid && a.renormalize) {
    // Softmax over the chosen: the same quotients, nothing to underflow.
    const float m = row_max<kLanes>(zj);
    s = mine >= 0 ? fast_exp(zj - m) : 0.0f;
  } else if (mine >= 0) {
    s = a.sigmoid ? sigmoid(zj) : fast_exp(zj - top) * inv;
  }
  w = s;
  if (a.renormalize) {
    const float sum = row_sum<kLanes>(s);
    w = sum != 0.0f ? s / sum : 0.0f;
  }
  w = nan ? NAN : w * a.scale;
  if (in && lane < a.k) {
    a.weights[row * a.k + lane] = mine >= 0 ? w : (nan ? NAN : 0.0f);
    a.experts[row * a.k + lane] = mine;
  }
}

struct RouteGradArgs {
  const void* logits;
  int64_t N;
  int E, dtype, k, sigmoid, renormalize;
  float scale;
  const int64_t* experts;
  const float* weights;
  const float* g;  // [N, k]: gradient of the weights
  void* dz;
};

// The gradient of a chosen expert's logit from its lane's weight gradient; a row's
// slots lie in kLanes lanes.  `dot`: the sum over them that the dense form takes off.
template <int kLanes>
DPC_DEVICE float chosen_grad(const RouteGradArgs& a, int64_t row, int slot, bool in, int* expert,
                             float* dot) {
  const int64_t at = row * a.k + slot;
  *expert = in && slot < a.k ? (int)a.experts[at] : -1;
  const bool on = *expert >= 0;
  const float g = on ? a.g[at] * a.scale : 0.0f;
  // The weight without its scale; a sigmoid again from its logit.
  const float share = on && a.scale != 0.0f ? a.weights[at] / a.scale : 0.0f;
  const float s = !a.sigmoid ? share
                             : (on ? sigmoid(load_logit(a.logits, row * a.E + *expert, a.dtype))
                                   : 0.0f);
  float x = g;
  *dot = row_sum<kLanes>(g * (a.renormalize ? share : s));
  if (a.renormalize) {
    x = g - *dot;
    if (a.sigmoid) {
      const float sum = row_sum<kLanes>(s);
      x = sum != 0.0f ? x / sum : 0.0f;
    } else {
      x *= share;
    }
  }
  return a.sigmoid ? x * (s * (1.0f - s)) : x;
}

// All but the softmax's own weights: only the chosen logits have a gradient.  A
// workgroup writes whole rows, zeros and all, from LDS in 16-byte stores: `rows` of
// them (a multiple of 8, so that they are whole 16-byte chunks).  Memory bounds it: 65536
// x 256 float32, 67 MB written in 16 us (4.3 TB/s).
template <int kLanes>
__global__ void __launch_bounds__(256) route_sparse_grad_kernel(RouteGradArgs a, int rows) {
  extern __shared__ __attribute__((aligned(16))) uint8_t tile[];
  const int lane = threadIdx.x % kLanes;
  const int64_t row0 = (int64_t)blockIdx.x * rows;
  const int here = (int)(a.N - row0 < rows ? a.N - row0 : rows);
  const int esz = a.dtype == DPC_F32 ? 4 : 2, bytes = rows * a.E * esz;
  for (int i = threadIdx.x * 16; i < bytes; i += 256 * 16)
    *reinterpret_cast<u32x4_t*>(tile + i) = u32x4_t{0u, 0u, 0u, 0u};
  __syncthreads();
  for (int r = threadIdx.x / kLanes; r < rows; r += 256 / kLanes) {
    int e;
    float dot;
    const float x = chosen_grad<kLanes>(a, row0 + r, lane, r < here, &e, &dot);
    if (e >= 0) {
      if (a.dtype == DPC_F32)
        reinterpret_cast<float*>(tile)[r * a.E + e] = x;
      else if (a.dtype == DPC_BF16)
        reinterpret_cast<uint16_t*>(tile)[r * a.E + e] = f32_to_bf16_bits(x);
      else
        reinterpret_cast<_Float16*>(tile)[r * a.E + e] = (_Float16)x;
    }
  }
  __syncthreads();
  uint8_t* out = static_cast<uint8_t*>(a.dz) + row0 * a.E * esz;
  const int whole = here * a.E * esz;
  for (int i = threadIdx.x * 16; i < whole; i += 256 * 16) {
    if (i + 16 <= whole)
      *reinterpret_cast<u32x4_t*>(out + i) = *reinterpret_cast<const u32x4_t*>(tile + i);
    else
      for (int b = i; b < whole; b += 2)
        *reinterpret_cast<uint16_t*>(out + b) = *reinterpret_cast<const uint16_t*>(tile + b);
  }
}

// The softmax's own weights: every logit of the row has one, p_e (y_e - dot), y the
// chosen experts' gradients.  kLanes lanes a row.  9981 tokens of 60 experts: 6 us, a
// launch's latency.
template <int kLanes>
__global__ void __launch_bounds__(256) route_dense_grad_kernel(RouteGradArgs a) {
  extern __shared__ float chosen[];  // [256 / kLanes][E]
  const int lane = threadIdx.x % kLanes, r = threadIdx.x / kLanes;
  const int64_t row = (int64_t)blockIdx.x * (256 / kLanes) + r;
  const bool in = row < a.N;
  float* y = chosen + r * a.E;
  for (int e = lane; e < a.E; e += kLanes) y[e] = 0.0f;
  __syncthreads();
  int e;
  float dot;
  const float x = chosen_grad<kLanes>(a, row, lane, in, &e, &dot);
  if (e >= 0) y[e] = x;
  __syncthreads();
  const int E = in ? a.E : 0;
  float top = -INFINITY, sum = 0.0f;
  for (int i = lane; i < E; i += kLanes)
    top = fmaxf(top, load_logit(a.logits, row * a.E + i, a.dtype));
  top = row_max<kLanes>(top);
  top = top > -INFINITY ? top : 0.0f;
  for (int i = lane; i < E; i += kLanes)
    sum += fast_exp(load_logit(a.logits, row * a.E + i, a.dtype) - top);
  sum = row_sum<kLanes>(sum);
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  for (int i = lane; i < E; i += kLanes) {
    const float p = fast_exp(load_logit(a.logits, row * a.E + i, a.dtype) - top) * inv;
    const float d = p * (y[i] - dot);
    if (a.dtype == DPC_F32)
      global_ptr<float>(a.dz)[row * a.E + i] = d;
    else if (a.dtype == DPC_BF16)
      global_ptr<uint16_t>(a.dz)[row * a.E + i] = f32_to_bf16_bits(d);
    else
      global_ptr<_Float16>(a.dz)[row * a.E + i] = (_Float16)d;
  }
}

bool valid_route(int64_t N, int E, int k, int dtype, int score) {
  return N >= 0 && N <= 0x7fffff00ll && E >= 1 && E <= 1024 && k >= 1 && k <= E && k <= 64 &&
         (dtype == DPC_F32 || dtype == DPC_BF16 || dtype == DPC_F16) &&
         (score == DPC_ROUTE_SOFTMAX || score == DPC_ROUTE_SIGMOID);
}

bool valid_scale(double scale) { return fabs(scale) <= FLT_MAX; }

template <int kLanes, int kVals>
int launch_route(const RouteArgs& a, bool by_two, hipStream_t s) {
  constexpr int kRows = 4 * (64 / kLanes);
  const dim3 grid((unsigned)((a.N + kRows - 1) / kRows));
  if (by_two)
    hipLaunchKernelGGL((route_kernel<kLanes, kVals, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((route_kernel<kLanes, kVals, false>), grid, dim3(256), 0, s, a);
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}

}  // namespace

extern "C" int dpc_route_topk(const void* logits, int64_t N, int E, int dtype, const float* bias,
                              int k, int score, int groups, int top_groups, int renormalize,
                              double scale, float* weights, int64_t* experts, void* stream) {
  const bool by_two = (score & DPC_ROUTE_GROUPS_BY_TWO) != 0 && top_groups < groups;
  score &= ~DPC_ROUTE_GROUPS_BY_TWO;
  if (!valid_route(N, E, k, dtype, score) || groups < 1 || E % groups || top_groups < 1 ||
      top_groups > groups || k > top_groups * (E / groups) || !valid_scale(scale))
    return DPC_EINVAL;
  if (N == 0) return DPC_OK;
  if (!logits || !weights || !experts) return DPC_EINVAL;
  const RouteArgs a = {logits, N, E, dtype, bias, k, score == DPC_ROUTE_SIGMOID, groups, top_groups,
                       renormalize != 0, (float)scale, weights, experts};
  hipStream_t s = (hipStream_t)stream;
  // As few lanes a row as hold its k slots, and its experts in 2 to 16 registers: 65536
  // tokens of 8 experts take 3.2 us in 4 lanes and 7.3 in 16, of 64 experts 14 in 16 and 56
  // in 64.  Up to 256 experts 16 lanes of 16 pay once there are tokens for them all (the
  // best 8 of 256: 6.4 us against 4.7 in 64 lanes at 2048 tokens, 6.5 against 6.4 at 4096,
  // 7.2 against 9.8 at 8192; k = 1 turns near 8192, k = 16 near 3500).
  if (k <= 4 && E <= 8) return launch_route<4, 2>(a, by_two, s);
  if (k <= 16 && E <= 64) return launch_route<16, 4>(a, by_two, s);
  if (k <= 16 && E <= 256 && N >= 4096) return launch_route<16, 16>(a, by_two, s);
  if (E <= 256) return launch_route<64, 4>(a, by_two, s);
  return launch_route<64, 16>(a, by_two, s);
}

extern "C" int dpc_route_topk_grad(const void* logits, int64_t N, int E, int dtype, int k, int score,
                                   int renormalize, double scale, const int64_t* experts,
                                   const float* weights, const float* grad_weights,
                                   void* grad_logits, void* stream) {
  if (!valid_route(N, E, k, dtype, score) || !valid_scale(scale)) return DPC_EINVAL;
  if (N == 0) return DPC_OK;
  if (!logits || !experts || !weights || !grad_weights || !grad_logits)
    return DPC_EINVAL;
  const RouteGradArgs a = {logits, N, E, dtype, k, score == DPC_ROUTE_SIGMOID, renormalize != 0,
                           (float)scale, experts, weights, grad_weights, grad_logits};
  if ((reinterpret_cast<uintptr_t>(grad_logits) & 15) != 0) return DPC_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  // Lanes a row by its slots, in both.  Dense, 65536 tokens: of 8 experts 6.7 us in 16 lanes
  // and 21 in 64, of 256 49 and 53 (16 tokens of 256: 10 and 4).  Sparse: 16384 tokens of 8
  // experts, k = 2, 4.4 us in 4 lanes and 12 in 16; 65536 of 256, k = 8, 13 in 16 and 18 in
  // 64.
  if (!a.sigmoid && !a.renormalize) {
    if (k <= 16)
      hipLaunchKernelGGL((route_dense_grad_kernel<16>), dim3((unsigned)((N + 15) / 16)), dim3(256),
                         16 * E * 4, s, a);
    else
      hipLaunchKernelGGL((route_dense_grad_kernel<64>), dim3((unsigned)((N + 3) / 4)), dim3(256),
                         4 * E * 4, s, a);
  } else {
    // Rows of about 16 KiB a workgroup, 8 at least.
    const int esz = dtype == DPC_F32 ? 4 : 2;
    int rows = 16384 / (E * esz) / 8 * 8;
    rows = rows < 8 ? 8 : (rows > 256 ? 256 : rows);
    const dim3 grid((unsigned)((N + rows - 1) / rows));
    if (k <= 4)
      hipLaunchKernelGGL((route_sparse_grad_kernel<4>), grid, dim3(256), rows * E * esz, s, a, rows);
    else if (k <= 16)
      hipLaunchKernelGGL((route_sparse_grad_kernel<16>), grid, dim3(256), rows * E * esz, s, a,
                         rows);
    else
      hipLaunchKernelGGL((route_sparse_grad_kernel<64>), grid, dim3(256), rows * E * esz, s, a,
                         rows);
  }
  DPC_HIP_CHECK(hipGetLastError());
  return DPC_OK;
}
