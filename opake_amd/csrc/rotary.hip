// Rotary positions of queries and keys, one launch for both (and one for both
// gradients, which are the opposite rotation).
//
//   turn_i = position * freq_i;  a' = amplitude (a cos turn - b sin turn)
//                                b' = amplitude (a sin turn + b cos turn)
//
// Pair i of a head is (x[i], x[pairs + i]) or, interleaved, (x[2 i], x[2 i + 1]);
// elements from 2 pairs on are copied.  The inverse takes -turn.
//
// Angles are formed in float64 and reduced there to a quarter of a turn, so that far
// positions lose nothing; sine and cosine of what is left (at most an eighth of a turn)
// are float32 Taylor sums.  All heads of a token share them: a workgroup makes the
// tables of its few tokens in LDS (one thread a pair) and then walks their heads.
//
// Memory bounds it: each element is read and written once.  (16 x 1024 tokens, 16 and 16
// heads of 128, bf16: 54 us, 5.0 TB/s; 5 x 1999 of 32 and 8, half of each head, neighbours:
// 46 us, 4.4 TB/s; 16 x 1024 of 16 and 16 in float32: 101 us, 5.3 TB/s.)
#include <math.h>

#include "common.h"

namespace {

// i / d for 0 <= i < 2^24, 1 <= d < 2^24: the float quotient is off by one at most.
struct Divisor {
  int d;
  float inv;
};
DPC_HOST_DEVICE Divisor divisor(int d) { return Divisor{d, 1.0f / (float)d}; }
DPC_DEVICE int divide(int i, const Divisor& v) {
  int r = (int)((float)i * v.inv);
  r -= r * v.d > i;
  r += (r + 1) * v.d <= i;
  return r;
}

struct Heads {
  const void* in;
  void* out;              // contiguous [B, T, heads, h]
  int64_t sb, st;         // input strides, elements
  int sh, heads;
};

struct RotaryArgs {
  Heads part[2];
  int64_t T, tokens;
  int64_t block0;            // workgroups in the launches before
  const int64_t* positions;  // or null: the token's index
  int64_t pos_b, pos_t;
  const double* freqs;
  int h, pairs, chunks, per_token, tokens_each;
  Divisor by_token, by_chunk;
  int interleaved;
  float amplitude, sign;
};

constexpr int kThreads = 256;
constexpr int kTable = 1024;  // (cos, sin) of a workgroup's tokens

DPC_DEVICE float2 cos_sin(double position, double freq) {
  const double quarters = position * freq * 0.63661977236758134308;  // 2 / pi
  const double whole = rint(quarters);
  const float t = (float)((quarters - whole) * 1.57079632679489661923);
  const int n = (int)(whole - 4.0 * floor(whole * 0.25));
  // |t| <= pi / 4: the first terms left out are 1.8e-9 (sine) and 1.2e-10 (cosine).
  const float t2 = t * t;
  float s = 2.7557319e-6f;
  s = fmaf(s, t2, -1.9841270e-4f);
  s = fmaf(s, t2, 8.3333333e-3f);
  s = fmaf(s, t2, -1.6666667e-1f);
  s = fmaf(s * t2, t, t);
  float c = -2.7557319e-7f;
  c = fmaf(c, t2, 2.4801587e-5f);
  c = fmaf(c, t2, -1.3888889e-3f);
  c = fmaf(c, t2, 4.1666667e-2f);
  c = fmaf(c, t2, -0.5f);
  c = fmaf(c, t2, 1.0f);
  const float cs = n & 1 ? s : c, sn = n & 1 ? c : s;
  return make_float2(n == 1 || n == 2 ? -cs : cs, n >= 2 ? -sn : sn);
}

template <typename T>
DPC_DEVICE float to_f32(T x);
template <>
DPC_DEVICE float to_f32(float x) { return x; }
template <>
DPC_DEVICE float to_f32(uint16_t x) { return bf16_bits_to_f32(x); }
template <typename T>
DPC_DEVICE T from_f32(float x);
template <>
DPC_DEVICE float from_f32(float x) { return x; }
template <>
DPC_DEVICE uint16_t from_f32(float x) { return f32_to_bf16_bits(x); }

// A chunk is kVec pairs (two vectors), or 2 kVec elements behind the pairs.
template <typename T, int kVec, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a) {
  typedef T pack_t __attribute__((ext_vector_type(kVec)));
  __shared__ float2 table[kTable];
  const int64_t first = (a.block0 + blockIdx.x) * a.tokens_each;
  const int tokens = (int)min((int64_t)a.tokens_each, a.tokens - first);
  for (int i = threadIdx.x; i < tokens * a.pairs; i += kThreads) {
    const int n = i / a.pairs, p = i - n * a.pairs;
    const int64_t tok = first + n, b = tok / a.T, t = tok - b * a.T;
    const int64_t at = a.positions ? a.positions[b * a.pos_b + t * a.pos_t] : t;
    const float2 cs = cos_sin((double)at, a.freqs[p]);
    table[i] = make_float2(cs.x * a.amplitude, cs.y * a.amplitude * a.sign);
  }
  __syncthreads();
  const int items = tokens * a.per_token;
  for (int i = threadIdx.x; i < items; i += kThreads) {
    const int n = divide(i, a.by_token), r = i - n * a.per_token;
    int head = divide(r, a.by_chunk);
    const int c = r - head * a.chunks;
    const int64_t tok = first + n, b = tok / a.T, t = tok - b * a.T;
    const bool second = head >= a.part[0].heads;
    head -= second ? a.part[0].heads : 0;
    const int heads = second ? a.part[1].heads : a.part[0].heads;
    const T* in = static_cast<const T*>(second ? a.part[1].in : a.part[0].in) +
                  b * (second ? a.part[1].sb : a.part[0].sb) +
                  t * (second ? a.part[1].st : a.part[0].st) +
                  (int64_t)head * (second ? a.part[1].sh : a.part[0].sh);
    T* out = static_cast<T*>(second ? a.part[1].out : a.part[0].out) + (tok * heads + head) * a.h;
    const int p = c * kVec;
    if (p >= a.pairs) {
      const int at = 2 * p;
      if (kVec > 1 || at + 2 <= a.h) {
        const pack_t lo = *reinterpret_cast<const pack_t*>(in + at),
                     hi = *reinterpret_cast<const pack_t*>(in + at + kVec);
        *reinterpret_cast<pack_t*>(out + at) = lo;
        *reinterpret_cast<pack_t*>(out + at + kVec) = hi;
      } else {
        out[at] = in[at];
      }
      continue;
    }
    const int at0 = kInterleaved ? 2 * p : p, at1 = kInterleaved ? at0 + kVec : a.pairs + p;
    T e[2 * kVec];
    const pack_t lo = *reinterpret_cast<const pack_t*>(in + at0),
                 hi = *reinterpret_cast<const pack_t*>(in + at1);
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      e[j] = lo[j];
      e[kVec + j] = hi[j];
    }
    const float2* cs = table + n * a.pairs + p;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      T &pa = kInterleaved ? e[2 * j] : e[j], &pb = kInterleaved ? e[2 * j + 1] : e[kVec + j];
      const float u = to_f32<T>(pa), v = to_f32<T>(pb);
      pa = from_f32<T>(u * cs[j].x - v * cs[j].y);
      pb = from_f32<T>(u * cs[j].y + v * cs[j].x);
    }
    pack_t to, ti;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      to[j] = e[j];
      ti[j] = e[kVec + j];
    }
    *reinterpret_cast<pack_t*>(out + at0) = to;
    *reinterpret_cast<pack_t*>(out + at1) = ti;
  }
}

// Whether every vector of kVec elements is aligned to itself and chunks divide a head.
bool whole_vectors(const RotaryArgs& a, int vec, int bytes) {
  if (a.pairs % vec || (a.h - 2 * a.pairs) % (2 * vec)) return false;
  for (const Heads& x : a.part) {
    if (!x.heads) continue;
    if (((uintptr_t)x.in | (uintptr_t)x.out) % (vec * bytes)) return false;
    if ((x.sb | x.st | x.sh) % vec) return false;
  }
  return true;
}

template <typename T, int kVec>
int launch(RotaryArgs& a, hipStream_t s) {
  a.chunks = ceil_div(a.h, 2 * kVec);
  a.per_token = a.chunks * (a.part[0].heads + a.part[1].heads);
  a.by_token = divisor(a.per_token);
  a.by_chunk = divisor(a.chunks);
  // Four chunks a thread, while that many tokens' tables fit.
  int each = 4 * kThreads / a.per_token;
  if (a.pairs && each > kTable / a.pairs) each = kTable / a.pairs;
  a.tokens_each = each < 1 ? 1 : each;
  const int64_t grid = (a.tokens + a.tokens_each - 1) / a.tokens_each;
  const int64_t most = UINT32_MAX / kThreads;  // a launch has fewer than 2^32 threads
  for (a.block0 = 0; a.block0 < grid; a.block0 += most) {
    const dim3 blocks((unsigned)(grid - a.block0 < most ? grid - a.block0 : most));
    if (a.interleaved)
      hipLaunchKernelGGL((rotary_kernel<T, kVec, true>), blocks, dim3(kThreads), 0, s, a);
    else
      hipLaunchKernelGGL((rotary_kernel<T, kVec, false>), blocks, dim3(kThreads), 0, s, a);
    DPC_HIP_CHECK(hipGetLastError());
  }
  return DPC_OK;
}

}  // namespace

extern "C" int dpc_rotary(const void* q, const void* k, int64_t B, int64_t T, int H, int KV, int h,
                          int dtype, const int64_t* strides, const int64_t* positions,
                          int64_t pos_stride_b, int64_t pos_stride_t, const double* freqs,
                          int pairs, int interleaved, double amplitude, int inverse, void* q_out,
                          void* k_out, void* stream) {
  if (B < 0 || T < 0 || H < 1 || KV < 0 || h < 1 || h > 2048 || pairs < 0 || 2 * pairs > h ||
      pairs > kTable || !strides || (dtype != DPC_F32 && dtype != DPC_BF16))
    return DPC_EINVAL;
  if ((int64_t)(H + (int64_t)KV) * h > (1 << 22)) return DPC_EINVAL;
  if (B == 0 || T == 0) return DPC_OK;
  if (B > INT64_MAX / T || !q || !q_out || (KV && (!k || !k_out)) || (pairs && !freqs))
    return DPC_EINVAL;
  for (int i = 2; i < 6; i += 3)
    if (strides[i] < INT32_MIN || strides[i] > INT32_MAX) return DPC_EINVAL;
  RotaryArgs a;
  a.part[0] = Heads{q, q_out, strides[0], strides[1], (int)strides[2], H};
  a.part[1] = Heads{k, k_out, strides[3], strides[4], (int)strides[5], KV};
  a.T = T;
  a.tokens = B * T;
  a.positions = positions;
  a.pos_b = pos_stride_b;
  a.pos_t = pos_stride_t;
  a.freqs = freqs;
  a.h = h;
  a.pairs = pairs;
  a.interleaved = interleaved != 0;
  a.amplitude = (float)amplitude;
  a.sign = inverse ? -1.f : 1.f;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DPC_BF16) {
    if (whole_vectors(a, 8, 2)) return launch<uint16_t, 8>(a, s);
    if (whole_vectors(a, 4, 2)) return launch<uint16_t, 4>(a, s);
    return launch<uint16_t, 1>(a, s);
  }
  if (whole_vectors(a, 4, 4)) return launch<float, 4>(a, s);
  return launch<float, 1>(a, s);
}
