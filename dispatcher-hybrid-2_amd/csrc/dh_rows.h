// Rows of a vocabulary's logits, read in 16-byte pieces from any element address: what the kernels that take a softmax over
// them (dh_distill.hip, dh_logprob.hip) share.
#pragma once

#include "dh_common.h"

constexpr double kLog2e = 1.4426950408889634;
constexpr double kLn2 = 0.6931471805599453;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// log2(e) over a temperature in two fp32 numbers
struct Scale {
  float hi, lo;
};
// An exponent in base 2, d times a scale: h rounded to fp32 and, in l, what the rounding left. h alone costs the result |h| half
// steps: nothing beside a bf16 gradient, 63 half steps at exponents of -80 beside an fp32 one. FULL puts l back, 2^h (1 + l ln 2),
// for five instructions (four in the forward's sums): 3 half steps whatever the exponent. fp32, V 50257, without and with it, in a
// graph: one exp 777 rows forward 33 and 35, backward 71 and 72 us, 2048 rows 81 and 82, 189 and 190; two exps 35 and 38, 75 and
// 76; 81 and 90, 189 and 193.
struct Exponent {
  float h, l;
};
template <bool FULL> __device__ __forceinline__ Exponent exponent_of(float d, Scale c) {
  const float h = d * c.hi;
  if constexpr (!FULL) return Exponent{h, 0.f};
  // (where h is infinite l would be too, or NaN: the median leaves a number, for 0 times it to be 0)
  return Exponent{h, __builtin_amdgcn_fmed3f(__builtin_fmaf(d, c.lo, __builtin_fmaf(d, c.hi, -h)), -1.f, 1.f)};
}
// 2 to the exponent's `times`, a power of two
template <bool FULL> __device__ __forceinline__ float exp_of(Exponent x, float times = 1.f) {
  const float e = exp2_hw(x.h * times);
  return FULL ? __builtin_fmaf(e * x.l, (float)kLn2 * times, e) : e;
}
template <bool FULL> __device__ __forceinline__ float exp_of(float d, Scale c) { return exp_of<FULL>(exponent_of<FULL>(d, c)); }
template <typename T> constexpr bool kFull = sizeof(T) == 4;
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }

template <typename T> constexpr int kE = 16 / (int)sizeof(T);

// 16 bytes from any element address, as fp32
template <typename T>
__device__ __forceinline__ uint4 load16(const T* p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
template <typename T> __device__ __forceinline__ void unpack(const uint4& v, float (&x)[kE<T>]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < kE<T>; ++j) {
    if constexpr (sizeof(T) == 2)
      x[j] = __uint_as_float((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
    else
      x[j] = __uint_as_float(w[j]);
  }
}
template <typename T> __device__ __forceinline__ uint4 pack(const float (&x)[kE<T>]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 2) {
      typedef float f2 __attribute__((ext_vector_type(2)));
      w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x[2 * j], x[2 * j + 1]}, dh_bf16x2));   // one v_cvt_pk
    } else
      w[j] = __float_as_uint(x[j]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// log of a sum: the exponent in fp64, the logarithm of the rest (at most ln 2 in size) in fp32
__device__ __forceinline__ double log_sum(float s) {
  int e;
  const float f = frexpf(s, &e);
  return isfinite(s) ? (double)e * kLn2 + (double)logf(f) : (double)s;         // (log 0 = -inf + 0)
}

// a whole number of 32 or 64 bits
__device__ __forceinline__ int64_t whole(const void* p, int wide, int64_t i) {
  return wide ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// A row in whole 16-byte pieces from its first 16-byte boundary, a stretch of them for each part, and the logits before and
// behind them, one by one with the first part.
struct Cut {
  int head, p0, p1, singles, tail;
  __device__ __forceinline__ int single(int i, int V) const { return i < head ? i : V - tail + (i - head); }
  // the part's elements are [lo, hi) and, with the first part, the singles
  __device__ __forceinline__ bool holds(int64_t i, int E, int V) const {
    return (i >= head + p0 * E && i < head + p1 * E) || (singles && i >= 0 && (i < head || (i >= V - tail && i < V)));
  }
};
template <typename T>
__device__ __forceinline__ Cut cut_row(const T* row, int V, int which, int parts) {
  constexpr int E = kE<T>;
  Cut c;
  c.head = min((int)((16u - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / (int)sizeof(T), V);
  const int pieces = (V - c.head) / E, per = (pieces + parts - 1) / parts;
  c.tail = V - c.head - pieces * E;
  c.p0 = min(which * per, pieces);
  c.p1 = min(c.p0 + per, pieces);
  c.singles = which == 0 ? c.head + c.tail : 0;
  return c;
}

// Gradients of kPast bytes or more are stored past the caches: what reads them next would find little of them there (the last
// level holds 256 MB), and unwritten lines no longer stand in the way of reading the logits (forward and backward of
// 4096 x 50257 bf16, 412 MB: 244 -> 227 us). Smaller ones stay for the product that takes them.
constexpr int64_t kPast = (int64_t)256 << 20;
