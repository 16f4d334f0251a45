// Distillation from a teacher's top logits, forward and backward, for gfx950. A row of V student logits z, up to K teacher
// logits t_j at tokens k_j, a temperature tau, a weight w and, optionally, the row's label:
//   p = softmax of t / tau over the row's live slots (k_j >= 0 and t_j > -inf), q = softmax(z / tau), P = softmax(z)
//   row  = w tau^2 sum_j p_j (log p_j - log q_{k_j}) + (1 - w) (-log P_label)
//   loss = the sum or mean of the rows that are not ignored (label == ignore_index), or every row (0 where ignored)
//   dz_v = g w tau (q_v - sum_{j: k_j = v} p_j) + g (1 - w) (P_v - [v = label])
// with g the upstream factor (over the number of rows for the mean). A row without a live slot has no first term.
//
// Forward: one pass over the row with the running maximum m and the sums of exp((z - m) / tau) and exp(z - m) (one sum where
// the two are equal or only one is used); the read of z bounds it. Few rows are split over several workgroups, whose sums
// are joined by a second launch. Backward: z once more, and dz; q and P come from m and the sums the forward kept. The
// tokens that the teacher or the label names are written again after the row, from fp32, by a wave that has them ready by then;
// a token named twice gets the sum of its slots in their order.
//
// 4096 x 50257 bf16, K 64, an eighth of the rows ignored: forward 73 us (360 MB, 4.9 TB/s), backward 154 us (772 MB, 5.0 TB/s).
//
// Exponents are taken of z - m (exact for bf16 inputs near m), never of z times a constant: rows of the type's lowest value
// stay finite. Exponentials of fp32 logits are good to fp32 (exp_of). The few operations on a row's sums are in fp64: log p - log q
// is a small difference of larger numbers.

#include "dh_common.h"

namespace {

constexpr int kT = 256;                    // threads that read a row (or its part); one more wave takes the named tokens
constexpr int kW = kT / 64;
constexpr int kMaxSlots = 256;
constexpr int kSlotsPerLane = kMaxSlots / 64;
constexpr int kMaxParts = 32;
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

// what a row is computed from (by value to every kernel)
struct Rows {
  const void* logits;
  int64_t sb, st;                          // strides of row (b, t), b = r / T
  int rows, T, V;
  const void* t_logits;
  const void* t_tokens;
  const void* labels;                      // null: none
  int64_t ignore;
  int t_bf16, token_wide, label_wide, K;
  float tau, weight;
  double inv_tau;
  int soft, hard;                          // which terms there are
  Scale c0, c1;                            // of the exponents: the soft term's (or, without one, the hard term's); the hard term's
};

template <typename T>
__device__ __forceinline__ const T* row_of(const Rows& a, int r) {
  return reinterpret_cast<const T*>(a.logits) + (r / a.T) * a.sb + (r % a.T) * a.st;
}
__device__ __forceinline__ int64_t whole(const void* p, int wide, int64_t i) {
  return wide ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}
__device__ __forceinline__ float teacher_logit(const Rows& a, int64_t i) {
  return a.t_bf16 ? bf16_to_f32(reinterpret_cast<const bf16_t*>(a.t_logits)[i]) : reinterpret_cast<const float*>(a.t_logits)[i];
}

// kept of a row for the backward pass: the maximum, the reciprocals of the two sums, and what there is to differentiate
struct Kept {
  float m, inv_soft, inv_hard;
  int terms;                               // bit 0: the row counts, bit 1: it has live slots
};

// How the two sums of exponentials are had: one alone (only one term, or tau = 1), both, or, where tau is 2 or 4, the second
// with the first's help, exp(z - m) = exp((z - m) / tau)^tau: for bf16 logits as one or two products in place of an exp, which
// takes as long as four (forward of 2048 x 50257 bf16: 38 -> 34 us); for fp32, since a power multiplies the relative error by
// tau, as the exp of tau times the first's exponent, rounded part included (forward of 2048 x 50257: 90 -> 86 us).
enum Mode { kOne = 1, kTwo = 2, kSquare = 3, kFourth = 4 };

struct Sums {
  float m, s0, s1;                         // s0: of exp(z - m) to the scale c0, s1: to c1
};
// exp(d) to the scale c0 and, unless M is kOne, to c1
template <int M, bool FULL> __device__ __forceinline__ void exps(float d, Scale c0, Scale c1, float& e0, float& e1) {
  const Exponent x = exponent_of<FULL>(d, c0);
  e0 = exp_of<FULL>(x);
  if constexpr (M == kTwo) {
    e1 = exp_of<FULL>(d, c1);
  } else if constexpr (M == kOne) {
    e1 = 0.f;
  } else if constexpr (FULL) {
    e1 = exp_of<FULL>(x, M == kSquare ? 2.f : 4.f);
  } else {
    e1 = e0 * e0;
    if constexpr (M == kFourth) e1 *= e1;
  }
}
// (a few a row: FULL whatever the logits' type)
template <int M>
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, Scale c0, Scale c1) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float ref = finite_ref(r.m);
  r.s0 = a.s0 * exp_of<true>(a.m - ref, c0) + b.s0 * exp_of<true>(b.m - ref, c0);
  r.s1 = M != kOne ? a.s1 * exp_of<true>(a.m - ref, c1) + b.s1 * exp_of<true>(b.m - ref, c1) : 0.f;
  return r;
}
template <int M>
__device__ __forceinline__ Sums wave_join(Sums v, Scale c0, Scale c1) {
  const float m = wave_max(v.m), ref = finite_ref(m);
  v.s0 = wave_sum(v.s0 * exp_of<true>(v.m - ref, c0));
  v.s1 = M != kOne ? wave_sum(v.s1 * exp_of<true>(v.m - ref, c1)) : 0.f;
  v.m = m;
  return v;
}

// log of a sum: the exponent in fp64, the logarithm of the rest (at most ln 2 in size) in fp32
__device__ __forceinline__ double log_sum(float s) {
  int e;
  const float f = frexpf(s, &e);
  return isfinite(s) ? (double)e * kLn2 + (double)logf(f) : (double)s;         // (log 0 = -inf + 0)
}

// The teacher's probabilities of a row, by one wave: slot lane + 64 i in p[i], token[i] (-1: empty) and t[i]. Returns the log
// of the sum of exp((t - top) / tau); live: there is a slot that is not empty; bad: a token past the vocabulary.
__device__ __forceinline__ double teacher_row(const Rows& a, int r, int lane, float (&p)[kSlotsPerLane],
                                              int (&token)[kSlotsPerLane], float (&t)[kSlotsPerLane], float& top, bool& live,
                                              bool& bad) {
  float most = -INFINITY;
  bool some = false, over = false;
#pragma unroll
  for (int i = 0; i < kSlotsPerLane; ++i) {
    const int j = i * 64 + lane;
    token[i] = -1;
    t[i] = -INFINITY;
    if (j < a.K) {
      const int64_t k = whole(a.t_tokens, a.token_wide, (int64_t)r * a.K + j);
      const float x = teacher_logit(a, (int64_t)r * a.K + j);
      if (k >= a.V) over = true;
      if (k >= 0 && k < a.V && !(x == -INFINITY)) {
        token[i] = (int)k;
        t[i] = x;
        some = true;
      }
    }
    most = fmaxf(most, t[i]);
  }
  live = __ballot(some) != 0;
  bad = __ballot(over) != 0;
  most = wave_max(most);
  top = finite_ref(most);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kSlotsPerLane; ++i) {
    p[i] = token[i] >= 0 ? exp_of<true>(t[i] - top, a.c0) : 0.f;               // (there is a soft term: c0 is its scale)
    s += p[i];
  }
  s = wave_sum(s);
#pragma unroll
  for (int i = 0; i < kSlotsPerLane; ++i) p[i] = token[i] >= 0 ? p[i] / s : 0.f;
  return live ? log_sum(s) : 0.0;
}

// What a row's loss needs of the logits that are named, without the sums over the vocabulary: the wave beside those that read
// the row has it by the time they end.
struct Named {
  double cross, mass;                      // sum_j p_j (log p_j - (z_{k_j} - ref) / tau), sum_j p_j
  float ref;                               // the largest of those z: near the row's own maximum, or as far below it as all
  float label;                             // the label's logit
  int terms;                               // bit 0: the row counts, bit 1: it has live slots, bit 2: its loss and gradient are
};                                         // NaN: a token or label past the vocabulary, a live slot of NaN or +inf

__device__ __forceinline__ bool counted(const Rows& a, int r) {
  return !a.labels || whole(a.labels, a.label_wide, r) != a.ignore;
}

template <typename T>
__device__ __forceinline__ Named named_of(const Rows& a, int r, int lane) {
  const T* z = row_of<T>(a, r);
  Named n{0.0, 0.0, 0.f, 0.f, 1};
  bool live = false, bad = false;
  if (a.labels) {
    const int64_t label = whole(a.labels, a.label_wide, r);
    bad = label < 0 || label >= a.V;
    if (a.hard && !bad) n.label = Elem<T>::load(z + label);
  }
  if (a.soft) {
    float p[kSlotsPerLane], t[kSlotsPerLane], top;
    int token[kSlotsPerLane];
    bool over;
    const double lt = teacher_row(a, r, lane, p, token, t, top, live, over);
    bad |= over;
    float x[kSlotsPerLane], most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kSlotsPerLane; ++i) {
      if (p[i] == 0.f) token[i] = -1;      // (0 log 0 = 0)
      x[i] = token[i] >= 0 ? Elem<T>::load(z + token[i]) : -INFINITY;
      most = fmaxf(most, x[i]);
    }
    n.ref = finite_ref(wave_max(most));
    double cross = 0.0, mass = 0.0;
#pragma unroll
    for (int i = 0; i < kSlotsPerLane; ++i)
      if (token[i] >= 0) {
        const double log_p = ((double)t[i] - (double)top) * a.inv_tau - lt;
        cross += (double)p[i] * (log_p - ((double)x[i] - (double)n.ref) * a.inv_tau);
        mass += (double)p[i];
      }
    n.cross = wave_sum64(cross);
    n.mass = wave_sum64(mass);
    bad |= n.mass != n.mass;               // (a softmax without a value: no logit of the row has a gradient either)
  }
  n.terms |= (live ? 2 : 0) | (bad ? 4 : 0);
  return n;
}

// the loss of a row that counts, and what the backward pass keeps of it, by one thread
__device__ __forceinline__ void finish_row(const Rows& a, int r, const Sums& v, const Named& n, float* losses, Kept* kept) {
  const float s1 = a.hard && a.soft && a.tau != 1.f ? v.s1 : v.s0;
  const bool live = n.terms & 2, bad = n.terms & 4;
  double row = 0.0;
  if (a.soft && live)
    row = (double)a.weight * (double)a.tau * (double)a.tau *
          (n.cross + n.mass * (((double)v.m - (double)n.ref) * a.inv_tau + log_sum(v.s0)));
  if (a.hard) row += (1.0 - (double)a.weight) * (log_sum(s1) - ((double)n.label - (double)v.m));
  const float nan = __builtin_nanf("");
  losses[r] = bad ? nan : (float)row;
  kept[r] = Kept{v.m, bad ? nan : 1.f / v.s0, bad ? nan : 1.f / s1, 1 | (live || bad ? 2 : 0)};
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

// ---- forward: a row, or one of its parts ----------------------------------------------------------------------------
template <typename T, int M>
__global__ __launch_bounds__(kT + 64) void forward_kernel(Rows a, int parts, Sums* part, Named* named, float* losses,
                                                          Kept* kept) {
  constexpr int E = kE<T>, U = 4;
  __shared__ Sums ws[kW];
  __shared__ Named wn;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = (int)blockIdx.x / parts;
  const int which = (int)blockIdx.x % parts;
  if (!counted(a, r)) {                    // uniform: the row is not read
    if (tid == 0 && which == 0) {
      losses[r] = 0.f;
      kept[r] = Kept{0.f, 0.f, 0.f, 0};
    }
    return;
  }
  const Scale c0 = a.c0, c1 = a.c1;
  if (wave == kW) {
    if (which == 0) {
      const Named n = named_of<T>(a, r, lane);
      if (lane == 0) {
        wn = n;
        if (parts > 1) named[r] = n;
      }
    }
  } else {
    const T* z = row_of<T>(a, r);
    const Cut c = cut_row(z, a.V, which, parts);
    const uint4* base = reinterpret_cast<const uint4*>(z + c.head);
    Sums v{-INFINITY, 0.f, 0.f};
    if (tid < c.singles) {                 // a logit outside the whole pieces
      v.m = Elem<T>::load(z + c.single(tid, a.V));
      const float d = v.m - finite_ref(v.m);
      v.s0 = exp_of<kFull<T>>(d, c0);
      if (M != kOne) v.s1 = exp_of<kFull<T>>(d, c1);
    }
    auto add = [&](const auto& q) {        // some pieces
      constexpr int N = sizeof(q) / sizeof(uint4);
      float x[N][E], most = v.m;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        unpack<T>(q[u], x[u]);
#pragma unroll
        for (int j = 0; j < E; ++j) most = fmaxf(most, x[u][j]);
      }
      const float ref = finite_ref(most);
      v.s0 *= exp_of<kFull<T>>(v.m - ref, c0);
      if (M != kOne) v.s1 *= exp_of<kFull<T>>(v.m - ref, c1);
      v.m = most;
      // sums of a piece, of the pieces, of all: a thread's sum is rounded once for N E exponentials (each added to it alone, the
      // rest of a row beside its largest logit was off by up to half a step for every one of them)
      constexpr float kTimes = M == kFourth ? 4.f : 2.f;
      float t0 = 0.f, t1 = 0.f, k0 = 0.f, k1 = 0.f;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        float p0 = 0.f, p1 = 0.f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          float e0, e1;
          const float d = x[u][j] - ref;
          if constexpr (kFull<T>) {        // the left parts' sum apart, put back after the loop
            const Exponent a0 = exponent_of<true>(d, c0);
            e0 = exp2_hw(a0.h);
            k0 = __builtin_fmaf(e0, a0.l, k0);
            if constexpr (M != kOne) {
              const Exponent a1 = M == kTwo ? exponent_of<true>(d, c1) : Exponent{a0.h * kTimes, a0.l * kTimes};
              e1 = exp2_hw(a1.h);
              k1 = __builtin_fmaf(e1, a1.l, k1);
            }
          } else {
            exps<M, false>(d, c0, c1, e0, e1);
          }
          p0 = j ? p0 + e0 : e0;
          if (M != kOne) p1 = j ? p1 + e1 : e1;
        }
        t0 = u ? t0 + p0 : p0;
        if (M != kOne) t1 = u ? t1 + p1 : p1;
      }
      v.s0 += kFull<T> ? __builtin_fmaf(k0, (float)kLn2, t0) : t0;
      if (M != kOne) v.s1 += kFull<T> ? __builtin_fmaf(k1, (float)kLn2, t1) : t1;
    };
    int p = c.p0 + tid;
    for (; p + (U - 1) * kT < c.p1; p += U * kT) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = base[p + u * kT];
      add(q);
    }
    for (; p < c.p1; p += kT) {
      uint4 q[1] = {base[p]};
      add(q);
    }
    v = wave_join<M>(v, c0, c1);
    if (lane == 0) ws[wave] = v;
  }
  __syncthreads();
  if (tid) return;
  Sums v = ws[0];
#pragma unroll
  for (int w = 1; w < kW; ++w) v = join<M>(v, ws[w], c0, c1);
  if (parts > 1)
    part[blockIdx.x] = v;
  else
    finish_row(a, r, v, wn, losses, kept);
}

// the sum or mean of the rows in a fixed order, and its divisor, by one workgroup
__device__ __forceinline__ void reduce_rows(const float* losses, const Kept* kept, int64_t rows, int mean, float* loss,
                                            float* divisor, double* red, int* cnt) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, W = blockDim.x >> 6;
  double s = 0.0;
  int n = 0;
  for (int64_t r = tid; r < rows; r += blockDim.x) {
    s += losses[r];
    n += kept[r].terms & 1;
  }
  s = wave_sum64(s);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
  if (lane == 0) {
    red[wave] = s;
    cnt[wave] = n;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < W; ++w) {
      s += red[w];
      n += cnt[w];
    }
    // (the mean of no rows is NaN)
    *loss = (float)(mean ? s / (double)n : s);
    *divisor = mean ? (float)n : 1.f;
  }
}

constexpr int kRT = 1024;                  // threads of the reduction, and of the join that ends with it

// rows split over workgroups: their sums joined, a wave a row; loss non-null: one workgroup, which reduces the rows too
template <int M>
__global__ __launch_bounds__(kRT) void join_kernel(Rows a, int parts, const Sums* part, const Named* named, float* losses,
                                                   Kept* kept, int mean, float* loss, float* divisor) {
  __shared__ double red[kRT / 64];
  __shared__ int cnt[kRT / 64];
  const int lane = threadIdx.x & 63, W = blockDim.x >> 6;
  const Scale c0 = a.c0, c1 = a.c1;
  for (int r = blockIdx.x * W + (threadIdx.x >> 6); r < a.rows; r += gridDim.x * W) {
    if (!counted(a, r)) continue;          // uniform; the first launch wrote it
    Sums v{-INFINITY, 0.f, 0.f};
    if (lane < parts) v = part[(int64_t)r * parts + lane];
    v = wave_join<M>(v, c0, c1);
    if (lane == 0) finish_row(a, r, v, named[r], losses, kept);
  }
  if (!loss) return;
  __syncthreads();
  reduce_rows(losses, kept, a.rows, mean, loss, divisor, red, cnt);
}

__global__ __launch_bounds__(kRT) void reduce_kernel(const float* losses, const Kept* kept, int64_t rows, int mean,
                                                     float* loss, float* divisor) {
  __shared__ double red[kRT / 64];
  __shared__ int cnt[kRT / 64];
  reduce_rows(losses, kept, rows, mean, loss, divisor, red, cnt);
}

// ---- backward -------------------------------------------------------------------------------------------------------
// Gradients of kPast bytes or more are stored past the caches: what reads them next would find little of them there (the last
// level holds 256 MB), and unwritten lines no longer stand in the way of reading the logits (forward and backward of
// 4096 x 50257 bf16, 412 MB: 244 -> 227 us). Smaller ones stay for the product that takes them.
constexpr int64_t kPast = (int64_t)256 << 20;

// Rows in descending order: the forward pass read the last rows last, and what the caches still hold of them is read first.
template <typename T, int M>
__global__ __launch_bounds__(kT + 64) void backward_kernel(Rows a, int parts, const Kept* kept, const float* dloss,
                                                           int64_t dloss_stride, const float* divisor, T* dz, int past) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  constexpr int E = kE<T>, U = 4;
  __shared__ float sp[kMaxSlots];
  __shared__ int stok[kMaxSlots];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = a.rows - 1 - (int)blockIdx.x / parts;
  const int which = (int)blockIdx.x % parts;
  const T* z = row_of<T>(a, r);
  T* out = dz + (int64_t)r * a.V;
  const Cut c = cut_row(out, a.V, which, parts);               // (by the output's 16-byte boundaries)
  uint4* to = reinterpret_cast<uint4*>(out + c.head);
  const Kept k = kept[r];
  const bool counts = k.terms & 1, soft = counts && a.soft && (k.terms & 2), hard = counts && a.hard;
  if (!soft && !hard) {                    // uniform: no gradient, whatever the row holds
    for (int p = c.p0 + tid; p < c.p1; p += kT + 64) to[p] = make_uint4(0u, 0u, 0u, 0u);
    if (tid < c.singles) Elem<T>::store(out + c.single(tid, a.V), 0.f);
    return;
  }
  const float g = dloss[dloss_stride * r] / (divisor ? *divisor : 1.f);
  const float gs = soft ? g * a.weight * a.tau : 0.f, gh = hard ? g * (1.f - a.weight) : 0.f;
  const Scale c0 = a.c0, c1 = a.c1;
  // dz of a logit without the teacher's and the label's part: f0 exp(z - m) to the scale c0, and f1 exp(z - m) to c1
  const float ref = finite_ref(k.m);
  // (a row without live slots has no soft term, and no 0 * inf)
  const float f0 = M == kOne ? (gs + gh) * k.inv_soft : soft ? gs * k.inv_soft : 0.f, f1 = gh * k.inv_hard;
  auto value = [&](float x) {
    float e0, e1;
    exps<M, kFull<T>>(x - ref, c0, c1, e0, e1);
    return M == kOne ? f0 * e0 : M == kSquare && !kFull<T> ? e0 * (f0 + f1 * e0) : f0 * e0 + f1 * e1;
  };
  // the named tokens of this part, by the wave beside those that write it: slots lane + 64 i, the label behind them
  const int K = soft ? a.K : 0;
  float y[kSlotsPerLane + 1];
  int64_t at[kSlotsPerLane + 1];
  if (wave == kW) {
    const int64_t label = hard ? whole(a.labels, a.label_wide, r) : -1;
    float p[kSlotsPerLane], t[kSlotsPerLane], top;
    int token[kSlotsPerLane];
    if (soft) {
      bool live, bad;
      teacher_row(a, r, lane, p, token, t, top, live, bad);
    }
#pragma unroll
    for (int i = 0; i <= kSlotsPerLane; ++i) {
      at[i] = i == kSlotsPerLane ? (lane == 0 ? label : -1) : soft ? token[i] : -1;
      if (!c.holds(at[i], E, a.V)) at[i] = -1;
      y[i] = at[i] >= 0 ? Elem<T>::load(z + at[i]) : 0.f;
      if (i < kSlotsPerLane && soft) {
        sp[i * 64 + lane] = p[i];
        stok[i * 64 + lane] = token[i];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    float sum[kSlotsPerLane + 1];
#pragma unroll
    for (int i = 0; i <= kSlotsPerLane; ++i) sum[i] = 0.f;
    for (int j = 0; j < K; ++j) {
      const int v = stok[j];
      const float q = sp[j];
#pragma unroll
      for (int i = 0; i <= kSlotsPerLane; ++i) sum[i] += at[i] == v ? q : 0.f;
    }
#pragma unroll
    for (int i = 0; i <= kSlotsPerLane; ++i) {
      y[i] = value(y[i]) - gs * sum[i];
      if (at[i] == label) y[i] -= gh;
    }
  } else {
    const T* from = z + c.head;
    auto put = [&](int p, const uint4& q) {
      float x[E];
      unpack<T>(q, x);
#pragma unroll
      for (int j = 0; j < E; ++j) x[j] = value(x[j]);
      const uint4 o = pack<T>(x);
      if (past)
        __builtin_nontemporal_store(words{o.x, o.y, o.z, o.w}, reinterpret_cast<words*>(to + p));
      else
        to[p] = o;
    };
    int p = c.p0 + tid;
    for (; p + (U - 1) * kT < c.p1; p += U * kT) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = load16(from + (int64_t)(p + u * kT) * E);
#pragma unroll
      for (int u = 0; u < U; ++u) put(p + u * kT, q[u]);
    }
    for (; p < c.p1; p += kT) put(p, load16(from + (int64_t)p * E));
    if (tid < c.singles) {
      const int i = c.single(tid, a.V);
      Elem<T>::store(out + i, value(Elem<T>::load(z + i)));
    }
  }
  __syncthreads();
  if (wave == kW) {
#pragma unroll
    for (int i = 0; i <= kSlotsPerLane; ++i)
      if (at[i] >= 0) Elem<T>::store(out + at[i], y[i]);
  }
}

// ---- sizes ----------------------------------------------------------------------------------------------------------
// workgroups a row: enough for 1024 in all, each with at least two pieces a thread
int parts_of(int64_t rows, int V, int dtype) {
  const int64_t pieces = ((int64_t)V * (dtype == DH_BF16 ? 2 : 4) + 15) / 16;
  int64_t p = 1024 / (rows > 0 ? rows : 1);
  const int64_t most = pieces / (2 * kT);
  if (p > most) p = most;
  if (p > kMaxParts) p = kMaxParts;
  return p < 1 ? 1 : (int)p;
}

int check(const char* who, int dtype, const Rows& a, int t_dtype, int token_bits, int label_bits) {
  DH_REQUIRE(dtype == DH_F32 || dtype == DH_BF16, DH_ERR_UNSUPPORTED_DTYPE, "%s: dtype %d", who, dtype);
  DH_REQUIRE(t_dtype == DH_F32 || t_dtype == DH_BF16, DH_ERR_UNSUPPORTED_DTYPE, "%s: teacher dtype %d", who, t_dtype);
  DH_REQUIRE((token_bits == 32 || token_bits == 64) && (!a.labels || label_bits == 32 || label_bits == 64),
             DH_ERR_UNSUPPORTED_DTYPE, "%s: tokens of %d bits, labels of %d", who, token_bits, label_bits);
  DH_REQUIRE(a.rows >= 0 && a.rows < (1 << 22) && a.T >= 1 && a.V >= 1 && a.V <= (1 << 24), DH_ERR_UNSUPPORTED_SHAPE,
             "%s: %d rows (-1: too many), T=%d V=%d", who, a.rows, a.T, a.V);
  DH_REQUIRE(a.K >= 1 && a.K <= kMaxSlots, DH_ERR_UNSUPPORTED_SHAPE, "%s: K=%d must be in [1, %d]", who, a.K, kMaxSlots);
  // (below the least normal number its reciprocal overflows)
  DH_REQUIRE(a.tau >= 0x1p-126f && a.tau < INFINITY && a.weight >= 0.f && a.weight <= 1.f, DH_ERR_INVALID_ARG,
             "%s: temperature %g, weight %g", who, (double)a.tau, (double)a.weight);
  DH_REQUIRE(a.rows == 0 || a.labels || a.weight == 1.f, DH_ERR_INVALID_ARG, "%s: weight %g without labels", who, (double)a.weight);
  DH_REQUIRE(a.rows == 0 || (a.logits && a.t_logits && a.t_tokens), DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE((uintptr_t)a.logits % (dtype == DH_BF16 ? 2 : 4) == 0 && (uintptr_t)a.t_logits % (t_dtype == DH_BF16 ? 2 : 4) == 0 &&
                 (uintptr_t)a.t_tokens % (token_bits / 8) == 0 && (!a.labels || (uintptr_t)a.labels % (label_bits / 8) == 0),
             DH_ERR_INVALID_ARG, "%s: operands not aligned to their elements", who);
  return 0;
}

Rows rows_of(const void* logits, int64_t sb, int64_t st, int64_t B, int T, int V, int t_dtype, const void* t_logits,
             const void* t_tokens, int token_bits, int K, const void* labels, int label_bits, int64_t ignore, float tau,
             float weight) {
  Rows a;
  a.logits = logits;
  a.sb = sb;
  a.st = st;
  a.rows = B < 0 || T < 0 || (T > 0 && B >= ((int64_t)1 << 22) / T + 1) ? -1 : (int)(B * T);       // -1: too many
  a.T = T;
  a.V = V;
  a.t_logits = t_logits;
  a.t_tokens = t_tokens;
  a.labels = labels;
  a.ignore = ignore;
  a.t_bf16 = t_dtype == DH_BF16;
  a.token_wide = token_bits == 64;
  a.label_wide = label_bits == 64;
  a.K = K;
  a.tau = tau;
  a.weight = weight;
  a.inv_tau = 1.0 / (double)tau;
  a.soft = weight > 0.f;
  a.hard = labels != nullptr && weight < 1.f;
  auto scale = [](double c) { return Scale{(float)c, (float)(c - (double)(float)c)}; };
  a.c1 = scale(kLog2e);
  a.c0 = a.soft ? scale(kLog2e / (double)tau) : a.c1;
  return a;
}

Mode mode_of(const Rows& a) {
  if (!(a.soft && a.hard && a.tau != 1.f)) return kOne;
  return a.tau == 2.f ? kSquare : a.tau == 4.f ? kFourth : kTwo;
}

template <typename T, int M>
int forward(const Rows& a, int parts, int reduction, float* losses, Kept* kept, float* loss, float* divisor, char* ws,
            hipStream_t s) {
  Named* named = (Named*)ws;
  Sums* part = (Sums*)(ws + a.rows * sizeof(Named));
  forward_kernel<T, M><<<dim3((unsigned)a.rows * parts), dim3(kT + 64), 0, s>>>(a, parts, part, named, losses, kept);
  if (int st = dh_check_launch("dh_distill_fwd")) return st;
  const int mean = reduction == 1;
  if (parts > 1) {
    const bool ends = reduction != 0 && a.rows <= 64;          // one workgroup joins all rows and reduces them
    if (ends)
      join_kernel<M><<<dim3(1), dim3(kRT), 0, s>>>(a, parts, part, named, losses, kept, mean, loss, divisor);
    else
      join_kernel<M><<<dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s>>>(a, parts, part, named, losses, kept, mean,
                                                                             nullptr, nullptr);
    if (int st = dh_check_launch("dh_distill_fwd")) return st;
    if (ends) return 0;
  }
  if (reduction == 0) return 0;
  reduce_kernel<<<dim3(1), dim3(kRT), 0, s>>>(losses, kept, a.rows, mean, loss, divisor);
  return dh_check_launch("dh_distill_fwd");
}
template <typename T, typename... A>
int forward_mode(const Rows& a, A... rest) {
  switch (mode_of(a)) {
    case kOne: return forward<T, kOne>(a, rest...);
    case kTwo: return forward<T, kTwo>(a, rest...);
    case kSquare: return forward<T, kSquare>(a, rest...);
    default: return forward<T, kFourth>(a, rest...);
  }
}

template <typename T, int M>
int backward(const Rows& a, int parts, const Kept* kept, const float* dloss, int64_t stride, const float* divisor, void* dz,
             hipStream_t s) {
  const int past = (int64_t)a.rows * a.V * (int)sizeof(T) >= kPast;
  backward_kernel<T, M><<<dim3((unsigned)a.rows * parts), dim3(kT + 64), 0, s>>>(a, parts, kept, dloss, stride, divisor, (T*)dz,
                                                                                past);
  return dh_check_launch("dh_distill_bwd");
}
template <typename T, typename... A>
int backward_mode(const Rows& a, A... rest) {
  switch (mode_of(a)) {
    case kOne: return backward<T, kOne>(a, rest...);
    case kTwo: return backward<T, kTwo>(a, rest...);
    case kSquare: return backward<T, kSquare>(a, rest...);
    default: return backward<T, kFourth>(a, rest...);
  }
}

}  // namespace

extern "C" int64_t dh_distill_workspace_bytes(int dtype, int64_t rows, int V) {
  const int parts = parts_of(rows, V, dtype);
  return parts > 1 ? rows * (int64_t)(sizeof(Named) + parts * sizeof(Sums)) : 0;
}

extern "C" int dh_distill_fwd(int dtype, const void* logits, int64_t stride_b, int64_t stride_t, int64_t B, int T, int V,
                              int teacher_dtype, const void* teacher_logits, const void* teacher_tokens, int token_bits, int K,
                              const void* labels, int label_bits, int64_t ignore_index, float temperature, float weight,
                              int reduction, float* row_loss, void* row_kept, float* loss, float* divisor, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const char* who = "dh_distill_fwd";
  const Rows a = rows_of(logits, stride_b, stride_t, B, T, V, teacher_dtype, teacher_logits, teacher_tokens, token_bits, K,
                         labels, label_bits, ignore_index, temperature, weight);
  if (int st = check(who, dtype, a, teacher_dtype, token_bits, label_bits)) return st;
  DH_REQUIRE(reduction >= 0 && reduction <= 2, DH_ERR_INVALID_ARG, "%s: reduction %d", who, reduction);
  DH_REQUIRE(a.rows == 0 || (row_loss && row_kept && (uintptr_t)row_kept % 16 == 0), DH_ERR_INVALID_ARG,
             "%s: null or unaligned pointer argument", who);
  DH_REQUIRE(reduction == 0 || (loss && divisor), DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE((uintptr_t)row_loss % 4 == 0 && (uintptr_t)loss % 4 == 0 && (uintptr_t)divisor % 4 == 0, DH_ERR_INVALID_ARG,
             "%s: results not aligned to their elements", who);
  const int64_t need = dh_distill_workspace_bytes(dtype, a.rows, V);
  DH_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 8 == 0)), DH_ERR_INVALID_ARG,
             "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes, (long long)need);
  hipStream_t s = (hipStream_t)stream;
  Kept* kept = (Kept*)row_kept;
  if (a.rows == 0) {
    if (reduction == 0) return 0;
    reduce_kernel<<<dim3(1), dim3(kRT), 0, s>>>(row_loss, kept, 0, reduction == 1, loss, divisor);
    return dh_check_launch(who);
  }
  const int parts = parts_of(a.rows, V, dtype);
  return dtype == DH_BF16 ? forward_mode<bf16_t>(a, parts, reduction, row_loss, kept, loss, divisor, (char*)workspace, s)
                          : forward_mode<float>(a, parts, reduction, row_loss, kept, loss, divisor, (char*)workspace, s);
}

extern "C" int dh_distill_bwd(int dtype, const void* logits, int64_t stride_b, int64_t stride_t, int64_t B, int T, int V,
                              int teacher_dtype, const void* teacher_logits, const void* teacher_tokens, int token_bits, int K,
                              const void* labels, int label_bits, int64_t ignore_index, float temperature, float weight,
                              const void* row_kept, const float* dloss, int64_t dloss_stride, const float* divisor, void* dlogits,
                              void* stream) {
  const char* who = "dh_distill_bwd";
  const Rows a = rows_of(logits, stride_b, stride_t, B, T, V, teacher_dtype, teacher_logits, teacher_tokens, token_bits, K,
                         labels, label_bits, ignore_index, temperature, weight);
  if (int st = check(who, dtype, a, teacher_dtype, token_bits, label_bits)) return st;
  if (a.rows == 0) return 0;
  DH_REQUIRE(row_kept && (uintptr_t)row_kept % 16 == 0 && dloss && dlogits && dloss_stride >= 0, DH_ERR_INVALID_ARG,
             "%s: null or unaligned pointer argument", who);
  DH_REQUIRE((uintptr_t)dloss % 4 == 0 && (uintptr_t)divisor % 4 == 0 && (uintptr_t)dlogits % (dtype == DH_BF16 ? 2 : 4) == 0,
             DH_ERR_INVALID_ARG, "%s: operands not aligned to their elements", who);
  const int parts = parts_of(a.rows, V, dtype);
  const Kept* kept = (const Kept*)row_kept;
  hipStream_t s = (hipStream_t)stream;
  return dtype == DH_BF16 ? backward_mode<bf16_t>(a, parts, kept, dloss, dloss_stride, divisor, dlogits, s)
                          : backward_mode<float>(a, parts, kept, dloss, dloss_stride, divisor, dlogits, s);
}
