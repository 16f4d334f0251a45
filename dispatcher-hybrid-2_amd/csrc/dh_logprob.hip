// Log-probabilities of given tokens and the losses made of them, forward and backward, for gfx950. A row of V logits z, a
// temperature tau, the row's token y:
//   p = softmax(z / tau),  lp = log p_y,  H = - sum_v p_v log p_v
//   dz_v = (a ([v = y] - p_v) - e p_v (log p_v + H)) / tau            with a, e the gradients in lp and H
// A row whose token is ignore_index is not read: lp = H = 0, a gradient of zeros. Three operators share the passes over z:
//   log-probabilities   lp and, wanted, H of every row; a, e are the caller's gradients
//   preference loss     sequences i and i + n are a pair. S = the sum (or mean) of a sequence's lp, R a reference's,
//                       D = (S - R)_i - (S - R)_{i+n}, x = beta D - margin, and of a pair
//                         sigmoid   - (1 - eps) log sigma(x) - eps log sigma(-x)
//                         hinge     max(0, 1 - x)
//                         squared   (D - 1 / (2 beta))^2
//   policy loss         r = exp(lp - old), an advantage A, d = reference - lp, and of a row
//                         - min(r A, clip(r, 1 - low, 1 + high) A) + kl (exp(d) - d - 1) - w H
//                       over the rows, their number, or each sequence's number and the number of sequences
//
// Forward: one pass over the row with the running maximum m and the sums of E = exp((z - m) / tau) and, for H, of E times its
// exponent; the read of z bounds it. Few long rows are split over several workgroups, whose sums a second launch joins. The losses
// add one launch over the rows' lp (and one that adds their parts), which also leaves a and e. Backward: z once more, and dz;
// m, 1 / sum and the mean exponent are all it needs of a row. A row with a = e = 0 (a clipped ratio, a pair behind the hinge)
// is not read. bytes bound both: 5994 of 8192 rows of 50257 bf16 forward 107 us (602 MB, 5.6 TB/s; a bare read reaches 6.1), backward
// 269 (1426 MB, 5.3 TB/s; a copy of 734 MB 5.2, of 2 GiB 4.9); with H, 5631 rows, 115 (VALU busy for 82% of it) and 261.
//
// Sums over V are fp32 (a thread's over 4 pieces at a time), what follows from a row's sums is fp64, lp included until it is
// returned: sequence sums, ratios and their comparison with the clip are of unrounded lp.

#include "dh_rows.h"

namespace {

typedef uint32_t words __attribute__((ext_vector_type(4)));

constexpr int kT = 256;                    // threads of a workgroup whose rows are split or short, and of the losses' launches
constexpr int kW = kT / 64;
constexpr int kWide = 512;                 // of one that takes a whole long row
constexpr int kMaxParts = 32;
constexpr float kFar = -200.f;             // an exponent in base 2 whose power is 0: stands in for -inf where it is a factor

struct Rows {
  const void* logits;
  int64_t sb, st;                          // strides of row (b, t), b = r / T
  int rows, T, V;
  const void* tokens;
  int wide;
  int64_t ignore;
  double inv_tau;
  double part;                             // 1 / tau = part times power, a power of two, 1 <= part < 2
  float power;
  Scale c;                                 // log2(e) / tau
};

template <typename T>
__device__ __forceinline__ const T* row_of(const Rows& a, int r) {
  return reinterpret_cast<const T*>(a.logits) + (r / a.T) * a.sb + (r % a.T) * a.st;
}

// kept of a row for the backward pass
struct Kept {
  float m, inv;                            // the maximum, 1 / sum of E (NaN: the row's token is outside the vocabulary)
  float lean;                              // sum of p (z - m) / tau: log p_v + H = (z_v - m) / tau - lean
  int live;
};
// where a row's results go (null: not wanted)
struct Results {
  float *lp, *ent;
  double *lp64, *ent64;
  Kept* kept;
};

struct Sums {
  float m, s, t;                           // t: the sum of E times its exponent in base 2
};
template <bool ENT>
__device__ __forceinline__ void move_to(Sums& v, float ref, Scale c) {
  const Exponent x = exponent_of<true>(v.m - ref, c);
  const float f = exp_of<true>(x);
  if constexpr (ENT) v.t = f * __builtin_fmaf(v.s, fmaxf(x.h, kFar), v.t);     // (no sum yet: 0 (0 kFar + 0))
  v.s *= f;
}
template <bool ENT>
__device__ __forceinline__ Sums join(Sums a, Sums b, Scale c) {
  const float m = fmaxf(a.m, b.m), ref = finite_ref(m);
  move_to<ENT>(a, ref, c);
  move_to<ENT>(b, ref, c);
  return Sums{m, a.s + b.s, ENT ? a.t + b.t : 0.f};
}
template <bool ENT>
__device__ __forceinline__ Sums wave_join(Sums v, Scale c) {
  const float m = wave_max(v.m);
  move_to<ENT>(v, finite_ref(m), c);
  return Sums{m, wave_sum(v.s), ENT ? wave_sum(v.t) : 0.f};
}

// the results of a row that is not ignored, by one thread; zy: its token's logit, unless the token is outside the vocabulary
template <bool ENT>
__device__ __forceinline__ void finish_row(const Rows& a, int r, const Sums& v, float zy, bool bad, const Results& o) {
  const double nan = __builtin_nan("");
  const double ls = log((double)v.s), lean = ENT ? (double)v.t * kLn2 / (double)v.s : 0.0;
  const double lp = bad ? nan : ((double)zy - (double)v.m) * a.inv_tau - ls, ent = bad ? nan : ls - lean;
  if (o.lp) o.lp[r] = (float)lp;
  if (o.lp64) o.lp64[r] = lp;
  if (ENT && o.ent) o.ent[r] = (float)ent;
  if (ENT && o.ent64) o.ent64[r] = ent;
  if (o.kept) o.kept[r] = Kept{v.m, bad ? (float)nan : 1.f / v.s, (float)lean, 1};
}
__device__ __forceinline__ void skip_row(int r, const Results& o) {
  if (o.lp) o.lp[r] = 0.f;
  if (o.lp64) o.lp64[r] = 0.0;
  if (o.ent) o.ent[r] = 0.f;
  if (o.ent64) o.ent64[r] = 0.0;
  if (o.kept) o.kept[r] = Kept{0.f, 0.f, 0.f, 0};
}

// ---- forward: a row, or one of its parts, by N threads ----------------------------------------------------------------
// Rows that the backward pass, which begins with the last, finds no more in the last level of cache (256 MB) are read past it: the
// reads are faster (8192 rows of 50257 bf16: 6.1 and 6.7 TB/s), and what stays is what is used again. By the bytes behind the row that
// count as past, MB (none / 128 / 192 / 256), forward and backward of the policy loss on 5631 of 8192 rows: 396 / 386 / 386 / 389 us,
// of 2048 rows (206 MB) 102 / 109 / 104 / 103.
constexpr int64_t kReread = (int64_t)192 << 20;

template <typename T, bool ENT, int N>
__device__ __forceinline__ Sums row_sums(const T* z, int V, int which, int parts, int tid, Scale c, bool far) {
  constexpr int E = kE<T>, U = 4;
  const Cut cut = cut_row(z, V, which, parts);
  const uint4* base = reinterpret_cast<const uint4*>(z + cut.head);
  Sums v{-INFINITY, 0.f, 0.f};
  if (tid < cut.singles) {                 // a logit outside the whole pieces
    v.m = Elem<T>::load(z + cut.single(tid, V));
    v.s = exp_of<kFull<T>>(v.m - finite_ref(v.m), c);          // (1, or 0 of -inf: its exponent is 0 or no term)
    if (ENT && v.s != v.s) v.t = v.s;
  }
  auto add = [&](const auto& q) {          // some pieces
    constexpr int P = sizeof(q) / sizeof(uint4);
    float x[P][E], most = v.m;
#pragma unroll
    for (int u = 0; u < P; ++u) {
      unpack<T>(q[u], x[u]);
#pragma unroll
      for (int j = 0; j < E; ++j) most = fmaxf(most, x[u][j]);
    }
    const float ref = finite_ref(most);
    const Exponent by = exponent_of<kFull<T>>(v.m - ref, c);
    const float f = exp_of<kFull<T>>(by);
    if (ENT) v.t = f * __builtin_fmaf(v.s, fmaxf(by.h, kFar), v.t);
    v.s *= f;
    v.m = most;
    // sums of a piece, of the pieces, of all: a thread's sum is rounded once for P E exponentials
    float s = 0.f, t = 0.f, left = 0.f, left_t = 0.f;
#pragma unroll
    for (int u = 0; u < P; ++u) {
      float p = 0.f, pt = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const Exponent h = exponent_of<kFull<T>>(x[u][j] - ref, c);
        const float e = exp2_hw(h.h);
        p = j ? p + e : e;
        if constexpr (kFull<T>) left = __builtin_fmaf(e, h.l, left);           // (put back after the loop)
        if constexpr (ENT) {
          const float eh = e * fmaxf(h.h, kFar);
          pt = j ? pt + eh : eh;
          if constexpr (kFull<T>) left_t = __builtin_fmaf(eh, h.l, left_t);
        }
      }
      s = u ? s + p : p;
      if (ENT) t = u ? t + pt : pt;
    }
    v.s += kFull<T> ? __builtin_fmaf(left, (float)kLn2, s) : s;
    if (ENT) v.t += kFull<T> ? __builtin_fmaf(left_t, (float)kLn2, t) : t;
  };
  auto get = [&](int i) {
    if (!far) return base[i];              // uniform
    const words v = __builtin_nontemporal_load(reinterpret_cast<const words*>(base + i));
    return make_uint4(v[0], v[1], v[2], v[3]);
  };
  int p = cut.p0 + tid;
  for (; p + (U - 1) * N < cut.p1; p += U * N) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = get(p + u * N);
    add(q);
  }
  for (; p < cut.p1; p += N) {
    uint4 q[1] = {base[p]};
    add(q);
  }
  return wave_join<ENT>(v, c);
}

// N = 256: a workgroup a part of a row. N = 512: a workgroup a row (V 50257 bf16, 5631 of 8192 rows: 118 us with 256, 111 with 512,
// 123 with 1024). N = 64: a wave a row, four to a workgroup
template <int N> constexpr int kThreads = N < kT ? kT : N;

template <typename T, bool ENT, int N>
__global__ __launch_bounds__(kThreads<N>) void forward_kernel(Rows a, int parts, Sums* part, Results o) {
  const int tid = threadIdx.x % N, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = N == 64 ? (int)blockIdx.x * kW + wave : N == kT ? (int)blockIdx.x / parts : (int)blockIdx.x;
  const int which = N == kT ? (int)blockIdx.x % parts : 0;
  if (r >= a.rows) return;                 // (N = 64: no barrier follows)
  const int64_t y = whole(a.tokens, a.wide, r);
  if (y == a.ignore) {                     // uniform: the row is not read
    if (tid == 0 && which == 0) skip_row(r, o);
    return;
  }
  const T* z = row_of<T>(a, r);
  const bool bad = y < 0 || y >= a.V;
  float zy = 0.f;
  if (tid == 0 && !bad) zy = Elem<T>::load(z + y);
  const bool far = (int64_t)(a.rows - r) * a.V * (int)sizeof(T) > kReread;
  Sums v = row_sums<T, ENT, N>(z, a.V, which, N == kT ? parts : 1, tid, a.c, far);
  if constexpr (N > 64) {
    __shared__ Sums ws[N / 64];
    if (lane == 0) ws[wave] = v;
    __syncthreads();
    if (tid) return;
    v = ws[0];
#pragma unroll
    for (int w = 1; w < N / 64; ++w) v = join<ENT>(v, ws[w], a.c);
    if constexpr (N == kT) {
      part[blockIdx.x] = v;
      return;
    }
  }
  if (N != kT && tid == 0) finish_row<ENT>(a, r, v, zy, bad, o);
}

// a row split over workgroups: its sums joined, by G lanes (r past the last row: nothing)
template <typename T, bool ENT, int G>
__device__ __forceinline__ void join_row(const Rows& a, int r, int parts, const Sums* part, const Results& o) {
  const int lane = threadIdx.x % G;
  const int64_t y = r < a.rows ? whole(a.tokens, a.wide, r) : a.ignore;
  const bool on = y != a.ignore, bad = y < 0 || y >= a.V;      // (the first launch wrote ignored rows)
  float zy = 0.f;
  if (lane == 0 && on && !bad) zy = Elem<T>::load(row_of<T>(a, r) + y);
  Sums v{-INFINITY, 0.f, 0.f};
  if (on)
    for (int k = lane; k < parts; k += G) v = join<ENT>(v, part[(int64_t)r * parts + k], a.c);
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = join<ENT>(v, Sums{__shfl_xor(v.m, o), __shfl_xor(v.s, o), ENT ? __shfl_xor(v.t, o) : 0.f}, a.c);
  if (lane == 0 && on) finish_row<ENT>(a, r, v, zy, bad, o);
}
template <typename T, bool ENT>
__global__ __launch_bounds__(kT) void join_kernel(Rows a, int parts, const Sums* part, Results o) {
  join_row<T, ENT, 16>(a, blockIdx.x * (kT / 16) + (threadIdx.x >> 4), parts, part, o);
}

// ---- the losses on the rows' log-probabilities ------------------------------------------------------------------------
// one workgroup's part of a loss: a sum, and what the mean divides it by
struct Part {
  double sum;
  int64_t n;
};

__device__ __forceinline__ Part wave_part(Part p) {
  p.sum = wave_sum64(p.sum);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) p.n += __shfl_xor(p.n, o);
  return p;
}
__device__ __forceinline__ void write_loss(const Part& p, int mean, float* loss, float* divisor) {
  *loss = (float)(mean ? p.sum / (double)p.n : p.sum);         // (the mean of none is NaN)
  *divisor = mean ? (float)p.n : 1.f;
}
// the parts in a fixed order, by one workgroup
__global__ __launch_bounds__(1024) void reduce_kernel(const Part* part, int64_t parts, int mean, float* loss, float* divisor) {
  __shared__ Part red[16];
  Part p{0.0, 0};
  for (int64_t i = threadIdx.x; i < parts; i += blockDim.x) {
    p.sum += part[i].sum;
    p.n += part[i].n;
  }
  p = wave_part(p);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = p;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < (int)blockDim.x / 64; ++w) {
    p.sum += red[w].sum;
    p.n += red[w].n;
  }
  write_loss(p, mean, loss, divisor);
}

struct Preference {
  int pairs, T, kind, average;
  double beta, margin, eps;
  const void* reference;                   // null: none
  int wide;                                // fp64
};

__device__ __forceinline__ double log1p_exp(double x) {        // log(1 + e^x)
  return x > 0.0 ? x + log1p(exp(-x)) : log1p(exp(x));
}

// Where the losses' results go: losses null where one is reduced, loss null where not.
struct LossResults {
  float *losses, *values, *by_lp, *by_ent; // values: a sequence's S; by_lp, by_ent: the derivatives without the divisor
  Part* part;
  int mean;
  float *loss, *divisor;
};

// pair i by a workgroup of N threads, half of them a sequence; the result is thread 0's
template <int N>
__device__ __forceinline__ Part preference_pair(const Preference& f, int i, const double* lp, const Kept* kept, const LossResults& o,
                                                Part (&red)[N / 64]) {
  constexpr int W = N / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = wave / (W / 2);
  const int64_t first = (int64_t)(half ? f.pairs + i : i) * f.T;
  Part p{0.0, 0};
#pragma unroll 4
  for (int t = threadIdx.x % (N / 2); t < f.T; t += N / 2) {
    p.sum += lp[first + t];
    p.n += kept[first + t].live;
  }
  p = wave_part(p);
  if (lane == 0) red[wave] = p;
  __syncthreads();
  if (threadIdx.x) return Part{0.0, 0};
  double gain[2], count[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    Part q = red[h * (W / 2)];
    for (int w = 1; w < W / 2; ++w) {
      q.sum += red[h * (W / 2) + w].sum;
      q.n += red[h * (W / 2) + w].n;
    }
    const int s = h ? f.pairs + i : i;
    count[h] = f.average && q.n > 1 ? (double)q.n : 1.0;
    const double S = q.sum / count[h];
    o.values[s] = (float)S;
    gain[h] = S;
    if (f.reference)
      gain[h] -= f.wide ? reinterpret_cast<const double*>(f.reference)[s] : (double)reinterpret_cast<const float*>(f.reference)[s];
  }
  const double D = gain[0] - gain[1], x = f.beta * D - f.margin;
  double l, slope;                         // the pair's loss, and its derivative in D
  if (f.kind == 0) {
    l = (1.0 - f.eps) * log1p_exp(-x) + (f.eps > 0.0 ? f.eps * log1p_exp(x) : 0.0);
    slope = f.beta * (f.eps / (1.0 + exp(-x)) - (1.0 - f.eps) / (1.0 + exp(x)));
  } else if (f.kind == 1) {
    l = x < 1.0 ? 1.0 - x : x >= 1.0 ? 0.0 : x;                // (NaN stays)
    slope = x < 1.0 ? -f.beta : x >= 1.0 ? 0.0 : x;
  } else {
    l = D - 0.5 / f.beta;
    slope = 2.0 * l;
    l *= l;
  }
  if (o.losses) o.losses[i] = (float)l;
  o.by_lp[i] = (float)(slope / count[0]);
  o.by_lp[f.pairs + i] = (float)(-slope / count[1]);
  return Part{l, 1};
}
__global__ __launch_bounds__(kT) void preference_kernel(Preference f, const double* lp, const Kept* kept, LossResults o) {
  __shared__ Part red[kW];
  const Part p = preference_pair<kT>(f, blockIdx.x, lp, kept, o, red);
  if (threadIdx.x || !o.loss) return;
  if (gridDim.x == 1)
    write_loss(p, o.mean, o.loss, o.divisor);
  else
    o.part[blockIdx.x] = p;
}
// few rows, split: joined by the workgroup that goes on with the pairs
constexpr int kJT = 1024;
template <typename T>
__global__ __launch_bounds__(kJT) void join_preference_kernel(Rows a, int parts, const Sums* part, Results rows, Preference f, LossResults o) {
  __shared__ Part red[kJT / 64];
  join_row<T, false, 16>(a, threadIdx.x >> 4, parts, part, rows);
  Part p{0.0, 0};
  for (int i = 0; i < f.pairs; ++i) {
    __syncthreads();                       // the rows, and the pair before
    const Part q = preference_pair<kJT>(f, i, rows.lp64, rows.kept, o, red);
    p.sum += q.sum;
    p.n += q.n;
  }
  if (threadIdx.x == 0 && o.loss) write_loss(p, o.mean, o.loss, o.divisor);
}

struct Policy {
  int64_t rows;
  int T;
  int unit;                                // rows a workgroup: a sequence's T, or any number
  int by_sequence;                         // divide by a sequence's rows and the number of sequences
  const float *old, *advantage, *reference;                    // reference null: no third term
  int adv_div;                             // rows an advantage holds for
  double low, high, kl, ent;               // 1 - clip, 1 + clip_high, the weights
};

// unit u of the rows by a workgroup of N threads; the result is thread 0's
template <int N>
__device__ __forceinline__ Part policy_unit(const Policy& f, int64_t u, const double* lp, const double* ent, const Kept* kept,
                                            const LossResults& o, Part (&red)[N / 64], int (&counts)[N / 64]) {
  constexpr int W = N / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t lo = u * f.unit, hi = lo + f.unit < f.rows ? lo + f.unit : f.rows;
  double share = 1.0;
  if (f.by_sequence) {
    int length = 0;
#pragma unroll 4
    for (int64_t r = lo + threadIdx.x; r < hi; r += N) length += kept[r].live;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) length += __shfl_xor(length, o);
    if (lane == 0) counts[wave] = length;
    __syncthreads();
    length = 0;
    for (int w = 0; w < W; ++w) length += counts[w];
    share = 1.0 / (double)(length > 0 ? length : 1);
  }
  Part p{0.0, 0};
  auto row = [&](int64_t r) {
    // (all asked for at once; what stands where a row is ignored is not looked at)
    const bool live = kept[r].live;
    const float advantage = f.advantage[r / f.adv_div], old = f.old[r], reference = f.reference ? f.reference[r] : 0.f;
    const double x = lp[r], h = o.by_ent ? ent[r] : 0.0;
    double l = 0.0, slope = 0.0;
    if (live) {
      const double A = (double)advantage, ratio = exp(x - (double)old);
      const bool off = (A > 0.0 && ratio > f.high) || (A < 0.0 && ratio < f.low);
      // (a ratio of NaN stays, as does an advantage of NaN)
      l = off ? -(A > 0.0 ? f.high : f.low) * A : -ratio * A;
      slope = off ? 0.0 : -ratio * A;
      if (f.reference) {
        const double d = (double)reference - x, more = expm1(d);
        l += f.kl * (more - d);
        slope -= f.kl * more;
      }
      if (o.by_ent) l -= f.ent * h;
      ++p.n;
    }
    p.sum += l;
    if (o.losses) o.losses[r] = (float)l;
    o.by_lp[r] = (float)(slope * share);
    if (o.by_ent) o.by_ent[r] = live ? (float)(-f.ent * share) : 0.f;
  };
#pragma unroll 2
  for (int64_t r = lo + threadIdx.x; r < hi; r += N) row(r);
  if (!o.loss) return p;                   // (not looked at)
  p = wave_part(p);
  if (lane == 0) red[wave] = p;
  __syncthreads();
  if (threadIdx.x) return Part{0.0, 0};
  for (int w = 1; w < W; ++w) {
    p.sum += red[w].sum;
    p.n += red[w].n;
  }
  if (f.by_sequence) {
    p.sum *= share;
    p.n = p.n > 0;
  }
  return p;
}
__global__ __launch_bounds__(kT) void policy_kernel(Policy f, const double* lp, const double* ent, const Kept* kept, LossResults o) {
  __shared__ Part red[kW];
  __shared__ int counts[kW];
  const Part p = policy_unit<kT>(f, blockIdx.x, lp, ent, kept, o, red, counts);
  if (threadIdx.x || !o.loss) return;
  if (gridDim.x == 1)
    write_loss(p, o.mean, o.loss, o.divisor);
  else
    o.part[blockIdx.x] = p;
}
// few rows, split: joined by the workgroup that goes on with the units
template <typename T, bool ENT>
__global__ __launch_bounds__(kJT) void join_policy_kernel(Rows a, int parts, const Sums* part, Results rows, Policy f, int units,
                                                          LossResults o) {
  __shared__ Part red[kJT / 64];
  __shared__ int counts[kJT / 64];
  join_row<T, ENT, 16>(a, threadIdx.x >> 4, parts, part, rows);
  Part p{0.0, 0};
  for (int u = 0; u < units; ++u) {
    __syncthreads();                       // the rows, and the unit before
    const Part q = policy_unit<kJT>(f, u, rows.lp64, rows.ent64, rows.kept, o, red, counts);
    p.sum += q.sum;
    p.n += q.n;
  }
  if (threadIdx.x == 0 && o.loss) write_loss(p, o.mean, o.loss, o.divisor);
}

// ---- backward ---------------------------------------------------------------------------------------------------------
// a row's gradients in lp and H
struct Upstream {
  const float* by_lp;                      // [r / lp_div * lp_stride]
  const float* by_ent;                     // [r * ent_stride]; null: none
  int64_t lp_div, lp_stride, ent_stride;
  const float* g;                          // a factor of both: [(r / g_div) % g_mod * g_stride]; null: 1
  int64_t g_div, g_mod, g_stride;
  const float* divisor;                    // of that factor
};

// Rows in descending order: the forward pass read the last rows last, and what the caches still hold of them is read first.
// (8 pieces a thread in flight: 379 us for the policy loss above, 386 with 4)
template <typename T, bool ENT, int N>
__global__ __launch_bounds__(kThreads<N>) void backward_kernel(Rows a, int parts, const Kept* kept, Upstream up, T* dz, int past) {
  constexpr int E = kE<T>, U = 8;
  const int tid = threadIdx.x % N;
  const int at = N == 64 ? (int)blockIdx.x * kW + (int)(threadIdx.x >> 6) : N == kT ? (int)blockIdx.x / parts : (int)blockIdx.x;
  const int which = N == kT ? (int)blockIdx.x % parts : 0;
  if (at >= a.rows) return;
  const int r = a.rows - 1 - at;
  T* out = dz + (int64_t)r * a.V;
  const Cut c = cut_row(out, a.V, which, N == kT ? parts : 1);  // (by the output's 16-byte boundaries)
  uint4* to = reinterpret_cast<uint4*>(out + c.head);
  auto store = [&](int p, const uint4& o) {
    if (past)
      __builtin_nontemporal_store(words{o.x, o.y, o.z, o.w}, reinterpret_cast<words*>(to + p));
    else
      to[p] = o;
  };
  const Kept k = kept[r];
  float ga = 0.f, ge = 0.f;
  if (k.live) {                            // uniform
    const float g = up.g ? up.g[(r / up.g_div) % up.g_mod * up.g_stride] / (up.divisor ? *up.divisor : 1.f) : 1.f;
    ga = g * up.by_lp[r / up.lp_div * up.lp_stride];
    if (ENT) ge = g * up.by_ent[r * up.ent_stride];
  }
  // no gradient, whatever the row holds; or none in a row whose probabilities are numbers
  if (!k.live || (ga == 0.f && ge == 0.f && k.inv <= 3.4028234e38f)) {
    for (int p = c.p0 + tid; p < c.p1; p += N) store(p, make_uint4(0u, 0u, 0u, 0u));
    if (tid < c.singles) Elem<T>::store(out + c.single(tid, a.V), 0.f);
    return;
  }
  const T* z = row_of<T>(a, r);
  const int64_t y = whole(a.tokens, a.wide, r);
  const float ref = finite_ref(k.m);
  // dz = power (E (f0 + f1 times the exponent in base 2) + [v = y] fy). The power of 1 / tau, up to 2^126, comes last, where it rounds
  // nothing: inside f0 and f1 it would overflow where E is 0 or the two cancel. (us, all of 1 / tau inside / so: 2048 rows of 50257 bf16
  // with entropies 84.2 / 84.8, 16384 of 4000 47.8 / 48.5; error of 300 fp32 rows at tau 0.9 6.1e-8 / 3.6e-8 of the gradient's norm, the
  // whole of 1 / tau in fp32 behind the sum 5.9e-8.)
  const double inv = (double)k.inv * a.part;
  const float f0 = (float)(((double)ge * k.lean - (double)ga) * inv), f1 = (float)(-(double)ge * kLn2 * inv), fy = (float)(ga * a.part);
  auto value = [&](float x) {
    const Exponent h = exponent_of<kFull<T>>(x - ref, a.c);
    const float e = exp_of<kFull<T>>(h);
    return ENT ? e * __builtin_fmaf(f1, fmaxf(h.h, kFar), f0) : e * f0;
  };
  const int yp = y >= c.head && y < a.V ? (int)(y - c.head) / E : -1, yj = (int)(y - c.head) % E;
  const T* from = z + c.head;
  auto put = [&](int p, const uint4& q) {
    float x[E];
    unpack<T>(q, x);
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = value(x[j]);
    if (p == yp) {
#pragma unroll
      for (int j = 0; j < E; ++j) x[j] += j == yj ? fy : 0.f;
    }
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] *= a.power;
    store(p, pack<T>(x));
  };
  int p = c.p0 + tid;
  for (; p + (U - 1) * N < c.p1; p += U * N) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = load16(from + (int64_t)(p + u * N) * E);
#pragma unroll
    for (int u = 0; u < U; ++u) put(p + u * N, q[u]);
  }
  for (; p < c.p1; p += N) put(p, load16(from + (int64_t)p * E));
  if (tid < c.singles) {
    const int i = c.single(tid, a.V);
    Elem<T>::store(out + i, (value(Elem<T>::load(z + i)) + (i == y ? fy : 0.f)) * a.power);
  }
}

// ---- sizes ------------------------------------------------------------------------------------------------------------
// workgroups a row: enough for 1024 in all, each with at least two pieces a thread
int64_t row_bytes(int V, int dtype) { return (int64_t)V * (dtype == DH_BF16 ? 2 : 4); }
int parts_of(int64_t rows, int V, int dtype) {
  int64_t p = 1024 / (rows > 0 ? rows : 1);
  const int64_t most = (row_bytes(V, dtype) + 15) / 16 / (2 * kT);
  if (p > most) p = most;
  if (p > kMaxParts) p = kMaxParts;
  return p < 1 ? 1 : (int)p;
}
// ... of the forward pass, where split rows cost a launch that joins them: few and long ones are split. us, whole / split: bf16 with
// entropies, V 8192 1 row 4.7 / 6.6, 512 rows 7.2 / 10.3; V 50257 1 row 7.7 / 7.3 (and less of the host's time), 16 8.6 / 8.3, 64 9.4 /
// 10.0, 256 11.1 / 14.6; V 80000 16 12.2 / 8.9, 128 13.4 / 13.1, 256 15.6 / 17.5; V 151936 64 17.3 / 12.7, 128 18.3 / 17.4, 256 24.1 /
// 27.8. fp32, V 50257 64 12.8 / 12.1, 128 13.2 / 14.3.
constexpr int64_t kWhole = 112 << 10;
int forward_parts(int64_t rows, int V, int dtype) {
  return rows >= 256 || row_bytes(V, dtype) <= kWhole * (rows < 64 ? 1 : rows / 64) ? 1 : parts_of(rows, V, dtype);
}
// A wave a row: rows of up to this many bytes, as many as fill the card so. us with a wave and with a workgroup a row, 16384 rows of
// bf16: V 6000 forward 42 and 58, backward 82 and 98; 8000 51 and 64, 114 and 110; 12000 74 and 95, 169 and 147; 16000 93 and 105, 224
// and 206. fp32, V 4000 49 and 63, 112 and 134; 8000 91 and 100, 222 and 212.
constexpr int kWaveForward = 32768, kWaveBackward = 16384;
bool by_waves(int64_t rows, int V, int dtype, int bytes) { return row_bytes(V, dtype) <= bytes && rows >= 1024; }

int check(const char* who, int dtype, const Rows& a, int token_bits, double tau) {
  DH_REQUIRE(dtype == DH_F32 || dtype == DH_BF16, DH_ERR_UNSUPPORTED_DTYPE, "%s: dtype %d", who, dtype);
  DH_REQUIRE(token_bits == 32 || token_bits == 64, DH_ERR_UNSUPPORTED_DTYPE, "%s: tokens of %d bits", who, token_bits);
  DH_REQUIRE(a.rows >= 0 && a.rows < (1 << 22) && a.T >= 1 && a.V >= 1 && a.V <= (1 << 24), DH_ERR_UNSUPPORTED_SHAPE,
             "%s: %d rows (-1: too many), T=%d V=%d", who, a.rows, a.T, a.V);
  DH_REQUIRE(tau >= 0x1p-126 && tau <= 0x1p126, DH_ERR_INVALID_ARG, "%s: temperature %g", who, tau);
  DH_REQUIRE(a.rows == 0 || (a.logits && a.tokens), DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE((uintptr_t)a.logits % (dtype == DH_BF16 ? 2 : 4) == 0 && (uintptr_t)a.tokens % (token_bits / 8) == 0,
             DH_ERR_INVALID_ARG, "%s: operands not aligned to their elements", who);
  return 0;
}

Rows rows_of(const void* logits, int64_t sb, int64_t st, int64_t B, int T, int V, const void* tokens, int token_bits,
             int64_t ignore, double tau) {
  Rows a;
  a.logits = logits;
  a.sb = sb;
  a.st = st;
  a.rows = B < 0 || T < 0 || (T > 0 && B >= ((int64_t)1 << 22) / T + 1) ? -1 : (int)(B * T);       // -1: too many
  a.T = T;
  a.V = V;
  a.tokens = tokens;
  a.wide = token_bits == 64;
  a.ignore = ignore;
  a.inv_tau = 1.0 / tau;
  int exponent = 0;
  a.part = 2.0 * frexp(a.inv_tau, &exponent);
  a.power = (float)ldexp(1.0, exponent - 1);
  const double c = kLog2e / tau;
  a.c = Scale{(float)c, (float)(c - (double)(float)c)};
  return a;
}

// joined: whether rows that are split are joined here
template <typename T, bool ENT>
int forward(const char* who, int dtype, const Rows& a, const Results& o, void* ws, bool joined, hipStream_t s) {
  if (by_waves(a.rows, a.V, dtype, kWaveForward)) {
    forward_kernel<T, ENT, 64><<<dim3((unsigned)((a.rows + kW - 1) / kW)), dim3(kT), 0, s>>>(a, 1, nullptr, o);
    return dh_check_launch(who);
  }
  const int parts = forward_parts(a.rows, a.V, dtype);
  if (parts == 1) {
    forward_kernel<T, ENT, kWide><<<dim3((unsigned)a.rows), dim3(kWide), 0, s>>>(a, 1, nullptr, o);
    return dh_check_launch(who);
  }
  forward_kernel<T, ENT, kT><<<dim3((unsigned)a.rows * parts), dim3(kT), 0, s>>>(a, parts, (Sums*)ws, o);
  if (int st = dh_check_launch(who)) return st;
  if (!joined) return 0;
  join_kernel<T, ENT><<<dim3((unsigned)((a.rows + kT / 16 - 1) / (kT / 16))), dim3(kT), 0, s>>>(a, parts, (const Sums*)ws, o);
  return dh_check_launch(who);
}
int forward(const char* who, int dtype, const Rows& a, bool ent, const Results& o, void* ws, bool joined, hipStream_t s) {
  if (a.rows == 0) return 0;
  if (dtype == DH_BF16)
    return ent ? forward<bf16_t, true>(who, dtype, a, o, ws, joined, s) : forward<bf16_t, false>(who, dtype, a, o, ws, joined, s);
  return ent ? forward<float, true>(who, dtype, a, o, ws, joined, s) : forward<float, false>(who, dtype, a, o, ws, joined, s);
}
// Split rows few enough for one workgroup to join them on its way to the loss, in units of its own or not at all: a launch less, us so /
// with a launch that joins them: V 50257 fp32, one pair of 24 12.3 / 13.5 where two pairs of 8 15.1 / 15.7, four 23.4 / 18.1.
constexpr int kFewRows = kJT / 16, kFewUnits = 2;
int few_parts(const Rows& a, int64_t units, int dtype) {
  const int parts = a.rows > 0 && a.rows <= kFewRows && units <= kFewUnits ? forward_parts(a.rows, a.V, dtype) : 1;
  return parts > 1 ? parts : 0;
}

template <typename T, bool ENT>
int backward(const char* who, int dtype, const Rows& a, const Kept* kept, const Upstream& up, void* dz, hipStream_t s) {
  const int past = (int64_t)a.rows * a.V * (int)sizeof(T) >= kPast;
  if (by_waves(a.rows, a.V, dtype, kWaveBackward)) {
    backward_kernel<T, ENT, 64><<<dim3((unsigned)((a.rows + kW - 1) / kW)), dim3(kT), 0, s>>>(a, 1, kept, up, (T*)dz, past);
    return dh_check_launch(who);
  }
  const int parts = parts_of(a.rows, a.V, dtype);
  if (parts == 1) {
    backward_kernel<T, ENT, kWide><<<dim3((unsigned)a.rows), dim3(kWide), 0, s>>>(a, 1, kept, up, (T*)dz, past);
    return dh_check_launch(who);
  }
  backward_kernel<T, ENT, kT><<<dim3((unsigned)a.rows * parts), dim3(kT), 0, s>>>(a, parts, kept, up, (T*)dz, past);
  return dh_check_launch(who);
}

// the workspace of a call: the sums of split rows, lp (and H) in fp64, a loss's parts
struct Layout {
  int64_t lp64, ent64, part, bytes;
};
constexpr int64_t kUnit = 256;             // rows a workgroup of the policy loss where sequences do not matter
Layout layout_of(int op, int64_t rows, int64_t units, int V, int dtype, bool ent) {
  Layout l;
  const int parts = forward_parts(rows, V, dtype);
  l.lp64 = parts > 1 ? (rows * parts * (int64_t)sizeof(Sums) + 7) / 8 * 8 : 0;
  l.ent64 = l.lp64 + (op ? rows * 8 : 0);
  l.part = l.ent64 + (op && ent ? rows * 8 : 0);
  l.bytes = l.part + (op ? units * (int64_t)sizeof(Part) : 0);
  return l;
}
bool fits(int64_t rows, int V) { return rows >= 0 && rows < (1 << 22) && V >= 1 && V <= (1 << 24); }

}  // namespace

extern "C" int64_t dh_logprob_workspace_bytes(int dtype, int64_t rows, int V) {
  return fits(rows, V) ? layout_of(0, rows, 0, V, dtype, false).bytes : -1;
}

extern "C" int dh_logprob_fwd(int dtype, const void* logits, int64_t stride_b, int64_t stride_t, int64_t B, int T, int V,
                              const void* tokens, int token_bits, int64_t ignore_index, double temperature, float* logprob,
                              float* entropy, void* row_kept, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "dh_logprob_fwd";
  const Rows a = rows_of(logits, stride_b, stride_t, B, T, V, tokens, token_bits, ignore_index, temperature);
  if (int st = check(who, dtype, a, token_bits, temperature)) return st;
  DH_REQUIRE(a.rows == 0 || logprob, DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE((uintptr_t)logprob % 4 == 0 && (uintptr_t)entropy % 4 == 0 && (uintptr_t)row_kept % 16 == 0, DH_ERR_INVALID_ARG,
             "%s: results not aligned to their elements", who);
  const int64_t need = dh_logprob_workspace_bytes(dtype, a.rows, V);
  DH_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 8 == 0)), DH_ERR_INVALID_ARG,
             "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes, (long long)need);
  return forward(who, dtype, a, entropy != nullptr, Results{logprob, entropy, nullptr, nullptr, (Kept*)row_kept}, workspace,
                 true, (hipStream_t)stream);
}

extern "C" int dh_logprob_bwd(int dtype, const void* logits, int64_t stride_b, int64_t stride_t, int64_t B, int T, int V,
                              const void* tokens, int token_bits, int64_t ignore_index, double temperature, const void* row_kept,
                              const float* by_logprob, int64_t logprob_div, int64_t logprob_stride, const float* by_entropy,
                              int64_t entropy_stride, const float* dloss, int64_t dloss_div, int64_t dloss_mod,
                              int64_t dloss_stride, const float* divisor, void* dlogits, void* stream) {
  const char* who = "dh_logprob_bwd";
  const Rows a = rows_of(logits, stride_b, stride_t, B, T, V, tokens, token_bits, ignore_index, temperature);
  if (int st = check(who, dtype, a, token_bits, temperature)) return st;
  if (a.rows == 0) return 0;
  DH_REQUIRE(row_kept && (uintptr_t)row_kept % 16 == 0 && by_logprob && dlogits, DH_ERR_INVALID_ARG,
             "%s: null or unaligned pointer argument", who);
  DH_REQUIRE(logprob_div >= 1 && logprob_stride >= 0 && entropy_stride >= 0 &&
                 (!dloss || (dloss_div >= 1 && dloss_mod >= 1 && dloss_stride >= 0)),
             DH_ERR_INVALID_ARG, "%s: strides and divisors of the gradients", who);
  DH_REQUIRE((uintptr_t)by_logprob % 4 == 0 && (uintptr_t)by_entropy % 4 == 0 && (uintptr_t)dloss % 4 == 0 &&
                 (uintptr_t)divisor % 4 == 0 && (uintptr_t)dlogits % (dtype == DH_BF16 ? 2 : 4) == 0,
             DH_ERR_INVALID_ARG, "%s: operands not aligned to their elements", who);
  const Upstream up{by_logprob, by_entropy, logprob_div, logprob_stride, entropy_stride, dloss, dloss_div, dloss_mod,
                    dloss_stride, divisor};
  const Kept* kept = (const Kept*)row_kept;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DH_BF16)
    return by_entropy ? backward<bf16_t, true>(who, dtype, a, kept, up, dlogits, s)
                      : backward<bf16_t, false>(who, dtype, a, kept, up, dlogits, s);
  return by_entropy ? backward<float, true>(who, dtype, a, kept, up, dlogits, s)
                    : backward<float, false>(who, dtype, a, kept, up, dlogits, s);
}

extern "C" int64_t dh_preference_workspace_bytes(int dtype, int64_t pairs, int T, int V) {
  if (pairs < 0 || pairs >= (1 << 21) || T < 0 || (T > 0 && pairs > (1 << 21) / T) || !fits(2 * pairs * T, V)) return -1;
  return layout_of(1, 2 * pairs * T, pairs, V, dtype, false).bytes;
}

extern "C" int dh_preference_fwd(int dtype, const void* logits, int64_t stride_b, int64_t stride_t, int64_t pairs, int T, int V,
                                 const void* tokens, int token_bits, int64_t ignore_index, const void* reference,
                                 int reference_bits, int kind, int average, double beta, double margin, double label_smoothing,
                                 int reduction, float* pair_loss, float* sums, float* coef, void* row_kept, float* loss,
                                 float* divisor, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "dh_preference_fwd";
  DH_REQUIRE(pairs >= 0 && T >= 0, DH_ERR_UNSUPPORTED_SHAPE, "%s: %lld pairs of %d", who, (long long)pairs, T);
  const int64_t need = dh_preference_workspace_bytes(dtype, pairs, T, V);
  DH_REQUIRE(need >= 0, DH_ERR_UNSUPPORTED_SHAPE, "%s: %lld pairs of %d rows, V=%d", who, (long long)pairs, T, V);
  const Rows a = rows_of(logits, stride_b, stride_t, T ? 2 * pairs : 0, T ? T : 1, V, tokens, token_bits, ignore_index, 1.0);
  if (int st = check(who, dtype, a, token_bits, 1.0)) return st;
  DH_REQUIRE(kind >= 0 && kind <= 2 && reduction >= 0 && reduction <= 2, DH_ERR_INVALID_ARG, "%s: kind %d, reduction %d", who, kind,
             reduction);
  DH_REQUIRE(beta > 0.0 && beta < INFINITY && margin > -INFINITY && margin < INFINITY && label_smoothing >= 0.0 &&
                 label_smoothing <= 0.5, DH_ERR_INVALID_ARG, "%s: beta %g, margin %g, label smoothing %g", who, beta, margin, label_smoothing);
  DH_REQUIRE(!reference || reference_bits == 32 || reference_bits == 64, DH_ERR_UNSUPPORTED_DTYPE, "%s: reference of %d bits",
             who, reference_bits);
  DH_REQUIRE(pairs == 0 || (sums && coef), DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE((a.rows == 0 || row_kept) && (uintptr_t)row_kept % 16 == 0, DH_ERR_INVALID_ARG, "%s: null or unaligned pointer argument", who);
  DH_REQUIRE(reduction ? loss && divisor : pairs == 0 || pair_loss, DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE((uintptr_t)pair_loss % 4 == 0 && (uintptr_t)sums % 4 == 0 && (uintptr_t)coef % 4 == 0 && (uintptr_t)loss % 4 == 0 &&
                 (uintptr_t)divisor % 4 == 0 && (!reference || (uintptr_t)reference % (reference_bits / 8) == 0),
             DH_ERR_INVALID_ARG, "%s: operands not aligned to their elements", who);
  DH_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 8 == 0)), DH_ERR_INVALID_ARG,
             "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes, (long long)need);
  hipStream_t s = (hipStream_t)stream;
  const Layout l = layout_of(1, a.rows, pairs, V, dtype, false);
  char* ws = (char*)workspace;
  double* lp = (double*)(ws + l.lp64);
  Part* part = (Part*)(ws + l.part);
  Kept* kept = (Kept*)row_kept;
  const Results rows{nullptr, nullptr, lp, nullptr, kept};
  const int parts = few_parts(a, pairs, dtype);
  if (int st = forward(who, dtype, a, false, rows, ws, parts == 0, s)) return st;
  const LossResults o{reduction ? nullptr : pair_loss, sums, coef, nullptr, part, reduction == 1, reduction ? loss : nullptr, divisor};
  const Preference f{(int)pairs, T, kind, average, beta, margin, label_smoothing, reference, reference_bits == 64};
  if (parts) {
    if (dtype == DH_BF16)
      join_preference_kernel<bf16_t><<<dim3(1), dim3(kJT), 0, s>>>(a, parts, (const Sums*)ws, rows, f, o);
    else
      join_preference_kernel<float><<<dim3(1), dim3(kJT), 0, s>>>(a, parts, (const Sums*)ws, rows, f, o);
    return dh_check_launch(who);
  }
  if (pairs) {
    preference_kernel<<<dim3((unsigned)pairs), dim3(kT), 0, s>>>(f, lp, kept, o);
    if (int st = dh_check_launch(who)) return st;
  }
  if (!reduction || pairs == 1) return 0;
  reduce_kernel<<<dim3(1), dim3(pairs > 64 ? 1024 : 64), 0, s>>>(part, pairs, reduction == 1, loss, divisor);
  return dh_check_launch(who);
}

extern "C" int64_t dh_policy_workspace_bytes(int dtype, int64_t B, int T, int V, int entropy) {
  if (B < 0 || T < 0 || (T > 0 && B > ((int64_t)1 << 22) / T) || !fits(B * T, V)) return -1;
  const int64_t rows = B * T, units = (rows + kUnit - 1) / kUnit;
  return layout_of(1, rows, T && B > units ? B : units, V, dtype, entropy != 0).bytes;
}

extern "C" int dh_policy_fwd(int dtype, const void* logits, int64_t stride_b, int64_t stride_t, int64_t B, int T, int V,
                             const void* tokens, int token_bits, int64_t ignore_index, double temperature,
                             const float* old_logprob, const float* advantage, int per_sequence,
                             const float* reference_logprob, double clip, double clip_high, double kl_weight,
                             double entropy_weight, int reduction, float* row_loss, float* logprob, float* by_logprob,
                             float* by_entropy, void* row_kept, float* loss, float* divisor, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const char* who = "dh_policy_fwd";
  DH_REQUIRE(B >= 0 && T >= 0, DH_ERR_UNSUPPORTED_SHAPE, "%s: B=%lld T=%d", who, (long long)B, T);
  const int64_t need = dh_policy_workspace_bytes(dtype, B, T, V, by_entropy != nullptr);
  DH_REQUIRE(need >= 0, DH_ERR_UNSUPPORTED_SHAPE, "%s: B=%lld T=%d V=%d", who, (long long)B, T, V);
  const Rows a = rows_of(logits, stride_b, stride_t, T ? B : 0, T ? T : 1, V, tokens, token_bits, ignore_index, temperature);
  if (int st = check(who, dtype, a, token_bits, temperature)) return st;
  DH_REQUIRE(reduction >= 0 && reduction <= 3, DH_ERR_INVALID_ARG, "%s: reduction %d", who, reduction);
  DH_REQUIRE(clip >= 0.0 && clip <= 1.0 && clip_high >= 0.0 && clip_high < INFINITY && kl_weight >= 0.0 && kl_weight < INFINITY &&
                 entropy_weight > -INFINITY && entropy_weight < INFINITY,
             DH_ERR_INVALID_ARG, "%s: clip %g and %g, weights %g and %g", who, clip, clip_high, kl_weight, entropy_weight);
  DH_REQUIRE(by_entropy || entropy_weight == 0.0, DH_ERR_INVALID_ARG, "%s: an entropy weight of %g, and no by_entropy", who, entropy_weight);
  DH_REQUIRE(a.rows == 0 || reference_logprob || kl_weight == 0.0, DH_ERR_INVALID_ARG, "%s: a KL weight of %g without a reference", who, kl_weight);
  DH_REQUIRE(a.rows == 0 || (old_logprob && advantage && logprob && by_logprob && row_kept), DH_ERR_INVALID_ARG,
             "%s: null pointer argument", who);
  DH_REQUIRE(reduction ? loss && divisor : a.rows == 0 || row_loss, DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE((uintptr_t)old_logprob % 4 == 0 && (uintptr_t)advantage % 4 == 0 && (uintptr_t)reference_logprob % 4 == 0 &&
                 (uintptr_t)row_loss % 4 == 0 && (uintptr_t)logprob % 4 == 0 && (uintptr_t)by_logprob % 4 == 0 &&
                 (uintptr_t)by_entropy % 4 == 0 && (uintptr_t)row_kept % 16 == 0 && (uintptr_t)loss % 4 == 0 &&
                 (uintptr_t)divisor % 4 == 0,
             DH_ERR_INVALID_ARG, "%s: operands not aligned to their elements", who);
  DH_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 8 == 0)), DH_ERR_INVALID_ARG,
             "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes, (long long)need);
  hipStream_t s = (hipStream_t)stream;
  const bool ent = by_entropy != nullptr, by_sequence = reduction == 3, mean = reduction == 1 || by_sequence;
  const int64_t units = by_sequence ? (T ? B : 0) : (a.rows + kUnit - 1) / kUnit;
  const Layout l = layout_of(1, a.rows, units, V, dtype, ent);
  char* ws = (char*)workspace;
  double *lp = (double*)(ws + l.lp64), *h = ent ? (double*)(ws + l.ent64) : nullptr;
  Part* part = (Part*)(ws + l.part);
  Kept* kept = (Kept*)row_kept;
  const Results rows{logprob, nullptr, lp, h, kept};
  const int parts = few_parts(a, units, dtype);
  if (int st = forward(who, dtype, a, ent, rows, ws, parts == 0, s)) return st;
  const LossResults o{reduction ? nullptr : row_loss, nullptr, by_logprob, by_entropy, part, mean, reduction ? loss : nullptr, divisor};
  const Policy f{a.rows, T, by_sequence ? T : (int)kUnit, by_sequence, old_logprob, advantage,
                 kl_weight > 0.0 ? reference_logprob : nullptr, per_sequence ? T : 1, 1.0 - clip, 1.0 + clip_high, kl_weight,
                 entropy_weight};
  if (parts) {
    const Sums* sums = (const Sums*)ws;
    const dim3 one(1), block(kJT);
    if (dtype == DH_BF16 && ent)
      join_policy_kernel<bf16_t, true><<<one, block, 0, s>>>(a, parts, sums, rows, f, (int)units, o);
    else if (dtype == DH_BF16)
      join_policy_kernel<bf16_t, false><<<one, block, 0, s>>>(a, parts, sums, rows, f, (int)units, o);
    else if (ent)
      join_policy_kernel<float, true><<<one, block, 0, s>>>(a, parts, sums, rows, f, (int)units, o);
    else
      join_policy_kernel<float, false><<<one, block, 0, s>>>(a, parts, sums, rows, f, (int)units, o);
    return dh_check_launch(who);
  }
  if (units) {
    policy_kernel<<<dim3((unsigned)units), dim3(kT), 0, s>>>(f, lp, h, kept, o);
    if (int st = dh_check_launch(who)) return st;
  }
  if (!reduction || units == 1) return 0;
  reduce_kernel<<<dim3(1), dim3(units > 64 ? 1024 : 64), 0, s>>>(part, units, mean, loss, divisor);
  return dh_check_launch(who);
}
