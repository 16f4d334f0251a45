// Log-probabilities of given tokens from the last hidden states and the vocabulary head's weight, without the logits in memory,
// for gfx950 (inference). For a row h (d wide), the weight W (V, d), a temperature tau and the row's token y:
//   z_v = h . W_v (fp32 sums; round_logits: rounded to the operands' type),  p = softmax(z / tau)
//   lp = log p_y,  H = - sum_v p_v log p_v
// A row whose token is ignore_index has lp = H = 0. It is not computed, but by few_kernel, whose join puts the zeros in its place.
//
// The product's tiles stay in the accumulators. A lane of a tile holds some columns of its rows and keeps, over all the tiles that
// its workgroup takes of a row, the running maximum m of z and the sums of e = exp((z - m) / tau) and of e times its exponent;
// lanes are joined when the workgroup ends with the row, workgroups by a last launch. A token's own logit is written by the lane
// that meets it. So a row leaves a few numbers for each workgroup instead of V logits. V 50257, d 1024, bf16: 5300 rows 427 us (1277
// TFLOP/s of products, on the matrix cores in 66% of the cycles), 16 rows 23 (the weight at 5.6 TB/s, and the join).
//
// Launches: the rows that count, in their order, and how the tiles are dealt out (compact_kernel; their number is known on the
// device only; up to 1024 rows the product's workgroups do this themselves); the product; the join. Up to 32 rows that are aligned, of
// whole 128-byte lines and beside the rings in LDS (64 KB of them, padded to 16 or 32 rows): the product (few_kernel, the weight's bytes
// bound it) and the join.

#include "dh_rows.h"

#include <utility>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kFar = -200.f;             // an exponent in base 2 whose power is 0: stands in for -inf where it is a factor
constexpr int kRowBytes = 128;             // bytes of a row of a K tile

struct State {
  float m, s, t;                           // the maximum, sums of e and of e times its exponent in base 2
};
__device__ __forceinline__ void move_to(State& v, float ref, float c) {
  const float h = (v.m - ref) * c, f = exp2_hw(h);
  v.t = f * __builtin_fmaf(v.s, fmaxf(h, kFar), v.t);          // (no sum yet: 0 (0 kFar + 0))
  v.s *= f;
}
__device__ __forceinline__ State join(State a, State b, float c) {
  const float m = fmaxf(a.m, b.m), ref = finite_ref(m);
  move_to(a, ref, c);
  move_to(b, ref, c);
  return State{m, a.s + b.s, a.t + b.t};
}
// N values of a row into its sums
template <bool ENT, int N>
__device__ __forceinline__ void add(State& v, const float (&x)[N], float c) {
  float most = v.m;
#pragma unroll
  for (int i = 0; i < N; ++i) most = fmaxf(most, x[i]);
  const float ref = finite_ref(most), back = (v.m - ref) * c, f = exp2_hw(back);
  if (ENT) v.t = f * __builtin_fmaf(v.s, fmaxf(back, kFar), v.t);
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float h = (x[i] - ref) * c, e = exp2_hw(h);
    s = i ? s + e : e;
    if (ENT) t = i ? __builtin_fmaf(e, fmaxf(h, kFar), t) : e * fmaxf(h, kFar);
  }
  v.m = most;
  v.s = __builtin_fmaf(v.s, f, s);
  if (ENT) v.t += t;
}

// how the product's tiles are dealt out: the live rows' tiles (mt of BM rows) times parts of the vocabulary's tiles
struct Plan {
  int live, mt, parts, per;                // per: column tiles of a part
};
struct Args {
  const void* h;
  int64_t ldh;
  const void* w;
  int64_t ldw;
  int rows, V, K, nt;                      // nt: column tiles
  const void* tokens;
  int wide;
  int64_t ignore;
  int round;                               // bf16 logits
  float c;                                 // log2(e) / tau
  double inv_tau;
  int self;                                // few enough rows for every workgroup of the product to sort them out itself
  Plan* plan;
  int* index;                              // the live rows; null: all
  State* part;                             // [compact row][slots]
  float* zy;                               // [compact row]
  float *lp, *ent;
};

__device__ __forceinline__ int row_at(const Args& a, int i) { return a.index ? a.index[i] : i; }

// ---- the rows that count ----------------------------------------------------------------------------------------------
constexpr int kCT = 1024;
// rows a workgroup: one a thread, more where the workgroups' reads of all rows before their own would add up
int chunk_of(int64_t rows) { return kCT * (int)(rows <= 32768 ? 1 : rows <= (1 << 20) ? rows / 32768 : 32); }

// How n live rows' tiles are dealt out, by a workgroup of N threads: the number of parts whose longest workgroup is shortest, rounds of
// the workgroups times the tiles of a part (and half a tile that beginning and ending one takes).
template <int N>
__device__ __forceinline__ Plan deal(int n, int nt, int bm, int groups, int64_t (&best)[N / 64]) {
  const int tid = threadIdx.x, mt = (n + bm - 1) / bm;
  if (mt == 0) return Plan{0, 0, 1, nt};   // uniform
  int64_t mine = INT64_MAX;
  const int most = max(1, min(nt, 2 * groups / mt));           // (mt p and the cost: at most some 2^27)
  for (int p = tid + 1; p <= most; p += N) {
    const uint32_t per = (uint32_t)(nt + p - 1) / (uint32_t)p, rounds = (uint32_t)(mt * p + groups - 1) / (uint32_t)groups;
    mine = min(mine, (int64_t)(rounds * (2 * per + 1)) << 20 | p);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int64_t other = __shfl_xor(mine, o);
    mine = min(mine, other);
  }
  if ((tid & 63) == 0) best[tid >> 6] = mine;
  __syncthreads();
  mine = best[0];
  for (int w = 1; w < N / 64; ++w) mine = min(mine, best[w]);
  const int p = __builtin_amdgcn_readfirstlane((int)(mine & 0xfffff)), per = (nt + p - 1) / p;
  return Plan{n, mt, (nt + per - 1) / per, per};
}
__device__ __forceinline__ bool counts(const Args& a, int r) { return whole(a.tokens, a.wide, r) != a.ignore; }
__device__ __forceinline__ void skip_row(const Args& a, int r) {
  a.lp[r] = 0.f;
  if (a.ent) a.ent[r] = 0.f;
}
// the live rows of [lo, hi), in their order, to list[at ...]; returns at and their number. write: whether the others' results are
template <int N, typename I>
__device__ __forceinline__ int sort_out(const Args& a, int lo, int hi, int at, I* list, bool write, int (&red)[N / 64]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int r0 = lo; r0 < hi; r0 += N) {    // uniform
    const int r = r0 + tid;
    const bool in = r < hi, on = in && counts(a, r);
    const uint64_t mask = __builtin_amdgcn_ballot_w64(on);
    __syncthreads();
    if (lane == 0) red[wave] = __popcll(mask);
    __syncthreads();
    int place = at + __popcll(mask & ((1ull << lane) - 1)), all = 0;
    for (int w = 0; w < N / 64; ++w) {
      if (w < wave) place += red[w];
      all += red[w];
    }
    if (on) list[place] = (I)r;
    if (write && in && !on) skip_row(a, r);
    at += __builtin_amdgcn_readfirstlane(all);
  }
  return at;
}

// A workgroup counts the live rows before its own and places those of its chunk. The last one deals out the tiles.
__global__ __launch_bounds__(kCT) void compact_kernel(Args a, int bm, int groups, int chunk) {
  __shared__ int red[kCT / 64];
  __shared__ int64_t best[kCT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lo = blockIdx.x * chunk, hi = min(lo + chunk, a.rows);
  int before = 0;
#pragma unroll 8
  for (int r = tid; r < lo; r += kCT) before += counts(a, r);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
  if (lane == 0) red[wave] = before;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kCT / 64; ++w) base += red[w];
  const int n = sort_out<kCT>(a, lo, hi, __builtin_amdgcn_readfirstlane(base), a.index, true, red);
  if ((int)blockIdx.x != (int)gridDim.x - 1) return;
  const Plan q = deal<kCT>(n, a.nt, bm, groups, best);
  if (tid == 0) *a.plan = q;
}

// What a workgroup of the product begins with: the plan, and where its rows are listed. Up to kSelf rows every one sorts them out
// itself, which takes less than a launch before it (128 rows 31.6 us with that, 29.0 so), and the first leaves plan and list for the join.
constexpr int kSelf = 1024;
typedef uint16_t listed;                   // (2 KB of LDS: four 64 x 64 staged workgroups on a CU, three with 4 KB)
template <int N>
__device__ __forceinline__ Plan begin(const Args& a, int bm, listed* list, int (&red)[N / 64], int64_t (&best)[N / 64]) {
  if (!a.self) return *a.plan;
  const bool first = blockIdx.x == 0;
  const int n = sort_out<N>(a, 0, a.rows, 0, list, first, red);
  const Plan q = deal<N>(n, a.nt, bm, gridDim.x, best);
  __syncthreads();
  if (first) {
    for (int i = threadIdx.x; i < n; i += N) a.index[i] = list[i];
    if (threadIdx.x == 0) *a.plan = q;
    __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));          // s_waitcnt vmcnt(0): what follows counts its own loads
  }
  return q;
}

// Item i of the tiles dealt out: row tile m, part p. Row tiles in groups of eight, a group's parts one after another, its row tiles
// inside a part: the 32 workgroups that one XCD takes (i = a contiguous eighth of a round) meet 8 row tiles and 4 parts.
__device__ __forceinline__ void item_at(const Plan& q, int i, int& m, int& p) {
  const int g = i / (8 * q.parts), rest = i - g * 8 * q.parts, width = min(8, q.mt - 8 * g);
  p = rest / width;
  m = 8 * g + (rest - p * width);
}
// item of a workgroup in a round: XCD id % 8 takes a contiguous eighth
__device__ __forceinline__ int item_of(int id, int groups) { return (id & 7) * (groups >> 3) + (id >> 3); }

// the token of a row as a column, -1: none
__device__ __forceinline__ int column_of(const Args& a, int r) {
  const int64_t k = whole(a.tokens, a.wide, r);
  return k >= 0 && k < a.V ? (int)k : -1;
}

// ---- the rows' results ------------------------------------------------------------------------------------------------
template <bool ENT>
__device__ __forceinline__ void finish(const Args& a, int r, const State& v, float zy, bool bad) {
  const double nan = __builtin_nan("");
  const double ls = log((double)v.s);
  a.lp[r] = (float)(bad ? nan : ((double)zy - (double)v.m) * a.inv_tau - ls);
  if (ENT) a.ent[r] = (float)(bad ? nan : ls - (double)v.t * kLn2 / (double)v.s);
}

// a wave a live row: its slots in their order, kAhead a lane at a time
template <bool ENT>
__global__ __launch_bounds__(256) void join_kernel(Args a, int slots_a_part, int slots_if_all) {
  constexpr int kAhead = 4;
  const int lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= a.rows) return;
  // (asked for at once; behind the last live row there is anything)
  const int live = a.plan ? a.plan->live : a.rows, slots = a.plan ? a.plan->parts * slots_a_part : slots_if_all;
  const int r = row_at(a, i);
  const float z = a.zy[i];
  if (i >= live) return;
  const int64_t y = whole(a.tokens, a.wide, r);
  const bool bad = y < 0 || y >= a.V;
  const float zy = bad ? 0.f : z;
  const State* part = a.part + (int64_t)i * slots;
  State v{-INFINITY, 0.f, 0.f};
  for (int k = lane; k < slots; k += 64 * kAhead) {
    State q[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) q[u] = k + 64 * u < slots ? part[k + 64 * u] : State{-INFINITY, 0.f, 0.f};
    float m = v.m;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) m = fmaxf(m, q[u].m);
    const float ref = finite_ref(m);
    move_to(v, ref, a.c);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      move_to(q[u], ref, a.c);
      v.s += q[u].s;
      v.t += q[u].t;
    }
    v.m = m;
  }
  const float m = wave_max(v.m);
  move_to(v, finite_ref(m), a.c);
  v = State{m, wave_sum(v.s), ENT ? wave_sum(v.t) : 0.f};
  if (lane) return;
  if (y == a.ignore) {                     // (rows that were not sorted out)
    a.lp[r] = 0.f;
    if (ENT) a.ent[r] = 0.f;
    return;
  }
  finish<ENT>(a, r, v, zy, bad);
}

// ---- a workgroup's tiles ------------------------------------------------------------------------------------------------
// acc[j][i] of lane (r, g): columns n + 16 j + 4 g .. + 3 of row 16 i + r, n the wave's first column
// ys: the tokens of the wave's rows, -1: none; zs: their logits, written as they are met
template <bool ENT, int TM, int TN>
__device__ __forceinline__ void take_tile(const Args& a, f32x4 (&acc)[TN][TM], State (&st)[TM], const int* ys, float* zs, int n) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  int y[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) y[i] = ys[16 * i + r];
  if (a.round) {                           // uniform
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][i][e] = Elem<bf16_t>::round(acc[j][i][e]);
  }
  // a token of these rows among these columns: its logit
  bool some = false;
#pragma unroll
  for (int i = 0; i < TM; ++i) some |= y[i] >= n && y[i] < n + 16 * TN;
  if (__builtin_amdgcn_ballot_w64(some)) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int k = y[i] - (n + 16 * j + 4 * g);
        if (k >= 0 && k < 4) {
          float z = acc[j][i][0];
#pragma unroll
          for (int e = 1; e < 4; ++e) z = k == e ? acc[j][i][e] : z;
          zs[16 * i + r] = z;
        }
      }
  }
  if (n + 16 * TN > a.V) {                 // uniform: columns past the vocabulary
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + 16 * j + 4 * g + e >= a.V) acc[j][i][e] = -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    float x[4 * TN];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * j + e] = acc[j][i][e];
    add<ENT>(st[i], x, a.c);
  }
}
// the lanes' sums of each row joined and written to the row's slot
template <int TM>
__device__ __forceinline__ void leave_rows(const Args& a, State (&st)[TM], int row0, int live, int slots, int slot) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    State v = st[i];
#pragma unroll
    for (int o = 16; o <= 32; o <<= 1) v = join(v, State{__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.t, o)}, a.c);
    const int row = row0 + 16 * i + (lane & 15);
    if (lane < 16 && row < live) a.part[(int64_t)row * slots + slot] = v;
  }
}

// a row's token among the columns [lo, hi) that a workgroup took: its logit
__device__ __forceinline__ void leave_token(const Args& a, int y, float z, int row, int64_t lo, int64_t hi) {
  if (y >= lo && y < hi) a.zy[row] = z;
}

// ---- any type, width, alignment -----------------------------------------------------------------------------------------
// The product with operands staged through registers: a workgroup of 4 waves (2 x 2) takes 32 TM rows x 32 TN columns a tile, K in
// tiles of 128 bytes a row, double-buffered in LDS with a 16-byte row pad.
template <typename T> struct Frag;
template <> struct Frag<bf16_t> {
  __device__ __forceinline__ static void mma(f32x4& acc, const uint4& w, const uint4& x) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
  }
};
template <> struct Frag<float> {
  __device__ __forceinline__ static void mma(f32x4& acc, const uint4& w, const uint4& x) {
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.x), __uint_as_float(x.x), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.y), __uint_as_float(x.y), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.z), __uint_as_float(x.z), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.w), __uint_as_float(x.w), acc, 0, 0, 0);
  }
};

// 16 bytes of a row of K elements from element k on, zeros past its end
template <typename T>
__device__ __forceinline__ uint4 load_k(const T* row, int k, int K) {
  constexpr int E = kE<T>;
  if (k + E <= K) return load16(row + k);
  T x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = k + e < K ? row[k + e] : T(0);
  uint4 v;
  __builtin_memcpy(&v, x, 16);
  return v;
}

template <typename T, bool ENT, int TM, int TN>
__global__ __launch_bounds__(256) void staged_kernel(Args a) {
  constexpr int BM = 32 * TM, BN = 32 * TN, E = kE<T>, kRS = kRowBytes + 16;
  __shared__ __align__(16) unsigned char sw[2][BN * kRS], sx[2][BM * kRS];
  __shared__ int sy[BM];
  __shared__ float sz[BM];
  __shared__ listed list[kSelf];
  __shared__ int red[4];
  __shared__ int64_t best[4];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave & 1, wn = wave >> 1;
  const Plan q = begin<256>(a, BM, list, red, best);
  auto live_row = [&](int i) { return a.self ? (int)list[i] : a.index[i]; };
  const int nk = (a.K + 8 * E - 1) / (8 * E), kc = (tid & 7) * E;
  for (int item = item_of(blockIdx.x, gridDim.x); item < q.mt * q.parts; item += gridDim.x) {
    int mt, part;
    item_at(q, item, mt, part);
    const int m0 = mt * BM, row0 = m0 + wm * 16 * TM;
    const T* xp[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i)
      xp[i] = (const T*)a.h + (int64_t)live_row(min(m0 + (tid >> 3) + 32 * i, q.live - 1)) * a.ldh;
    State st[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) st[i] = State{-INFINITY, 0.f, 0.f};
    __syncthreads();                       // the item before has read its tokens
    if (tid < BM) sy[tid] = m0 + tid < q.live ? column_of(a, live_row(m0 + tid)) : -1;
    const int n_end = min((part + 1) * q.per, a.nt);
    for (int nt = part * q.per; nt < n_end; ++nt) {
      const int n0 = nt * BN;
      const T* wp[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) wp[j] = (const T*)a.w + (int64_t)min(n0 + (tid >> 3) + 32 * j, a.V - 1) * a.ldw;
      uint4 rx[TM], rw[TN];
      auto fetch = [&](int kt) {
        const int k = kt * 8 * E + kc;
#pragma unroll
        for (int j = 0; j < TN; ++j) rw[j] = load_k(wp[j], k, a.K);
#pragma unroll
        for (int i = 0; i < TM; ++i) rx[i] = load_k(xp[i], k, a.K);
      };
      auto stage = [&](int buf) {
        const int off = (tid >> 3) * kRS + (tid & 7) * 16;
#pragma unroll
        for (int j = 0; j < TN; ++j) *reinterpret_cast<uint4*>(&sw[buf][off + 32 * j * kRS]) = rw[j];
#pragma unroll
        for (int i = 0; i < TM; ++i) *reinterpret_cast<uint4*>(&sx[buf][off + 32 * i * kRS]) = rx[i];
      };
      f32x4 acc[TN][TM];
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      fetch(0);
      __syncthreads();                     // the tile before has been read
      stage(0);
      __syncthreads();
      for (int kt = 0; kt < nk; ++kt) {
        const int cur = kt & 1;
        if (kt + 1 < nk) fetch(kt + 1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint4 wf[TN], xf[TM];
          const int kb = ks * 64 + g * 16;
#pragma unroll
          for (int j = 0; j < TN; ++j) wf[j] = *reinterpret_cast<const uint4*>(&sw[cur][(wn * 16 * TN + j * 16 + r) * kRS + kb]);
#pragma unroll
          for (int i = 0; i < TM; ++i) xf[i] = *reinterpret_cast<const uint4*>(&sx[cur][(wm * 16 * TM + i * 16 + r) * kRS + kb]);
#pragma unroll
          for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int i = 0; i < TM; ++i) Frag<T>::mma(acc[j][i], wf[j], xf[i]);
        }
        if (kt + 1 < nk) stage(cur ^ 1);
        __syncthreads();
      }
      take_tile<ENT>(a, acc, st, sy + wm * 16 * TM, sz + wm * 16 * TM, n0 + wn * 16 * TN);
    }
    leave_rows(a, st, row0, q.live, q.parts * 2, part * 2 + wn);
    __syncthreads();
    if (tid < BM) leave_token(a, sy[tid], sz[tid], m0 + tid, (int64_t)part * q.per * BN, (int64_t)n_end * BN);
  }
}

// ---- bf16 with rows of 16-byte pieces, d a multiple of 64 ---------------------------------------------------------------
// LDS byte address of a __shared__ pointer (the M0 operand of global_load_lds)
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// 16 bytes a lane from base + voff into LDS at lds + 16 lane. M0 is an input operand bound to the register itself, so the compiler
// writes it and knows that its value is live across the statement.
__device__ __forceinline__ void dma16(const void* base, uint32_t voff, uint32_t lds) {
  asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "{m0}"(lds) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_vm() {  // s_waitcnt vmcnt(N), other counters untouched
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// Operands through LDS by the DMA path, S stages (S - 1 K tiles on their way while one is multiplied); the fragments of a K tile's
// two halves in two register sets, one read while the other is multiplied. Reads and loads stand between the products: in a burst
// behind the barrier they hold both waves of a SIMD up (5631 rows, 256 x 256 tiles: 506 us in bursts, 478 so). The K tiles of a
// workgroup's column tiles follow each other without a pause: the next column tile's first are on their way while the sums of the
// last take its accumulators. Slot p of LDS row R holds the row's chunk p ^ (R & 7), which makes the fragment reads free of bank
// conflicts.
template <typename T, bool ENT, int TM, int TN, int WGM, int WGN, int S>
__global__ __launch_bounds__(64 * WGM * WGN) void dma_kernel(Args a) {
  constexpr int NW = WGM * WGN, BM = 16 * TM * WGM, BN = 16 * TN * WGN, GX = BM / 8 / NW, GW = BN / 8 / NW;
  static_assert(GX * 8 * NW == BM && GW * 8 * NW == BN, "tile rows must split into 8-row groups per wave");
  // fragments read beside the products of one column tile. fp32 fragments are four products in a chain each, which the compiler
  // has to mix (held apart as bf16's: 329 rows 309 us, 292 free)
  constexpr bool kSpread = sizeof(T) == 2;
  constexpr int FJ = kSpread ? (TM + TN + TN - 1) / TN : TM + TN;
  constexpr int PER = GX + GW, E = kE<T>;
  __shared__ __align__(1024) unsigned char sw[S][BN * kRowBytes], sx[S][BM * kRowBytes];
  __shared__ int sy[BM];
  __shared__ float sz[BM];
  __shared__ listed list[kSelf];
  __shared__ int red[NW];
  __shared__ int64_t best[NW];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WGM, wn = wave / WGM;
  const Plan q = begin<64 * NW>(a, BM, list, red, best);
  auto live_row = [&](int i) { return a.self ? (int)list[i] : a.index[i]; };
  const int nk = a.K / (8 * E);
  const int fw = (wn * 16 * TN + r) * kRowBytes, fx = (wm * 16 * TM + r) * kRowBytes;
  const int c0 = (g ^ (r & 7)) << 4, c1 = ((4 + g) ^ (r & 7)) << 4;
  // the f-th fragment of a K tile's half
  auto read = [&](uint4 (&wf)[TN], uint4 (&xf)[TM], int f, int st, int c) {
    if (f < TM)
      xf[f < TM ? f : 0] = *reinterpret_cast<const uint4*>(&sx[st][fx + f * 16 * kRowBytes + c]);
    else
      wf[f < TM ? 0 : f - TM] = *reinterpret_cast<const uint4*>(&sw[st][fw + (f - TM) * 16 * kRowBytes + c]);
  };
  f32x4 acc[TN][TM];
  for (int item = item_of(blockIdx.x, gridDim.x); item < q.mt * q.parts; item += gridDim.x) {
    int mt, part;
    item_at(q, item, mt, part);
    const int m0 = mt * BM, row0 = m0 + wm * 16 * TM;
    const int n_first = part * q.per, n_end = min(n_first + q.per, a.nt);
    // load group u of this wave: rows 8 G .. 8 G + 7, G = NW u + wave; lane -> row 8 G + lane / 8, slot lane % 8
    uint32_t xo[GX], wo[GW];
#pragma unroll
    for (int u = 0; u < GX; ++u) {
      const int R = 8 * (NW * u + wave) + (lane >> 3);
      xo[u] = ((uint32_t)live_row(min(m0 + R, q.live - 1)) * (uint32_t)a.ldh + (uint32_t)(((lane & 7) ^ (R & 7)) * E)) * (uint32_t)sizeof(T);
    }
    int next_n = n_first, next_k = 0;      // what is loaded next
    const char* wbase = nullptr;
    auto columns = [&]() {                 // the offsets of column tile next_n
      const int n0 = next_n * BN;
      wbase = (const char*)a.w + (int64_t)n0 * a.ldw * (int)sizeof(T);
#pragma unroll
      for (int u = 0; u < GW; ++u) {
        const int R = 8 * (NW * u + wave) + (lane >> 3);
        wo[u] = ((uint32_t)min(R, a.V - 1 - n0) * (uint32_t)a.ldw + (uint32_t)(((lane & 7) ^ (R & 7)) * E)) * (uint32_t)sizeof(T);
      }
    };
    auto load_one = [&](int u, int st) {   // the u-th of a K tile's PER loads
      const int kb = next_k * kRowBytes;
      if (u < GW)
        dma16(wbase + kb, wo[u < GW ? u : 0], lds_addr(&sw[st][(NW * u + wave) * 1024]));
      else
        dma16((const char*)a.h + kb, xo[u < GW ? 0 : u - GW], lds_addr(&sx[st][(NW * (u - GW) + wave) * 1024]));
    };
    auto advance = [&] {
      if (++next_k == nk) {                // (behind the last tile its own again: read by nobody)
        next_k = 0;
        next_n = min(next_n + 1, n_end - 1);
        columns();
      }
    };
    auto issue = [&](int st) {
#pragma unroll
      for (int u = 0; u < PER; ++u) load_one(u, st);
      advance();
    };
    State sums[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) sums[i] = State{-INFINITY, 0.f, 0.f};
    columns();
    __syncthreads();                       // the item before has been read
    if (tid < BM) sy[tid] = m0 + tid < q.live ? column_of(a, live_row(m0 + tid)) : -1;
#pragma unroll
    for (int u = 0; u < S - 1; ++u) issue(u);
    wait_vm<(S - 2) * PER>();              // loads return in their order
    __syncthreads();
    issue(S - 1);
    uint4 aw[TN], ax[TM], bw[TN], bx[TM];
#pragma unroll
    for (int f = 0; f < TM + TN; ++f) read(aw, ax, f, 0, c0);
    int st = 0;
    for (int nt = n_first; nt < n_end; ++nt) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int kt = 0; kt < nk; ++kt) {
        // step 0's products, with the reads of step 1's fragments between them
#pragma unroll
        for (int j = 0; j < TN; ++j) {
#pragma unroll
          for (int f = j * FJ; f < (j + 1) * FJ && f < TM + TN; ++f) read(bw, bx, f, st, c1);
#pragma unroll
          for (int i = 0; i < TM; ++i) Frag<T>::mma(acc[j][i], aw[j], ax[i]);
          if (kSpread) __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        wait_vm<(S - 2) * PER>();          // the next K tile is there (nothing else was stored or loaded since)
        __syncthreads();                   // for everyone, and this one has been read
        const int nst = st + 1 == S ? 0 : st + 1;
        // step 1's products, with the reads of the next K tile's step 0 and the loads into this one's place between them
#pragma unroll
        for (int j = 0; j < TN; ++j) {
#pragma unroll
          for (int f = j * FJ; f < (j + 1) * FJ && f < TM + TN; ++f) read(aw, ax, f, nst, c0);
#pragma unroll
          for (int u = j * PER / TN; u < (j + 1) * PER / TN; ++u) load_one(u, st);
#pragma unroll
          for (int i = 0; i < TM; ++i) Frag<T>::mma(acc[j][i], bw[j], bx[i]);
          if (kSpread) __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        advance();
        st = nst;
      }
      take_tile<ENT>(a, acc, sums, sy + wm * 16 * TM, sz + wm * 16 * TM, nt * BN + wn * 16 * TN);
    }
    leave_rows(a, sums, row0, q.live, q.parts * WGN, part * WGN + wn);
    __syncthreads();
    if (tid < BM) leave_token(a, sy[tid], sz[tid], m0 + tid, (int64_t)n_first * BN, (int64_t)n_end * BN);
    wait_vm<0>();                          // also the loads that nobody reads
  }
}

// ---- few rows -----------------------------------------------------------------------------------------------------------
// The weight's bytes are what counts: every wave streams column tiles of 16 weight rows by DMA through a ring of its own of kRing K
// tiles (whole 128-byte lines, kRing - 1 of them on their way; no barrier) against all rows, which lie in LDS: K tiles of 128 bytes a
// row, chunk p of row R at p ^ (R & 7), as those of the ring. Rows of 16-byte pieces, d a multiple of 128 bytes.
constexpr int kFewWaves = 8, kFewGroups = 256, kFewLds = 64 * 1024, kRing = 5;

template <typename T, bool ENT, int TM>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(Args a) {
  constexpr int BM = 16 * TM, E = kE<T>, kTile = 16 * kRowBytes;
  extern __shared__ __align__(1024) unsigned char lds[];
  __shared__ int sy[BM];
  __shared__ float sz[BM];
  __shared__ State red[kFewWaves][BM];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), id = blockIdx.x * kFewWaves + wave;
  const int nk = a.K / (8 * E);            // K tiles
  const int tiles = (a.V + 15) / 16, waves = gridDim.x * kFewWaves, per = (tiles + waves - 1) / waves;
  const int first = min(id * per, tiles), end = min(first + per, tiles), total = (end - first) * nk;
  unsigned char *ring = lds + wave * kRing * kTile, *sx = lds + kFewWaves * kRing * kTile;
  const uint32_t slot = (uint32_t)(((lane & 7) ^ (lane >> 3)) * 16);           // (8 rows a load: their chunks' places)
  for (int c = wave; c < nk * 2 * TM; c += kFewWaves) {        // the rows: first, as loads return in their order
    const int kt = c / (2 * TM), R = 8 * (c - kt * 2 * TM) + (lane >> 3);
    const uint32_t at = (uint32_t)min(R, a.rows - 1) * (uint32_t)a.ldh * (uint32_t)sizeof(T) + slot;
    dma16((const char*)a.h + kt * kRowBytes, at, lds_addr(sx) + (uint32_t)(c * 1024));
  }
  int tile = first, kt = 0;                // what is loaded next
  uint32_t wo[2];
  const char* wbase = nullptr;
  auto columns = [&] {
    wbase = (const char*)a.w + (int64_t)tile * 16 * a.ldw * (int)sizeof(T);
#pragma unroll
    for (int u = 0; u < 2; ++u)
      wo[u] = (uint32_t)min(8 * u + (lane >> 3), a.V - 1 - tile * 16) * (uint32_t)a.ldw * (uint32_t)sizeof(T) + slot;
  };
  auto issue = [&](int place) {
#pragma unroll
    for (int u = 0; u < 2; ++u) dma16(wbase + kt * kRowBytes, wo[u], lds_addr(ring + place * kTile + u * 1024));
    if (++kt == nk) {
      kt = 0;
      tile = min(tile + 1, tiles - 1);
      columns();
    }
  };
  if (total) {                             // uniform
    columns();
    for (int u = 0; u < min(kRing, total); ++u) issue(u);
  }
  State sums[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) sums[i] = State{-INFINITY, 0.f, 0.f};
  f32x4 acc[1][TM];
  if (total >= kRing)
    wait_vm<2 * kRing>();
  else
    wait_vm<0>();
  __builtin_amdgcn_sched_barrier(0);
  if (tid < BM) sy[tid] = tid < a.rows ? column_of(a, tid) : -1;
  __syncthreads();
  int t = 0, place = 0;
  for (int at = first; at < end; ++at) {
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[0][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < nk; ++k, ++t) {
      if (t + kRing <= total)
        wait_vm<2 * (kRing - 1)>();        // the oldest of kRing tiles
      else
        wait_vm<0>();
      __builtin_amdgcn_sched_barrier(0);
      uint4 w[2], x[2][TM];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = ((4 * h + g) ^ (r & 7)) << 4;
        w[h] = *reinterpret_cast<const uint4*>(ring + place * kTile + r * kRowBytes + c);
#pragma unroll
        for (int i = 0; i < TM; ++i) x[h][i] = *reinterpret_cast<const uint4*>(sx + (k * BM + 16 * i + r) * kRowBytes + c);
      }
      __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));   // s_waitcnt lgkmcnt(0): the tile has been read
      __builtin_amdgcn_sched_barrier(0);
      if (t + kRing < total) issue(place);
      place = place + 1 == kRing ? 0 : place + 1;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < TM; ++i) Frag<T>::mma(acc[0][i], w[h], x[h][i]);
    }
    take_tile<ENT>(a, acc, sums, sy, sz, at * 16);
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    State v = sums[i];
#pragma unroll
    for (int o = 16; o <= 32; o <<= 1) v = join(v, State{__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.t, o)}, a.c);
    if (lane < 16) red[wave][16 * i + r] = v;
  }
  __syncthreads();
  if (tid >= BM || tid >= a.rows) return;
  State v = red[0][tid];
#pragma unroll
  for (int u = 1; u < kFewWaves; ++u) v = join(v, red[u][tid], a.c);
  a.part[(int64_t)tid * gridDim.x + blockIdx.x] = v;
  const int64_t lo = (int64_t)blockIdx.x * kFewWaves * per * 16;
  leave_token(a, sy[tid], sz[tid], tid, lo, lo + (int64_t)kFewWaves * per * 16);
}

// ---- sizes ------------------------------------------------------------------------------------------------------------
// A form of the product. kind 0: staged through registers, 1: by DMA, 2: few rows. groups: workgroups; slots: a part's slots
struct Form {
  int kind, bm, bn, groups, slots, id;
};
// The forms of the DMA kernel, and what a tile of each takes at K = 1024, microseconds on a full card: the form whose rounds of tiles
// take least, of all rows (how many count is known on the device only). us of a call without entropies, weights that no cache holds (three
// in turn, a graph), V 50257, d 1024. bf16 by rows, 256 x 256 / 128 x 256 / 64 x 256 / 64 x 64: 64 41 / 33 / 31 / 32; 128 39 / 32 / 36 / 44;
// 256 41 / 42 / 56 / 63; 512 64 / 68 / 84 / 100; 640 86 / 69 / 103 / 127; 1024 112 / 107 / 145 / 178; 4096 329 / 349 / 517 / 658; 5300
// 426 / 449 / 673 / 850. (A few large tiles leave most of the card idle: 2000 rows of V 1000 are 32 of 256 x 256.) fp32 is bound by its
// products whatever the tile, and 32 x 128 tiles have the fewest empty rows: 200, 329, 501, 4096 rows 200, 289, 413, 3055. (Chosen on an
// earlier version, whose rows were sorted out by a launch of 5 us: 205, 292, 413, 3090; 64 x 64 236, 321, 412, 3055; 128 x 128 255, 372,
// 491, 2995.)
struct Timed {
  Form form;
  float us;
};
constexpr Timed kBf16[] = {{{1, 256, 256, 256, 2, 0}, 25.f}, {{1, 128, 256, 256, 2, 1}, 13.6f}, {{1, 64, 256, 256, 2, 2}, 8.7f},
                           {{1, 64, 64, 512, 2, 3}, 5.9f}};
constexpr Form kFp32 = {1, 32, 128, 512, 2, 0};
// Staged through registers, the same rule. V 50257, d 1001, us by rows, 64 x 64 / 128 x 128 tiles: bf16 1 39 / 42; 64 50 / 51; 128 75 /
// 51; 512 187 / 142; 4096 1164 / 775; fp32 64 100 / 156; 128 183 / 157; 1024 1073 / 1011. V 5000, d 777: bf16 512 29 / 31; fp32 512 79 / 123.
constexpr Timed kStagedBf16[] = {{{0, 64, 64, 1024, 2, 0}, 22.f}, {{0, 128, 128, 512, 2, 1}, 26.f}};
constexpr Timed kStagedFp32[] = {{{0, 64, 64, 1024, 2, 0}, 82.f}, {{0, 128, 128, 512, 2, 1}, 140.f}};

template <int N>
Form least(const Timed (&forms)[N], int64_t rows, int V) {
  int best = 0;
  double us = 1e30;
  for (int i = 0; i < N; ++i) {
    const Form& f = forms[i].form;
    const int64_t tiles = ((rows + f.bm - 1) / f.bm) * ((V + f.bn - 1) / f.bn);
    const double takes = (double)((tiles + f.groups - 1) / f.groups) * forms[i].us;
    if (takes < us) {
      us = takes;
      best = i;
    }
  }
  return forms[best].form;
}
// up to 32 rows (as many as LDS holds beside the rings) the form for few: 16 rows 23 us, the 64 x 256 tiles 31; fp32 51 us, its tiles 54
Form form_of(int dtype, int64_t rows, int d, int V, bool fast) {
  if (!fast) return dtype == DH_F32 ? least(kStagedFp32, rows, V) : least(kStagedBf16, rows, V);
  if (rows <= 32 && (rows <= 16 ? 16 : 32) * (int64_t)d * (dtype == DH_BF16 ? 2 : 4) <= kFewLds)
    return Form{2, 0, 0, kFewGroups, 1, 0};
  return dtype == DH_F32 ? kFp32 : least(kBf16, rows, V);
}
struct Layout {
  int64_t index, part, zy, bytes;
};
Layout layout_of(const Form& t, int64_t rows) {
  Layout l;
  if (t.kind == 2) {
    l.index = 0;
    l.part = 0;
    l.zy = rows * t.groups * (int64_t)sizeof(State);
    l.bytes = l.zy + rows * 4;
    return l;
  }
  // a row tile has at most max(1, 2 groups / row tiles) parts
  const int64_t mt = (rows + t.bm - 1) / t.bm, padded = mt * t.bm;
  const int64_t slots = (padded > 2 * (int64_t)t.groups * t.bm ? padded : 2 * (int64_t)t.groups * t.bm) * t.slots;
  l.index = 256;
  l.part = l.index + (rows * 4 + 255) / 256 * 256;
  l.zy = l.part + slots * (int64_t)sizeof(State);
  l.bytes = l.zy + rows * 4;
  return l;
}

template <typename T, bool ENT, int TM>
int run_few(Args& a, int groups, hipStream_t s, const char* who) {
  const size_t lds = (size_t)16 * TM * a.K * sizeof(T) + kFewWaves * kRing * 16 * kRowBytes;
  // (the same on every call, so that no host thread lowers it before another's launch)
  if (hipFuncSetAttribute((const void*)few_kernel<T, ENT, TM>, hipFuncAttributeMaxDynamicSharedMemorySize,
                          kFewLds + kFewWaves * kRing * 16 * kRowBytes) != hipSuccess)
    return dh_fail(DH_ERR_LAUNCH_FAILED, "%s: %d bytes of LDS", who, kFewLds);
  few_kernel<T, ENT, TM><<<dim3((unsigned)groups), dim3(64 * kFewWaves), lds, s>>>(a);
  return dh_check_launch(who);
}

template <typename T, bool ENT>
int run(Args& a, const Form& t, char* ws, const Layout& l, hipStream_t s, const char* who) {
  a.part = (State*)(ws + l.part);
  a.zy = (float*)(ws + l.zy);
  if (t.kind == 2) {
    // as few workgroups as have every wave take the same number of column tiles
    const int tiles = (a.V + 15) / 16, per = (tiles + t.groups * kFewWaves - 1) / (t.groups * kFewWaves);
    const int groups = (tiles + per * kFewWaves - 1) / (per * kFewWaves);
    const int st = a.rows <= 16 ? run_few<T, ENT, 1>(a, groups, s, who) : run_few<T, ENT, 2>(a, groups, s, who);
    if (st) return st;
    join_kernel<ENT><<<dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s>>>(a, 0, groups);
    return dh_check_launch(who);
  }
  a.nt = (a.V + t.bn - 1) / t.bn;
  a.plan = (Plan*)ws;
  a.index = (int*)(ws + l.index);
  a.self = a.rows <= kSelf;
  if (!a.self) {
    const int chunk = chunk_of(a.rows);
    compact_kernel<<<dim3((unsigned)((a.rows + chunk - 1) / chunk)), dim3(kCT), 0, s>>>(a, t.bm, t.groups, chunk);
    if (int st = dh_check_launch(who)) return st;
  }
  const dim3 grid((unsigned)t.groups);
  if (t.kind == 1) {
    if (sizeof(T) == 4) {
      dma_kernel<float, ENT, 1, 4, 2, 2, 3><<<grid, dim3(256), 0, s>>>(a);
    } else {
      switch (t.id) {
        case 0: dma_kernel<bf16_t, ENT, 4, 8, 4, 2, 2><<<grid, dim3(512), 0, s>>>(a); break;
        case 1: dma_kernel<bf16_t, ENT, 2, 8, 4, 2, 3><<<grid, dim3(512), 0, s>>>(a); break;
        case 2: dma_kernel<bf16_t, ENT, 1, 8, 4, 2, 3><<<grid, dim3(512), 0, s>>>(a); break;
        default: dma_kernel<bf16_t, ENT, 2, 2, 2, 2, 4><<<grid, dim3(256), 0, s>>>(a); break;
      }
    }
  } else if (t.id == 0) {
    staged_kernel<T, ENT, 2, 2><<<grid, dim3(256), 0, s>>>(a);
  } else {
    staged_kernel<T, ENT, 4, 4><<<grid, dim3(256), 0, s>>>(a);
  }
  if (int st = dh_check_launch(who)) return st;
  join_kernel<ENT><<<dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s>>>(a, t.slots, 0);
  return dh_check_launch(who);
}

}  // namespace

extern "C" int64_t dh_head_logprob_workspace_bytes(int dtype, int64_t rows, int V) {
  if ((dtype != DH_F32 && dtype != DH_BF16) || rows < 0 || rows >= (1 << 22) || V < 1 || V > (1 << 24)) return -1;
  // (whatever form d and the operands' alignment allow)
  int64_t most = layout_of(form_of(dtype, rows, 0, V, false), rows).bytes;
  for (int d : {0, 1 << 20}) {
    const int64_t bytes = layout_of(form_of(dtype, rows, d, V, true), rows).bytes;
    if (bytes > most) most = bytes;
  }
  return most;
}

extern "C" int dh_head_logprob(int dtype, const void* hidden, int64_t hidden_stride, int64_t rows, int d, const void* weight,
                               int64_t weight_stride, int V, const void* tokens, int token_bits, int64_t ignore_index,
                               double temperature, int round_logits, float* logprob, float* entropy, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  const char* who = "dh_head_logprob";
  DH_REQUIRE(dtype == DH_F32 || dtype == DH_BF16, DH_ERR_UNSUPPORTED_DTYPE, "%s: dtype %d", who, dtype);
  DH_REQUIRE(token_bits == 32 || token_bits == 64, DH_ERR_UNSUPPORTED_DTYPE, "%s: tokens of %d bits", who, token_bits);
  DH_REQUIRE(rows >= 0 && rows < (1 << 22) && d >= 1 && d <= (1 << 20) && V >= 1 && V <= (1 << 24), DH_ERR_UNSUPPORTED_SHAPE,
             "%s: %lld rows, d=%d V=%d", who, (long long)rows, d, V);
  DH_REQUIRE(temperature >= 0x1p-126 && temperature <= 0x1p126, DH_ERR_INVALID_ARG, "%s: temperature %g", who, temperature);
  const int size = dtype == DH_BF16 ? 2 : 4;
  DH_REQUIRE(rows == 0 || (hidden && weight && tokens && logprob), DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE(hidden_stride >= 0 && weight_stride >= 0, DH_ERR_INVALID_ARG, "%s: strides %lld, %lld", who, (long long)hidden_stride,
             (long long)weight_stride);
  DH_REQUIRE((uintptr_t)hidden % size == 0 && (uintptr_t)weight % size == 0 && (uintptr_t)tokens % (token_bits / 8) == 0 &&
                 (uintptr_t)logprob % 4 == 0 && (uintptr_t)entropy % 4 == 0,
             DH_ERR_INVALID_ARG, "%s: operands not aligned to their elements", who);
  if (rows == 0) return 0;
  const int64_t need = dh_head_logprob_workspace_bytes(dtype, rows, V);
  DH_REQUIRE(workspace_bytes >= need && workspace && (uintptr_t)workspace % 16 == 0, DH_ERR_INVALID_ARG,
             "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes, (long long)need);
  // (offsets of a lane in 32 bits)
  const int e = 16 / size;
  const bool fast = d % (8 * e) == 0 && hidden_stride % e == 0 && weight_stride % e == 0 && (uintptr_t)hidden % 16 == 0 &&
                    (uintptr_t)weight % 16 == 0 && (rows - 1) * hidden_stride + d < (int64_t)1 << 30 && weight_stride < (1 << 21);
  const Form t = form_of(dtype, rows, d, V, fast);
  const Layout l = layout_of(t, rows);
  Args a{};
  a.h = hidden;
  a.ldh = hidden_stride;
  a.w = weight;
  a.ldw = weight_stride;
  a.rows = (int)rows;
  a.V = V;
  a.K = d;
  a.tokens = tokens;
  a.wide = token_bits == 64;
  a.ignore = ignore_index;
  a.round = round_logits && dtype == DH_BF16;
  a.c = (float)(kLog2e / temperature);
  a.inv_tau = 1.0 / temperature;
  a.lp = logprob;
  a.ent = entropy;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  if (dtype == DH_BF16) return entropy ? run<bf16_t, true>(a, t, ws, l, s, who) : run<bf16_t, false>(a, t, ws, l, s, who);
  return entropy ? run<float, true>(a, t, ws, l, s, who) : run<float, false>(a, t, ws, l, s, who);
}
