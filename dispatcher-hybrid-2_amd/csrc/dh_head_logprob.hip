// Log-probabilities of given tokens from the last hidden states and the vocabulary head's weight, without the logits in memory,
// for gfx950 (inference). For a row h (d wide), the weight W (V, d), a temperature tau and the row's token y:
//   z_v = h . W_v (fp32 sums; round_logits: rounded to the operands' type),  p = softmax(z / tau)
//   lp = log p_y,  H = - sum_v p_v log p_v
// A row whose token is ignore_index is not computed: lp = H = 0.
//
// The product's tiles stay in the accumulators. A lane of a tile holds some columns of its rows and keeps, over all the tiles that
// its workgroup takes of a row, the running maximum m of z and the sums of e = exp((z - m) / tau) and of e times its exponent;
// lanes are joined when the workgroup ends with the row, workgroups by a last launch. A token's own logit is written by the lane
// that meets it. So a row leaves a few numbers for each workgroup instead of V logits.
//
// Launches: the rows that count, in their order, and how the tiles are dealt out (compact_kernel; their number is known on the
// device only); the product; the join. Up to 64 rows: the product (few_kernel, the weight's bytes bound it) and the join.

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
  const Plan* plan;
  const int* index;                        // the live rows; null: all
  State* part;                             // [compact row][slots]
  float* zy;                               // [compact row]
  float *lp, *ent;
};

__device__ __forceinline__ int row_at(const Args& a, int i) { return a.index ? a.index[i] : i; }

// ---- the rows that count ----------------------------------------------------------------------------------------------
constexpr int kCT = 1024, kChunk = 4 * kCT;                    // threads, rows a workgroup

// A workgroup counts the live rows before its own (all of them read by every one: 8 MB a million rows, beside a product of 70 ms)
// and places those of its chunk. The last one deals out the tiles: the number of parts whose longest workgroup is shortest.
__global__ __launch_bounds__(kCT) void compact_kernel(Args a, int bm, int groups, int* index, Plan* plan) {
  __shared__ int red[kCT / 64], base, total;
  __shared__ int64_t best[kCT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lo = blockIdx.x * kChunk, hi = min(lo + kChunk, a.rows);
  auto live = [&](int r) { return whole(a.tokens, a.wide, r) != a.ignore; };
  int before = 0;
  for (int r = tid; r < lo; r += kCT) before += live(r);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
  if (lane == 0) red[wave] = before;
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    for (int w = 0; w < kCT / 64; ++w) n += red[w];
    base = n;
  }
  __syncthreads();
  int at = base;
  for (int r0 = lo; r0 < hi; r0 += kCT) {  // uniform
    const int r = r0 + tid;
    const bool in = r < hi, on = in && live(r);
    const uint64_t mask = __builtin_amdgcn_ballot_w64(on);
    __syncthreads();
    if (lane == 0) red[wave] = __popcll(mask);
    __syncthreads();
    int place = at + __popcll(mask & ((1ull << lane) - 1)), all = 0;
    for (int w = 0; w < kCT / 64; ++w) {
      if (w < wave) place += red[w];
      all += red[w];
    }
    if (on) index[place] = r;
    if (in && !on) {
      a.lp[r] = 0.f;
      if (a.ent) a.ent[r] = 0.f;
    }
    at += all;
  }
  if ((int)blockIdx.x != (int)gridDim.x - 1) return;
  if (tid == 0) total = at;
  __syncthreads();
  const int n = total, mt = (n + bm - 1) / bm;
  if (mt == 0) {
    if (tid == 0) *plan = Plan{0, 0, 1, a.nt};
    return;
  }
  // rounds of the workgroups times the tiles of a part (and half a tile that beginning and ending one takes)
  int64_t mine = INT64_MAX;
  const int most = max(1, min(a.nt, 2 * groups / mt));
  for (int p = tid + 1; p <= most; p += kCT) {
    const int64_t per = (a.nt + p - 1) / p, rounds = ((int64_t)mt * p + groups - 1) / groups;
    const int64_t cost = rounds * (2 * per + 1);
    mine = min(mine, cost << 20 | p);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int64_t other = __shfl_xor(mine, o);
    mine = min(mine, other);
  }
  if (lane == 0) best[wave] = mine;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kCT / 64; ++w) mine = min(mine, best[w]);
    const int p = (int)(mine & 0xfffff), per = (a.nt + p - 1) / p;
    *plan = Plan{n, mt, (a.nt + per - 1) / per, per};
  }
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

// ---- the rows' results ------------------------------------------------------------------------------------------------
template <bool ENT>
__device__ __forceinline__ void finish(const Args& a, int r, const State& v, float zy, bool bad) {
  const double nan = __builtin_nan("");
  const double ls = log((double)v.s);
  a.lp[r] = (float)(bad ? nan : ((double)zy - (double)v.m) * a.inv_tau - ls);
  if (ENT) a.ent[r] = (float)(bad ? nan : ls - (double)v.t * kLn2 / (double)v.s);
}

// a wave a live row: its slots joined in their order
template <bool ENT>
__global__ __launch_bounds__(256) void join_kernel(Args a, int slots_a_part, int slots_if_all) {
  const int lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int live = a.plan ? a.plan->live : a.rows;
  if (i >= live) return;
  const int slots = a.plan ? a.plan->parts * slots_a_part : slots_if_all;
  const int r = row_at(a, i);
  const int64_t y = whole(a.tokens, a.wide, r);
  State v{-INFINITY, 0.f, 0.f};
  for (int k = lane; k < slots; k += 64) v = join(v, a.part[(int64_t)i * slots + k], a.c);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    v = join(v, State{__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.t, o)}, a.c);
  if (lane) return;
  if (y == a.ignore) {                     // (rows that were not sorted out)
    a.lp[r] = 0.f;
    if (ENT) a.ent[r] = 0.f;
    return;
  }
  const bool bad = y < 0 || y >= a.V;
  finish<ENT>(a, r, v, bad ? 0.f : a.zy[i], bad);
}

// ---- a workgroup's tiles ------------------------------------------------------------------------------------------------
// acc[j][i] of lane (r, g): columns n + 16 j + 4 g .. + 3 of row 16 i + r, n the wave's first column
template <bool ENT, int TM, int TN>
__device__ __forceinline__ void take_tile(const Args& a, f32x4 (&acc)[TN][TM], State (&st)[TM], const int (&y)[TM], int n, int row0,
                                          int live) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
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
        const int k = y[i] - (n + 16 * j + 4 * g), row = row0 + 16 * i + r;
        if (k >= 0 && k < 4 && row < live) {
          float z = acc[j][i][0];
#pragma unroll
          for (int e = 1; e < 4; ++e) z = k == e ? acc[j][i][e] : z;
          a.zy[row] = z;
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
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave & 1, wn = wave >> 1;
  const Plan q = *a.plan;
  const int nk = (a.K + 8 * E - 1) / (8 * E), kc = (tid & 7) * E;
  for (int item = item_of(blockIdx.x, gridDim.x); item < q.mt * q.parts; item += gridDim.x) {
    int mt, part;
    item_at(q, item, mt, part);
    const int m0 = mt * BM, row0 = m0 + wm * 16 * TM;
    const T* xp[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i)
      xp[i] = (const T*)a.h + (int64_t)row_at(a, min(m0 + (tid >> 3) + 32 * i, q.live - 1)) * a.ldh;
    int y[TM];
    State st[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = row0 + 16 * i + r;
      const int64_t k = row < q.live ? whole(a.tokens, a.wide, row_at(a, row)) : -1;
      y[i] = k >= 0 && k < a.V ? (int)k : -1;
      st[i] = State{-INFINITY, 0.f, 0.f};
    }
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
      take_tile<ENT>(a, acc, st, y, n0 + wn * 16 * TN, row0, q.live);
    }
    leave_rows(a, st, row0, q.live, q.parts * 2, part * 2 + wn);
  }
}

// ---- sizes ------------------------------------------------------------------------------------------------------------
struct Tile {
  int bm, bn, groups, slots;
};
Tile tile_of(int dtype, int64_t rows) {
  if (dtype == DH_F32 && rows <= 512) return Tile{64, 64, 1024, 2};
  return Tile{128, 128, 512, 2};
}
struct Layout {
  int64_t index, part, zy, bytes;
};
Layout layout_of(int dtype, int64_t rows) {
  const Tile t = tile_of(dtype, rows);
  // a row tile has at most max(1, 2 groups / row tiles) parts
  const int64_t mt = (rows + t.bm - 1) / t.bm, padded = mt * t.bm;
  const int64_t slots = (padded > 2 * (int64_t)t.groups * t.bm ? padded : 2 * (int64_t)t.groups * t.bm) * t.slots;
  Layout l;
  l.index = 256;
  l.part = l.index + (rows * 4 + 255) / 256 * 256;
  l.zy = l.part + slots * (int64_t)sizeof(State);
  l.bytes = l.zy + rows * 4;
  return l;
}

template <typename T, bool ENT>
int run(Args& a, int dtype, char* ws, const Layout& l, hipStream_t s, const char* who) {
  const Tile t = tile_of(dtype, a.rows);
  a.nt = (a.V + t.bn - 1) / t.bn;
  a.plan = (Plan*)ws;
  a.index = (int*)(ws + l.index);
  a.part = (State*)(ws + l.part);
  a.zy = (float*)(ws + l.zy);
  compact_kernel<<<dim3((unsigned)((a.rows + kChunk - 1) / kChunk)), dim3(kCT), 0, s>>>(a, t.bm, t.groups, (int*)(ws + l.index),
                                                                                       (Plan*)ws);
  if (int st = dh_check_launch(who)) return st;
  if (t.bm == 64)
    staged_kernel<T, ENT, 2, 2><<<dim3((unsigned)t.groups), dim3(256), 0, s>>>(a);
  else
    staged_kernel<T, ENT, 4, 4><<<dim3((unsigned)t.groups), dim3(256), 0, s>>>(a);
  if (int st = dh_check_launch(who)) return st;
  join_kernel<ENT><<<dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s>>>(a, t.slots, 0);
  return dh_check_launch(who);
}

}  // namespace

extern "C" int64_t dh_head_logprob_workspace_bytes(int dtype, int64_t rows, int V) {
  if ((dtype != DH_F32 && dtype != DH_BF16) || rows < 0 || rows >= (1 << 22) || V < 1 || V > (1 << 24)) return -1;
  return layout_of(dtype, rows).bytes;
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
  const Layout l = layout_of(dtype, rows);
  DH_REQUIRE(workspace_bytes >= l.bytes && workspace && (uintptr_t)workspace % 16 == 0, DH_ERR_INVALID_ARG,
             "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes, (long long)l.bytes);
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
  if (dtype == DH_BF16) return entropy ? run<bf16_t, true>(a, dtype, ws, l, s, who) : run<bf16_t, false>(a, dtype, ws, l, s, who);
  return entropy ? run<float, true>(a, dtype, ws, l, s, who) : run<float, false>(a, dtype, ws, l, s, who);
}
