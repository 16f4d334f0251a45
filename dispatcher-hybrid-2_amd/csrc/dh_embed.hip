// Embedding rows and their gradient, for gfx950:
//   out[n] = rnd(scale W[id_n])                       (dh_embed_fwd)
//   dW[v]  = rnd(scale sum_{n: id_n = v} dy[n])       (dh_embed_bwd; every row of dW is written)
// The parallel forward's embedding (reference dispatcher_hybrid/modeling_dispatcher.py:340) and its autograd gradient.
//
// The gradient groups the positions by token: sums in fp32 over stretches of a token's positions in ascending order, split and
// joined as the ids and the sizes say (chunks, eighths of a token's chunks, sixteenths in the one launch), so the same call gives
// the same bits whatever the launch order. Three launches:
//   place  every workgroup owns every 256th token id and reads ALL ids itself (8 n bytes from L2, cheaper than the launches
//          of a sort that shares work between workgroups): it counts the ids of the owners before it (its offset in the
//          grouped order) and its own per (wave, token), scans, and writes its (token, position) pairs, positions
//          ascending.
//   sum    the grouped list in equal chunks, whatever the distribution of the tokens: a wave adds the dy rows of a chunk and
//          writes a token's row when the token's positions all lie in the chunk; the sums of a first or last token that
//          reaches into the neighbouring chunks go to the workspace. Beside it, the rows of tokens without a position are
//          filled with zeros.
//   join   adds the chunk sums of every token that lies in more than one chunk, as `sum` noted them.
// Bytes: n d read, V d written (and the ids): 32768 x 1024 bf16, V 50257: place 13, sum 29 (5.9 TB/s), join 5 us. Ids outside
// [0, V) hold no gradient (their rows of `out` are NaN).

#include <type_traits>

#include "dh_common.h"

namespace {

// ---- elements in registers: N values of a 16-byte piece (any d otherwise: one) --------------------------------------
template <typename T, int N> struct Piece;
template <> struct Piece<bf16_t, 8> {
  typedef uint4 raw;
  __device__ __forceinline__ static void unpack(const uint4& v, float (&o)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[2 * j] = __uint_as_float(w[j] << 16);
      o[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ static uint4 pack(const float (&o)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (uint32_t)f32_to_bf16(o[2 * j]) | ((uint32_t)f32_to_bf16(o[2 * j + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Piece<float, 4> {
  typedef uint4 raw;
  __device__ __forceinline__ static void unpack(const uint4& v, float (&o)[4]) {
    o[0] = __uint_as_float(v.x);
    o[1] = __uint_as_float(v.y);
    o[2] = __uint_as_float(v.z);
    o[3] = __uint_as_float(v.w);
  }
  __device__ __forceinline__ static uint4 pack(const float (&o)[4]) {
    return make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
  }
};
template <typename T> struct Piece<T, 1> {
  typedef T raw;
  __device__ __forceinline__ static void unpack(const T& v, float (&o)[1]) { o[0] = Elem<T>::load(&v); }
  __device__ __forceinline__ static T pack(const float (&o)[1]) {
    T v;
    Elem<T>::store(&v, o[0]);
    return v;
  }
};

__device__ __forceinline__ int64_t load_id(const void* ids, int wide, int64_t i) {
  return wide ? reinterpret_cast<const int64_t*>(ids)[i] : (int64_t) reinterpret_cast<const int32_t*>(ids)[i];
}

// ---- lookup ---------------------------------------------------------------------------------------------------------
constexpr int kLT = 256;                   // threads

// 2^lg lanes hold R rows of `pieces` pieces; R 2^(8 - lg) rows a workgroup
template <typename T, int N, int R>
__global__ __launch_bounds__(kLT) void lookup_kernel(const T* W, int64_t ldw, int64_t V, const void* ids, int wide, int64_t n,
                                                     float scale, int64_t zero_token, T* out, int64_t ldo, int pieces,
                                                     int lg) {
  typedef Piece<T, N> P;
  const int64_t row = (((int64_t)blockIdx.x << (8 - lg)) + (threadIdx.x >> lg)) * R;
  if (row >= n) return;
  const float stray = zero_token < 0 ? __builtin_nanf("") : 0.f;
  int64_t id[R];
#pragma unroll
  for (int r = 0; r < R; ++r) id[r] = load_id(ids, wide, min(row + r, n - 1));
  for (int c = threadIdx.x & ((1 << lg) - 1); c < pieces; c += 1 << lg) {
    typename P::raw q[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      q[r] = reinterpret_cast<const typename P::raw*>(W + ((uint64_t)id[r] < (uint64_t)V ? id[r] : 0) * ldw)[c];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row + r >= n) break;
      const bool ok = (uint64_t)id[r] < (uint64_t)V, none = id[r] == zero_token;
      float v[N];
      P::unpack(q[r], v);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = !ok ? stray : none ? 0.f : v[j] * scale;
      reinterpret_cast<typename P::raw*>(out + (row + r) * ldo)[c] = P::pack(v);
    }
  }
}

// ---- gradient: place ------------------------------------------------------------------------------------------------
constexpr int kPT = 1024;                  // threads of `place`
constexpr int kPW = kPT / 64;
constexpr int kMaxRange = 480;             // most ids a workgroup owns: with the lists below 62 KB of LDS
constexpr int kBatch = 8;                  // id loads in flight a lane
constexpr int kList = 256;                 // own ids a wave keeps in LDS; a wave with more of them reads its ids again

struct Pair {
  int32_t token, pos;
};

// Which ids a workgroup of `place` owns: those equal to its number modulo 2^lg. Low ids are the frequent ones of a
// vocabulary ordered by frequency, so neighbouring ids go to different workgroups (contiguous ranges: 130 us in place of 28
// at 32768 tokens of text, two fifths of them in the first of 256 ranges). The grouped order is by (owner, id).
struct Owners {
  int lg, range;                           // 2^lg workgroups of `range` ids
  __host__ __device__ int slot(int token) const { return (token & ((1 << lg) - 1)) * range + (token >> lg); }
  __host__ __device__ int slots() const { return range << lg; }
};

// Few positions (SMALL): the owner of a token adds its rows too, in the same launch. A token of few rows is a wave's, one of
// many (kMany) the workgroup's, each wave a sixteenth of them. Up to kSmallRows rows of kSmallNumbers in all, since one token
// may hold all of them and a CU reads some 50 GB/s. Against three launches in a graph, bf16: 200 x 64, V 1000 6.0 and 15.3 us;
// 128 x 1024, V 50257 21.5 and 22.1; 512 x 1024 of one token 29.7 and 23.6, 4096 x 128 of one token 56 and 20. Two launches and
// the workspace fewer for the host.
constexpr int64_t kSmallNumbers = 1 << 18;
constexpr int kSmallRows = 512;
static_assert(kSmallRows <= kPW * kList, "a wave's ids all fit its list");
constexpr int kMany = 64;
constexpr int kFew = 16;                   // dy rows in flight a wave

// bytes of dynamic LDS: counters, starts of the ids and their end, positions
constexpr int small_lds(int range, int n) { return (kPW * range + range + 1 + n) * (int)sizeof(int); }

struct Starter {
  int32_t token, last;
};

struct Sink {                              // what SMALL adds to
  const void* dy;
  int64_t ldy;
  void* dW;
  float scale;
  int pieces;
};

template <typename T, int N, bool SMALL>
__global__ __launch_bounds__(kPT) void place_kernel(const void* ids, int wide, int n, int64_t V, Owners own, int64_t skip,
                                                    int* starts, Pair* pairs, Sink to) {
  extern __shared__ int counts[];          // [wave][id owned]; SMALL: behind them the starts of the ids and all positions
  __shared__ __align__(16) Pair lists[kPW][kList];
  __shared__ int wsum[kPW], wbelow[kPW], many;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // (uniform: masks stay scalar)
  const int me = blockIdx.x, mask = (1 << own.lg) - 1, range = own.range;
  for (int i = tid; i < kPW * range; i += kPT) counts[i] = 0;
  __syncthreads();

  // a wave's ids: whole groups of 64, one stretch a wave, so that (wave, group, lane) ascends with the position
  const int groups = (n + 63) / 64, per = (groups + kPW - 1) / kPW;   // (no group where n is 0: nothing is read)
  const int g0 = min(wave * per, groups), g1 = min(g0 + per, groups);
  int* mine = counts + wave * range;
  Pair* list = lists[wave];
  // fn(token, position, mask of the lanes whose token is owned) for every group that has one, in order
  int below = 0;
  auto scan = [&](auto&& fn) {
    below = 0;
    auto batch = [&](int g, auto full) {   // kBatch groups; full: all of the wave's stretch and of the ids
      uint32_t id[kBatch];
      uint64_t live[kBatch];
      if (wide) {
        int64_t v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int i = (g + k) * 64 + lane;
          v[k] = reinterpret_cast<const int64_t*>(ids)[full ? i : min(i, n - 1)];
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          id[k] = (uint32_t)v[k];
          live[k] = __ballot((uint64_t)v[k] < (uint64_t)V);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int i = (g + k) * 64 + lane;
          id[k] = reinterpret_cast<const uint32_t*>(ids)[full ? i : min(i, n - 1)];
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) live[k] = __ballot(id[k] < (uint32_t)V);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int pos = (g + k) * 64 + lane;
        if (!full) live[k] = g + k < g1 ? live[k] & __ballot(pos < n) : 0ull;
        const uint64_t in = live[k] & __ballot(id[k] != (uint32_t)skip);
        const uint32_t owner = id[k] & mask;
        below += __popcll(in & __ballot(owner < (uint32_t)me));
        const uint64_t hits = in & __ballot(owner == (uint32_t)me);
        if (hits) fn((int)id[k], pos, hits);
      }
    };
    int g = g0;
    for (; g + kBatch <= g1 && (g + kBatch) * 64 <= n; g += kBatch) batch(g, std::true_type{});
    for (; g < g1; g += kBatch) batch(g, std::false_type{});
  };
  // fn(lane mask of a token, the token, its first lane) for every token among `left`, a token each turn (uniform)
  auto tokens = [&](int token, uint64_t left, auto&& fn) {
    while (left) {
      const int lead = __builtin_ctzll(left), its = __builtin_amdgcn_readlane(token, lead);
      const uint64_t same = left & __ballot(token == its);
      fn(same, its, lead);
      left &= ~same;
    }
  };
  // the first of them to the list, counted behind it 64 at a time; the others counted as they come
  int found = 0, listed = 0;
  scan([&](int token, int pos, uint64_t hits) {
    const int c = __popcll(hits);
    if (found == listed && found + c <= kList) {
      if ((hits >> lane) & 1) list[found + __popcll(hits & ((1ull << lane) - 1))] = Pair{token, pos};
      listed += c;
    } else {
      tokens(token, hits, [&](uint64_t same, int its, int lead) {
        if (lane == lead) atomicAdd(&mine[its >> own.lg], __popcll(same));
      });
    }
    found += c;
  });
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");       // (the list is the wave's own; LDS answers it in order)
  for (int i = lane; i < listed; i += 64) atomicAdd(&mine[list[i].token >> own.lg], 1);
  if (lane == 0) wbelow[wave] = below;
  __syncthreads();

  // exclusive scan: over the ids owned (a thread each), then over an id's waves
  int total = 0;
  if (tid < range)
    for (int w = 0; w < kPW; ++w) total += counts[w * range + tid];
  int incl = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();
  int at = incl - total;
  for (int w = 0; w < kPW; ++w) at += (SMALL ? 0 : wbelow[w]) + (w < wave ? wsum[w] : 0);
  int* const from = counts + kPW * range;                      // (SMALL) start of every id, their end
  int* const order = from + range + 1;                         // (SMALL) positions by id
  if (tid < range) {
    if (SMALL) {
      from[tid] = at;
      if (tid == range - 1) from[range] = at + total;
    } else {
      starts[me * range + tid] = at;
      if (me == mask && tid == range - 1) starts[own.slots()] = at + total;
    }
    for (int w = 0; w < kPW; ++w) {
      const int c = counts[w * range + tid];
      counts[w * range + tid] = at;
      at += c;
    }
  }
  __syncthreads();

  // the pairs, in order of the position within a token: the first lane that holds a token draws the places of all that do
  auto place = [&](int token, int pos, uint64_t hits) {
    tokens(token, hits, [&](uint64_t same, int its, int lead) {
      int base = 0;
      if (lane == lead) {
        base = mine[its >> own.lg];
        mine[its >> own.lg] = base + __popcll(same);
      }
      base = __builtin_amdgcn_readlane(base, lead);
      if ((same >> lane) & 1) {
        const int i = base + __popcll(same & ((1ull << lane) - 1));
        if (SMALL)
          order[i] = pos;
        else
          pairs[i] = Pair{its, pos};
      }
    });
  };
  if (SMALL || found == listed) {
    for (int i = 0; i < found; i += 64) {
      const Pair p = list[min(i + lane, found - 1)];
      place(p.token, p.pos, __ballot(i + lane < found));
    }
  } else {
    scan(place);
  }

  if constexpr (SMALL) {
    typedef Piece<T, N> P;
    typedef typename P::raw raw;
    const T* dy = reinterpret_cast<const T*>(to.dy);
    raw* dW = reinterpret_cast<raw*>(to.dW);
    const int pieces = to.pieces;
    // the sum of the rows at order[i0, i1), piece c of them (its lanes past the row read its last piece)
    auto add = [&](int i0, int i1, int c, float (&acc)[N]) {
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = 0.f;
      for (int i = i0; i < i1; i += kFew) {
        const int pos = order[min(i + (lane & (kFew - 1)), i1 - 1)];
        raw v[kFew];
#pragma unroll
        for (int k = 0; k < kFew; ++k)
          v[k] = reinterpret_cast<const raw*>(dy + (int64_t)__builtin_amdgcn_readlane(pos, k) * to.ldy)[min(c, pieces - 1)];
#pragma unroll
        for (int k = 0; k < kFew; ++k) {
          float x[N];
          P::unpack(v[k], x);
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] += i + k < i1 ? x[j] : 0.f;
        }
      }
    };
    if (tid == 0) many = 0;
    __syncthreads();
    int* const big = counts;               // (the counters are done with)
    for (int r = wave; r < range; r += kPW) {
      const int64_t token = ((int64_t)r << own.lg) + me;
      if (token >= V) break;
      const int i0 = __builtin_amdgcn_readfirstlane(from[r]), i1 = __builtin_amdgcn_readfirstlane(from[r + 1]);
      if (i1 - i0 > kMany) {
        if (lane == 0) big[atomicAdd(&many, 1)] = r;
        continue;
      }
      for (int c = lane; c - lane < pieces; c += 64) {
        float acc[N];
        add(i0, i1, c, acc);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = i1 > i0 ? acc[j] * to.scale : 0.f;
        if (c < pieces) dW[token * pieces + c] = P::pack(acc);
      }
    }
    __syncthreads();
    float* const parts = reinterpret_cast<float*>(&lists[0][0]);               // [wave][64 N]
    static_assert(sizeof(lists) >= kPW * 64 * N * sizeof(float), "the partial sums lie over the lists");
    for (int b = 0; b < many; ++b) {
      const int r = big[b], i0 = from[r], i1 = from[r + 1], stretch = (i1 - i0 + kPW - 1) / kPW;
      const int j0 = __builtin_amdgcn_readfirstlane(min(i0 + wave * stretch, i1)), j1 = min(j0 + stretch, i1);
      for (int first = 0; first < pieces; first += 64) {
        float acc[N];
        add(j0, j1, first + lane, acc);
#pragma unroll
        for (int j = 0; j < N; ++j) parts[(wave * 64 + lane) * N + j] = acc[j];
        __syncthreads();
        const int e = first * N + tid;
        if (tid < 64 * N && e < pieces * N) {
          float x = 0.f;
#pragma unroll
          for (int w = 0; w < kPW; ++w) x += parts[w * 64 * N + tid];
          Elem<T>::store(reinterpret_cast<T*>(to.dW) + (((int64_t)r << own.lg) + me) * pieces * N + e, x * to.scale);
        }
        __syncthreads();
      }
    }
  }
}

// ---- gradient: sum and join -----------------------------------------------------------------------------------------
constexpr int kST = 256;                   // threads of `sum`: four waves, a chunk and 64 pieces of the row each
constexpr int kRows = 32;                  // dy rows in flight a wave: a whole chunk of up to 32768 positions, so that the
                                           // rows cost one round trip (8 in flight: 33 us in place of 19 at 32768 x 1024)

constexpr int kZero = 16;                  // tokens a wave of `sum` looks up that finds rows to fill with zeros

// The first `sums` workgroups add, the others fill the rows that no position holds with zeros: most of dW's bytes, written
// while the dy rows are read (by `place` instead: 28 us in all in place of 22 at 128 x 1024 bf16, V 50257; the same at 32768).
// starter[c]: the token that began in chunk c and goes on behind it, and the last chunk that holds it (token -1: none).
// partial sums of chunk c: [2 c] of a first token that began in an earlier chunk, [2 c + 1] of a last token that began in
// this chunk and goes on in the next; d floats each
template <typename T, int N>
__global__ __launch_bounds__(kST) void sum_kernel(const T* dy, int64_t ldy, const Pair* pairs, const int* starts, int64_t V,
                                                  Owners own, int sums, int chunk, int slices, float scale, T* dW, int d,
                                                  int pieces, float* part, Starter* starter) {
  typedef Piece<T, N> P;
  typedef typename P::raw raw;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x >= sums) {
    const int64_t first = ((int64_t)((int)blockIdx.x - sums) * (kST / 64) + wave) * kZero;
    const int64_t mine = first + lane;
    bool empty = false;
    if (lane < kZero && mine < V) {
      const int slot = own.slot((int)mine);
      empty = starts[slot] == starts[slot + 1];
    }
    float z[N];
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = 0.f;
    const raw zero = P::pack(z);
    for (uint64_t left = __ballot(empty); left; left &= left - 1) {            // uniform in the wave
      raw* row = reinterpret_cast<raw*>(dW) + (first + __builtin_ctzll(left)) * pieces;
      for (int c = lane; c < pieces; c += 64) row[c] = zero;
    }
    return;
  }
  const int unit = __builtin_amdgcn_readfirstlane((int)blockIdx.x * (kST / 64) + wave);
  const int c = unit / slices;
  const int piece = (unit % slices) * 64 + lane;
  const int m = load_uniform(starts + own.slots());
  const int64_t b64 = (int64_t)c * chunk;
  const bool notes = unit % slices == 0 && lane == 0;          // (one of the chunk's waves)
  if (b64 >= m) {
    if (notes) starter[c] = Starter{-1, 0};
    return;
  }
  const int b = (int)b64, e = min(b + chunk, m);
  const int col = min(piece, pieces - 1);                      // (lanes past the row read its last piece and write nothing)
  const bool in = piece < pieces;
  const int before = b > 0 ? pairs[b - 1].token : -1, after = e < m ? pairs[e].token : -1;
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  int token = -1;
  bool open = false;                                           // the token in hand began before this chunk
  auto flush = [&](bool ends) {
    if (!open && ends) {
      float o[N];
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = acc[j] * scale;
      if (in) reinterpret_cast<raw*>(dW)[(int64_t)token * pieces + piece] = P::pack(o);
    } else if (in) {
      float* p = part + (2 * (int64_t)c + (open ? 0 : 1)) * d + piece * N;
#pragma unroll
      for (int j = 0; j < N; ++j) p[j] = acc[j];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    open = false;
  };
  for (int i = b; i < e; i += kRows) {
    const Pair pr = pairs[min(i + (lane & (kRows - 1)), e - 1)];
    raw v[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k)                            // (behind the chunk's end: its last row again)
      v[k] = reinterpret_cast<const raw*>(dy + (int64_t)__builtin_amdgcn_readlane(pr.pos, k) * ldy)[col];
    if (i == b) {
      token = __builtin_amdgcn_readlane(pr.token, 0);
      open = token == before;
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (i + k < e) {                                         // uniform
        const int t = __builtin_amdgcn_readlane(pr.token, k);
        if (t != token) {
          flush(true);
          token = t;
        }
        float x[N];
        P::unpack(v[k], x);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += x[j];
      }
    }
  }
  if (notes) {
    const bool starts_here = !open && token == after;
    starter[c] = Starter{starts_here ? token : -1, starts_here ? (starts[own.slot(token) + 1] - 1) / chunk : 0};
  }
  flush(token != after);
}

constexpr int kJW = 8;                     // waves of `join`: each an eighth of a token's chunks, 64 lanes of M columns

template <typename T, int M>
__global__ __launch_bounds__(kJW * 64) void join_kernel(const Starter* starter, float scale, const float* part, T* dW, int d) {
  __shared__ float eighth[kJW][64 * M];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t c = blockIdx.x;
  const Starter s0 = starter[c];
  const int token = s0.token;
  if (token < 0) return;                                       // uniform
  const int count = s0.last - (int)c + 1, per = (count + kJW - 1) / kJW;      // chunks c .. last hold the token
  const int k0 = min(wave * per, count), k1 = min(k0 + per, count);
  const int first = blockIdx.y * 64 * M, col = first + lane * M;
  float s[M];
#pragma unroll
  for (int j = 0; j < M; ++j) s[j] = 0.f;
  if (col < d) {
#pragma unroll 8
    for (int k = k0; k < k1; ++k) {
      const float* p = part + (2 * (c + k) + (k == 0 ? 1 : 0)) * d + col;
#pragma unroll
      for (int j = 0; j < M; ++j) s[j] += p[j];
    }
  }
#pragma unroll
  for (int j = 0; j < M; ++j) eighth[wave][lane * M + j] = s[j];
  __syncthreads();
  if (tid < 64 * M && first + tid < d) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kJW; ++w) x += eighth[w][tid];
    Elem<T>::store(dW + (int64_t)token * d + first + tid, x * scale);
  }
}

// ---- sizes ----------------------------------------------------------------------------------------------------------
Owners owners_of(int64_t V) {              // one workgroup of `place` a CU, or as many as kMaxRange asks for
  Owners o{8, 0};
  while (((V + (1 << o.lg) - 1) >> o.lg) > kMaxRange) ++o.lg;
  o.range = (int)((V + (1 << o.lg) - 1) >> o.lg);
  return o;
}
int chunk_of(int64_t n) {                  // positions a wave adds: 32, or up to 1024 chunks
  int64_t c = 32;
  while (c * 1024 < n) c *= 2;
  return (int)c;
}
int64_t align16(int64_t b) { return (b + 15) / 16 * 16; }

struct Layout {
  int64_t starts, pairs, starter, part, bytes, chunks;
};
Layout layout_of(int64_t n, int64_t V, int d) {
  Layout l;
  const int c = chunk_of(n);
  l.chunks = (n + c - 1) / c;
  l.starts = 0;
  l.pairs = align16((owners_of(V).slots() + 1) * 4);
  l.starter = l.pairs + align16(n * (int64_t)sizeof(Pair));
  // (waves of the last workgroup past the chunks note too)
  l.part = l.starter + align16((l.chunks + kST / 64) * (int64_t)sizeof(Starter));
  l.bytes = l.part + 2 * l.chunks * d * 4;
  return l;
}

bool small(int64_t n, int d) { return n <= kSmallRows && n * d <= kSmallNumbers; }
bool aligned(int dtype, const void* p) { return (uintptr_t)p % (dtype == DH_BF16 ? 2 : 4) == 0; }
bool sizes_ok(int64_t n, int64_t V, int d) {
  return n >= 0 && n < ((int64_t)1 << 24) && V >= 1 && V <= ((int64_t)1 << 24) && d >= 1 && d <= (1 << 20);
}

template <typename T, int N>
int lookup(const void* W, int64_t ldw, int64_t V, int d, const void* ids, int wide, int64_t n, float scale, int64_t zero,
           void* out, int64_t ldo, hipStream_t s) {
  const int pieces = d / N;
  int lg = 0;
  while (lg < 8 && (1 << lg) < pieces) ++lg;
  // four rows a lane where that still leaves 4096 waves
  const int R = n * pieces >= (int64_t)4096 * 64 * 4 ? 4 : 1;
  const int64_t per = (int64_t)R << (8 - lg);
  const dim3 grid((unsigned)((n + per - 1) / per));
  if (R == 4)
    lookup_kernel<T, N, 4><<<grid, dim3(kLT), 0, s>>>((const T*)W, ldw, V, ids, wide, n, scale, zero, (T*)out, ldo, pieces, lg);
  else
    lookup_kernel<T, N, 1><<<grid, dim3(kLT), 0, s>>>((const T*)W, ldw, V, ids, wide, n, scale, zero, (T*)out, ldo, pieces, lg);
  return dh_check_launch("dh_embed_fwd");
}

template <typename T, int N>
int gradient(const void* dy, int64_t ldy, const void* ids, int wide, int64_t n, int64_t V, int d, float scale, int64_t skip,
             void* dW, char* ws, hipStream_t s) {
  const int pieces = d / N, chunk = chunk_of(n);
  const Owners own = owners_of(V);
  const Layout l = layout_of(n, V, d);
  int* starts = (int*)(ws + l.starts);
  Pair* pairs = (Pair*)(ws + l.pairs);
  Starter* starter = (Starter*)(ws + l.starter);
  float* part = (float*)(ws + l.part);
  const Sink to{dy, ldy, dW, scale, pieces};
  const dim3 owners(1u << own.lg);
  if (small(n, d)) {
    const int lds = small_lds(own.range, (int)n);
    if (lds > 28 << 10) {                  // (64 KB with the lists)
      // the kernel's limit is the process's: always the same, so that no host thread lowers it before another's launch
      constexpr int most = small_lds(kMaxRange, kSmallRows);
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&place_kernel<T, N, true>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, most);
      if (e != hipSuccess) return dh_fail(DH_ERR_LAUNCH_FAILED, "dh_embed_bwd: %d bytes of LDS: %s", most, hipGetErrorString(e));
    }
    place_kernel<T, N, true><<<owners, dim3(kPT), lds, s>>>(ids, wide, (int)n, V, own, skip, starts, pairs, to);
    return dh_check_launch("dh_embed_bwd");
  }
  place_kernel<T, N, false><<<owners, dim3(kPT), kPW * own.range * sizeof(int), s>>>(ids, wide, (int)n, V, own, skip, starts,
                                                                                    pairs, to);
  if (int st = dh_check_launch("dh_embed_bwd")) return st;
  const int slices = (pieces + 63) / 64;
  const int sums = (int)((l.chunks * slices + kST / 64 - 1) / (kST / 64));
  const int zeros = (int)((V + kZero * (kST / 64) - 1) / (kZero * (kST / 64)));
  sum_kernel<T, N><<<dim3((unsigned)(sums + zeros)), dim3(kST), 0, s>>>((const T*)dy, ldy, pairs, starts, V, own, sums, chunk,
                                                                       slices, scale, (T*)dW, d, pieces, part, starter);
  if (int st = dh_check_launch("dh_embed_bwd")) return st;
  if (l.chunks > 1) {
    constexpr int M = N == 1 ? 1 : 4;
    join_kernel<T, M><<<dim3((unsigned)(l.chunks - 1), (unsigned)((d + 64 * M - 1) / (64 * M))), dim3(kJW * 64), 0, s>>>(
        starter, scale, part, (T*)dW, d);
    return dh_check_launch("dh_embed_bwd");
  }
  return 0;
}

}  // namespace

extern "C" int dh_embed_fwd(int dtype, const void* W, int64_t ldw, int64_t V, int d, const void* ids, int ids_bits, int64_t n,
                            float scale, int64_t zero_token, void* out, int64_t ldo, void* stream) {
  const char* who = "dh_embed_fwd";
  DH_REQUIRE(dtype == DH_F32 || dtype == DH_BF16, DH_ERR_UNSUPPORTED_DTYPE, "%s: dtype %d", who, dtype);
  DH_REQUIRE(ids_bits == 32 || ids_bits == 64, DH_ERR_UNSUPPORTED_DTYPE, "%s: ids of %d bits", who, ids_bits);
  DH_REQUIRE(sizes_ok(n, V, d), DH_ERR_UNSUPPORTED_SHAPE, "%s: n=%lld V=%lld d=%d", who, (long long)n, (long long)V, d);
  DH_REQUIRE(zero_token >= -1 && zero_token <= V, DH_ERR_INVALID_ARG, "%s: zero_token %lld", who, (long long)zero_token);
  DH_REQUIRE(ldw >= d && ldo >= d, DH_ERR_INVALID_ARG, "%s: row strides %lld, %lld below d=%d", who, (long long)ldw,
             (long long)ldo, d);
  if (n == 0) return 0;
  DH_REQUIRE(W && ids && out, DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE(aligned(dtype, W) && aligned(dtype, out) && (uintptr_t)ids % (ids_bits / 8) == 0, DH_ERR_INVALID_ARG,
             "%s: operands not aligned to their elements", who);
  hipStream_t s = (hipStream_t)stream;
  const int wide = ids_bits == 64;
  const int N = dtype == DH_BF16 ? 8 : 4;
  // 16-byte pieces where every row of both sides starts on one, single elements otherwise
  const bool pieces = d % N == 0 && ldw % N == 0 && ldo % N == 0 && (uintptr_t)W % 16 == 0 && (uintptr_t)out % 16 == 0;
  if (dtype == DH_BF16)
    return pieces ? lookup<bf16_t, 8>(W, ldw, V, d, ids, wide, n, scale, zero_token, out, ldo, s)
                  : lookup<bf16_t, 1>(W, ldw, V, d, ids, wide, n, scale, zero_token, out, ldo, s);
  return pieces ? lookup<float, 4>(W, ldw, V, d, ids, wide, n, scale, zero_token, out, ldo, s)
                : lookup<float, 1>(W, ldw, V, d, ids, wide, n, scale, zero_token, out, ldo, s);
}

extern "C" int64_t dh_embed_bwd_workspace_bytes(int64_t n, int64_t V, int d) {
  return !sizes_ok(n, V, d) ? -1 : small(n, d) ? 0 : layout_of(n, V, d).bytes;
}

extern "C" int dh_embed_bwd(int dtype, const void* dy, int64_t ldy, const void* ids, int ids_bits, int64_t n, int64_t V, int d,
                            float scale, int64_t skip_token, void* dW, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const char* who = "dh_embed_bwd";
  DH_REQUIRE(dtype == DH_F32 || dtype == DH_BF16, DH_ERR_UNSUPPORTED_DTYPE, "%s: dtype %d", who, dtype);
  DH_REQUIRE(ids_bits == 32 || ids_bits == 64, DH_ERR_UNSUPPORTED_DTYPE, "%s: ids of %d bits", who, ids_bits);
  DH_REQUIRE(sizes_ok(n, V, d), DH_ERR_UNSUPPORTED_SHAPE, "%s: n=%lld V=%lld d=%d", who, (long long)n, (long long)V, d);
  DH_REQUIRE(skip_token >= -1 && skip_token < V, DH_ERR_INVALID_ARG, "%s: skip_token %lld", who, (long long)skip_token);
  DH_REQUIRE(ldy >= d, DH_ERR_INVALID_ARG, "%s: row stride %lld below d=%d", who, (long long)ldy, d);
  const int64_t need = dh_embed_bwd_workspace_bytes(n, V, d);
  DH_REQUIRE(dW && (n == 0 || (dy && ids)), DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE(workspace_bytes >= need && (need == 0 || workspace) && (uintptr_t)workspace % 16 == 0, DH_ERR_INVALID_ARG,
             "%s: workspace of %lld bytes, 16-byte aligned %lld needed", who, (long long)workspace_bytes, (long long)need);
  DH_REQUIRE(aligned(dtype, dy) && aligned(dtype, dW) && (uintptr_t)ids % (ids_bits / 8) == 0, DH_ERR_INVALID_ARG,
             "%s: operands not aligned to their elements", who);
  hipStream_t s = (hipStream_t)stream;
  const int wide = ids_bits == 64;
  const int N = dtype == DH_BF16 ? 8 : 4;
  const bool pieces = d % N == 0 && ldy % N == 0 && (uintptr_t)dy % 16 == 0 && (uintptr_t)dW % 16 == 0;
  char* ws = (char*)workspace;
  if (dtype == DH_BF16)
    return pieces ? gradient<bf16_t, 8>(dy, ldy, ids, wide, n, V, d, scale, skip_token, dW, ws, s)
                  : gradient<bf16_t, 1>(dy, ldy, ids, wide, n, V, d, scale, skip_token, dW, ws, s);
  return pieces ? gradient<float, 4>(dy, ldy, ids, wide, n, V, d, scale, skip_token, dW, ws, s)
                : gradient<float, 1>(dy, ldy, ids, wide, n, V, d, scale, skip_token, dW, ws, s);
}
