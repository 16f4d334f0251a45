// Embedding rows and their gradient, for gfx950:
//   out[n] = rnd(scale W[id_n])                       (dh_embed_fwd)
//   dW[v]  = rnd(scale sum_{n: id_n = v} dy[n])       (dh_embed_bwd; every row of dW is written)
// The parallel forward's embedding (reference dispatcher_hybrid/modeling_dispatcher.py:340) and its autograd gradient.
//
// The gradient groups the positions by token: sums in fp32 over a token's positions in ascending order, split at fixed
// places, so the same call gives the same bits whatever the launch order. Three launches:
//   place  every workgroup owns a range of token ids and reads ALL ids itself (8 n bytes from L2, cheaper than the launches
//          of a sort that shares work between workgroups): it counts the ids below its range (its offset in the grouped
//          order) and its own per (wave, token), scans, and writes its (token, position) pairs, positions ascending. The
//          rows of its range that no position holds it fills with zeros: most of dW's bytes, written while other
//          workgroups still count.
//   sum    the grouped list in equal chunks, whatever the distribution of the tokens: a wave adds the dy rows of a chunk and
//          writes a token's row when the token's positions all lie in the chunk; the sums of a first or last token that
//          reaches into the neighbouring chunks go to the workspace.
//   join   adds the chunk sums of every token that lies in more than one chunk.
// Bytes: n d read, V d written (and the ids). Ids outside [0, V) hold no gradient (their rows of `out` are NaN).

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

// 2^lg lanes hold a row of `pieces` pieces; 2^(8 - lg) rows a workgroup
template <typename T, int N>
__global__ __launch_bounds__(kLT) void lookup_kernel(const T* W, int64_t ldw, int64_t V, const void* ids, int wide, int64_t n,
                                                     float scale, int64_t zero_token, T* out, int64_t ldo, int pieces,
                                                     int lg) {
  typedef Piece<T, N> P;
  const int64_t row = ((int64_t)blockIdx.x << (8 - lg)) + (threadIdx.x >> lg);
  if (row >= n) return;
  const int64_t id = load_id(ids, wide, row);
  const bool ok = id >= 0 && id < V, none = id == zero_token;
  const typename P::raw* src = reinterpret_cast<const typename P::raw*>(W + (ok ? id : 0) * ldw);
  typename P::raw* dst = reinterpret_cast<typename P::raw*>(out + row * ldo);
  for (int c = threadIdx.x & ((1 << lg) - 1); c < pieces; c += 1 << lg) {
    float v[N];
    P::unpack(src[c], v);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = none ? 0.f : ok ? v[j] * scale : __builtin_nanf("");
    dst[c] = P::pack(v);
  }
}

// ---- gradient: place ------------------------------------------------------------------------------------------------
constexpr int kPT = 1024;                  // threads of `place`
constexpr int kPW = kPT / 64;
constexpr int kMaxRange = 512;             // most ids a workgroup owns: kPW * kMaxRange counters, 32 KB of LDS
constexpr int kBatch = 8;                  // id loads in flight a lane

struct Pair {
  int32_t token, pos;
};

template <typename T, int N>
__global__ __launch_bounds__(kPT) void place_kernel(const void* ids, int wide, int n, int64_t V, int range, int64_t skip,
                                                    int* starts, Pair* pairs, T* dW, int pieces) {
  extern __shared__ int counts[];          // [wave][token of the range]
  __shared__ int wsum[kPW], wbelow[kPW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = (int64_t)blockIdx.x * range;
  const int own = (int)min((int64_t)range, V - first);
  for (int i = tid; i < kPW * range; i += kPT) counts[i] = 0;
  __syncthreads();

  // a wave's ids: whole groups of 64, one stretch a wave, so that (wave, group, lane) ascends with the position
  const int groups = (n + 63) / 64, per = (groups + kPW - 1) / kPW;
  const int g0 = min(wave * per, groups), g1 = min(g0 + per, groups);
  int* mine = counts + wave * range;
  int below = 0;
  for (int g = g0; g < g1; g += kBatch) {
    int64_t id[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = (g + k) * 64 + lane;
      id[k] = g + k < g1 && i < n ? load_id(ids, wide, i) : -1;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const bool live = id[k] >= 0 && id[k] < V && id[k] != skip;
      below += live && id[k] < first;
      if (live && id[k] >= first && id[k] < first + own) atomicAdd(&mine[(int)(id[k] - first)], 1);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o);
  if (lane == 0) wbelow[wave] = below;
  __syncthreads();

  // exclusive scan: over the tokens of the range (a thread each), then over a token's waves
  int total = 0;
  if (tid < own)
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
  for (int w = 0; w < kPW; ++w) at += wbelow[w] + (w < wave ? wsum[w] : 0);
  if (tid < own) {
    starts[first + tid] = at;
    if (first + tid == V - 1) starts[V] = at + total;
    for (int w = 0; w < kPW; ++w) {
      const int c = counts[w * range + tid];
      counts[w * range + tid] = at;
      at += c;
    }
  }
  __syncthreads();

  // the pairs, in order of the position within a token: of the lanes that hold one token the first draws their places
  for (int g = g0; g < g1; g += kBatch) {
    int64_t id[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = (g + k) * 64 + lane;
      id[k] = g + k < g1 && i < n ? load_id(ids, wide, i) : -1;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const bool hit = id[k] >= first && id[k] < first + own && id[k] != skip;
      const int t = hit ? (int)(id[k] - first) : -1;
      uint64_t left = __ballot(hit);
      while (left) {                                           // uniform; a token leaves in each turn
        const int lead = __builtin_ctzll(left);
        const int lt = __builtin_amdgcn_readlane(t, lead);
        const uint64_t same = __ballot(hit && t == lt);
        int base = 0;
        if (lane == lead) base = atomicAdd(&mine[lt], __popcll(same));
        base = __builtin_amdgcn_readlane(base, lead);
        if (hit && t == lt)
          pairs[base + __popcll(same & ((1ull << lane) - 1))] = Pair{(int32_t)id[k], (g + k) * 64 + lane};
        left &= ~same;
      }
    }
  }

  // rows that no position holds
  __syncthreads();
  if (tid < own) counts[tid] = total;
  __syncthreads();
  typedef typename Piece<T, N>::raw raw;
  raw zero;
  {
    float z[N];
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = 0.f;
    zero = Piece<T, N>::pack(z);
  }
  for (int r = wave; r < own; r += kPW) {
    if (counts[r]) continue;                                   // uniform in the wave
    raw* row = reinterpret_cast<raw*>(dW) + (first + r) * pieces;
    for (int c = lane; c < pieces; c += 64) row[c] = zero;
  }
}

// ---- gradient: sum and join -----------------------------------------------------------------------------------------
constexpr int kST = 256;                   // threads of `sum`: four waves, a chunk and 64 pieces of the row each
constexpr int kRows = 8;                   // dy rows in flight

// partial sums of chunk c: [2 c] of a first token that began in an earlier chunk, [2 c + 1] of a last token that began in
// this chunk and goes on in the next; d floats each
template <typename T, int N>
__global__ __launch_bounds__(kST) void sum_kernel(const T* dy, int64_t ldy, const Pair* pairs, const int* count, int chunk,
                                                  int slices, float scale, T* dW, int d, int pieces, float* part) {
  typedef Piece<T, N> P;
  typedef typename P::raw raw;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (kST / 64) + (threadIdx.x >> 6);
  const int64_t c = unit / slices;
  const int piece = (int)(unit % slices) * 64 + lane;
  const int m = load_uniform(count);
  const int64_t b = c * chunk;
  if (b >= m) return;
  const int e = (int)min(b + chunk, (int64_t)m);
  const bool in = piece < pieces;
  const int before = b > 0 ? pairs[b - 1].token : -1, after = e < m ? pairs[e].token : -1;
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  int token = pairs[b].token;
  bool open = token == before;             // the token in hand began before this chunk
  auto flush = [&](bool ends) {
    if (in) {
      if (!open && ends) {
        float o[N];
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = acc[j] * scale;
        reinterpret_cast<raw*>(dW)[(int64_t)token * pieces + piece] = P::pack(o);
      } else {
        float* p = part + (2 * c + (open ? 0 : 1)) * d + piece * N;
#pragma unroll
        for (int j = 0; j < N; ++j) p[j] = acc[j];
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    open = false;
  };
  for (int i = (int)b; i < e; i += kRows) {
    Pair pr[kRows];
    raw v[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      pr[k] = pairs[min(i + k, e - 1)];
      if (in) v[k] = reinterpret_cast<const raw*>(dy + (int64_t)pr[k].pos * ldy)[piece];
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (i + k < e) {
        if (pr[k].token != token) {
          flush(true);
          token = pr[k].token;
        }
        if (in) {
          float x[N];
          P::unpack(v[k], x);
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] += x[j];
        }
      }
    }
  }
  flush(token != after);
}

constexpr int kJT = 256;                   // threads of `join`: four waves, each a quarter of a token's chunks, 64 columns

template <typename T>
__global__ __launch_bounds__(kJT) void join_kernel(const Pair* pairs, const int* starts, int64_t V, int chunk, float scale,
                                                   const float* part, T* dW, int d) {
  __shared__ float quarter[kJT / 64][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m = load_uniform(starts + V);
  const int64_t c = blockIdx.x;
  const int64_t e = (c + 1) * chunk;
  if (e >= m) return;                                          // uniform: the last chunk, or none
  const int token = pairs[e - 1].token;
  if (pairs[e].token != token) return;
  if (starts[token] < c * chunk) return;                       // began earlier: that chunk joins it
  const int last = (starts[token + 1] - 1) / chunk;            // chunks c .. last hold the token
  const int count = last - (int)c + 1, per = (count + 3) / 4;
  const int k0 = min(wave * per, count), k1 = min(k0 + per, count);
  const int col = blockIdx.y * 64 + lane;
  float s = 0.f;
  if (col < d)
#pragma unroll 8
    for (int k = k0; k < k1; ++k) s += part[(2 * (c + k) + (k == 0 ? 1 : 0)) * d + col];
  quarter[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < d)
    Elem<T>::store(dW + (int64_t)token * d + col,
                   ((quarter[0][lane] + quarter[1][lane]) + (quarter[2][lane] + quarter[3][lane])) * scale);
}

// ---- sizes ----------------------------------------------------------------------------------------------------------
int range_of(int64_t V) {                  // ids a workgroup of `place` owns: one workgroup a CU, or kMaxRange
  const int64_t r = (V + 255) / 256;
  return (int)(r < kMaxRange ? r : kMaxRange);
}
int chunk_of(int64_t n) {                  // positions a wave adds: 32, or up to 1024 chunks
  int64_t c = 32;
  while (c * 1024 < n) c *= 2;
  return (int)c;
}
int64_t align16(int64_t b) { return (b + 15) / 16 * 16; }

struct Layout {
  int64_t starts, pairs, part, bytes, chunks;
};
Layout layout_of(int64_t n, int64_t V, int d) {
  Layout l;
  const int c = chunk_of(n);
  l.chunks = (n + c - 1) / c;
  l.starts = 0;
  l.pairs = align16((V + 1) * 4);
  l.part = l.pairs + align16(n * (int64_t)sizeof(Pair));
  l.bytes = l.part + 2 * l.chunks * d * 4;
  return l;
}

bool sizes_ok(int64_t n, int64_t V, int d) {
  return n >= 0 && n < ((int64_t)1 << 24) && V >= 1 && V <= ((int64_t)1 << 24) && d >= 1 && d <= (1 << 20);
}

template <typename T, int N>
int lookup(const void* W, int64_t ldw, int64_t V, int d, const void* ids, int wide, int64_t n, float scale, int64_t zero,
           void* out, int64_t ldo, hipStream_t s) {
  const int pieces = d / N;
  int lg = 0;
  while (lg < 8 && (1 << lg) < pieces) ++lg;
  const int64_t per = (int64_t)1 << (8 - lg);
  const int64_t grid = (n + per - 1) / per;
  lookup_kernel<T, N><<<dim3((unsigned)grid), dim3(kLT), 0, s>>>((const T*)W, ldw, V, ids, wide, n, scale, zero, (T*)out,
                                                                 ldo, pieces, lg);
  return dh_check_launch("dh_embed_fwd");
}

template <typename T, int N>
int gradient(const void* dy, int64_t ldy, const void* ids, int wide, int64_t n, int64_t V, int d, float scale, int64_t skip,
             void* dW, char* ws, hipStream_t s) {
  const int pieces = d / N, range = range_of(V), chunk = chunk_of(n);
  const Layout l = layout_of(n, V, d);
  int* starts = (int*)(ws + l.starts);
  Pair* pairs = (Pair*)(ws + l.pairs);
  float* part = (float*)(ws + l.part);
  place_kernel<T, N><<<dim3((unsigned)((V + range - 1) / range)), dim3(kPT), kPW * range * sizeof(int), s>>>(
      ids, wide, (int)n, V, range, skip, starts, pairs, (T*)dW, pieces);
  if (int st = dh_check_launch("dh_embed_bwd")) return st;
  if (n == 0) return 0;
  const int slices = (pieces + 63) / 64;
  const int64_t units = l.chunks * slices;
  sum_kernel<T, N><<<dim3((unsigned)((units + kST / 64 - 1) / (kST / 64))), dim3(kST), 0, s>>>(
      (const T*)dy, ldy, pairs, starts + V, chunk, slices, scale, (T*)dW, d, pieces, part);
  if (int st = dh_check_launch("dh_embed_bwd")) return st;
  if (l.chunks > 1) {
    join_kernel<T><<<dim3((unsigned)(l.chunks - 1), (unsigned)((d + 63) / 64)), dim3(kJT), 0, s>>>(
        pairs, starts, V, chunk, scale, part, (T*)dW, d);
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
  DH_REQUIRE(ldw >= d && ldo >= d, DH_ERR_INVALID_ARG, "%s: row strides %lld, %lld below d=%d", who, (long long)ldw,
             (long long)ldo, d);
  if (n == 0) return 0;
  DH_REQUIRE(W && ids && out, DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
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
  return sizes_ok(n, V, d) ? layout_of(n, V, d).bytes : -1;
}

extern "C" int dh_embed_bwd(int dtype, const void* dy, int64_t ldy, const void* ids, int ids_bits, int64_t n, int64_t V, int d,
                            float scale, int64_t skip_token, void* dW, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const char* who = "dh_embed_bwd";
  DH_REQUIRE(dtype == DH_F32 || dtype == DH_BF16, DH_ERR_UNSUPPORTED_DTYPE, "%s: dtype %d", who, dtype);
  DH_REQUIRE(ids_bits == 32 || ids_bits == 64, DH_ERR_UNSUPPORTED_DTYPE, "%s: ids of %d bits", who, ids_bits);
  DH_REQUIRE(sizes_ok(n, V, d), DH_ERR_UNSUPPORTED_SHAPE, "%s: n=%lld V=%lld d=%d", who, (long long)n, (long long)V, d);
  DH_REQUIRE(ldy >= d, DH_ERR_INVALID_ARG, "%s: row stride %lld below d=%d", who, (long long)ldy, d);
  DH_REQUIRE(dW && workspace && (n == 0 || (dy && ids)), DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  DH_REQUIRE(workspace_bytes >= layout_of(n, V, d).bytes && (uintptr_t)workspace % 16 == 0, DH_ERR_INVALID_ARG,
             "%s: workspace of %lld bytes, 16-byte aligned %lld needed", who, (long long)workspace_bytes,
             (long long)layout_of(n, V, d).bytes);
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
