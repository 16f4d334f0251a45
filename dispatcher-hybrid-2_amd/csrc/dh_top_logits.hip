// The K largest logits of every row and their tokens, for gfx950: a teacher's targets for distillation.
//   values[r, 0 .. K) = the K largest of logits[r], falling;  tokens[r, j] = where they stand, the lower token first where
//   values are equal (0.0 and -0.0 are), NaN above every number.
//
// A value and its token make one 64-bit key, different for every element: an order-preserving 32-bit image of the value
// above the complement of the token. The K largest keys are the answer, with no case for ties.
//
// Compares only, so the one read of the row bounds it. Up to 65536 logits a workgroup keeps its whole
// row in registers (held_kernel):
//   - each thread's largest value; the K-th largest of those, or a value slightly below it (bisection over their images by one
//     wave, ended once K to K + kSlack of them are at least that value), is a lower bound of the K-th largest logit;
//   - the logits at least as large (K and a few tens more: a thread rarely holds two) go to LDS as keys;
//   - a key's rank is the number of larger keys; ranks below K write their value and token.
// Ties at the bound (masked vocabularies, constant rows) take the lower tokens first; rows whose large values all stand
// where few threads read them, more than LDS holds, are bisected as a whole, slowly.
// Longer rows are streamed (stream_kernel): a wave reads its part and keeps, in LDS, every element above the value of about
// the K-th best so far; when the next tile might not fit it cuts the buffer back and that value rises (two to four cuts for
// values in no order, one a tile for rising ones). Several waves share a row where rows are few; their lists are sorted
// together.

#include "dh_common.h"

namespace {

constexpr int kBuf = 1024;                 // keys a wave holds: more than kMaxK plus a tile
constexpr int kMaxK = 256;
constexpr int kPer = kBuf / 64;
constexpr int kLoads = 4;                  // 16-byte loads in flight a lane
constexpr int kSlack = 32;                 // keys more than K that end a bisection

__device__ __forceinline__ uint32_t image_of(float x) {        // a < b  <=>  image(a) < image(b); NaN above all
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);                // -0.0 as 0.0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

__device__ __forceinline__ int below_me(uint64_t mask) {       // set bits of the lanes below this one
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Cuts the wave's keys buf[0, n) (n > K) to their K largest, or to K .. K + slack of them where the bisection meets such a
// count first, in no order; n becomes their number. Returns the image that every key kept is at least: first of all keys,
// then, where more than K + slack share it, the keys of the lower tokens.
__device__ __forceinline__ uint32_t cut(uint64_t* buf, int& n, int K, int slack, int lane) {
  uint32_t hi[kPer], lo[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const uint64_t k = j * 64 + lane < n ? buf[j * 64 + lane] : 0ull;
    hi[j] = (uint32_t)(k >> 32);
    lo[j] = (uint32_t)k;
  }
  uint32_t a = 1u, b = 0xffffffffu;                            // the largest image v with count(hi >= v) >= K
  int at_least = n;                                            // count(hi >= a)
  while (a < b && at_least > K + slack) {
    const uint32_t mid = a + ((b - a) >> 1) + ((b - a) & 1u);
    int c = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) c += __popcll(__ballot(hi[j] >= mid));
    if (c >= K) {
      a = mid;
      at_least = c;
    } else {
      b = mid - 1u;
    }
  }
  uint32_t t = 0u;                                             // least complement of a token kept at image a
  if (at_least > K + slack) {                                  // ties at a: the lowest tokens of them
    int above = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) above += __popcll(__ballot(hi[j] > a));
    const int need = K - above;
    uint32_t ta = 0u, tb = 0xffffffffu;
    while (ta < tb) {
      const uint32_t mid = ta + ((tb - ta) >> 1) + ((tb - ta) & 1u);
      int c = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) c += __popcll(__ballot(hi[j] == a && lo[j] >= mid));
      if (c >= need) ta = mid; else tb = mid - 1u;
    }
    t = ta;
  }
  int at = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const bool keep = hi[j] != 0u && (hi[j] > a || (hi[j] == a && lo[j] >= t));
    const uint64_t mask = __ballot(keep);
    const uint64_t k = ((uint64_t)hi[j] << 32) | lo[j];
    if (keep) buf[at + below_me(mask)] = k;
    at += __popcll(mask);
  }
  n = at;
  return a;
}

template <typename T>
__device__ __forceinline__ float element(const uint32_t (&w)[4], int j) {      // element j of 16 bytes
  if constexpr (sizeof(T) == 2)
    return __uint_as_float((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
  else
    return __uint_as_float(w[j]);
}

// W waves a row (a workgroup). mis: elements between the 16-byte boundary at or below the row and the row.
template <typename T>
__global__ __launch_bounds__(1024) void stream_kernel(const T* logits, int64_t stride, int V, int K, T* values, int64_t* tokens) {
  extern __shared__ uint64_t keys[];       // kBuf a wave
  __shared__ int held[16];
  constexpr int E = 16 / sizeof(T);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, W = blockDim.x >> 6;
  const T* row = logits + (int64_t)blockIdx.x * stride;
  const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
  const uint4* base = reinterpret_cast<const uint4*>(row - mis);
  const int pieces = (mis + V + E - 1) / E;
  const int tiles = (pieces + 63) / 64, per = (tiles + W - 1) / W;
  const int t0 = min(wave * per, tiles), t1 = min(t0 + per, tiles);
  uint64_t* buf = keys + wave * kBuf;
  int n = 0;
  bool full = false;                       // K elements held: only larger values matter (a later token loses a tie)
  float least = 0.f;
  for (int t = t0; t < t1; t += kLoads) {
    uint4 q[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int p = (t + u) * 64 + lane;
      q[u] = make_uint4(0u, 0u, 0u, 0u);
      if (t + u < t1 && p < pieces) q[u] = base[p];
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      if (t + u >= t1) break;              // uniform
      const uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
      const int i0 = ((t + u) * 64 + lane) * E - mis;
      const bool edge = t + u == 0 || t + u == tiles - 1;      // uniform: the tile may hold elements of others
      float x[E];
      uint64_t pass[E];
      uint64_t any = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        x[j] = element<T>(w, j);
        pass[j] = __ballot(!(x[j] <= least) || !full);
        if (edge) pass[j] &= __ballot(i0 + j >= 0 && i0 + j < V);
        any |= pass[j];
      }
      if (any == 0) continue;              // uniform
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if (pass[j] == 0) continue;        // uniform
        if ((pass[j] >> lane) & 1)
          buf[n + below_me(pass[j])] = ((uint64_t)image_of(x[j]) << 32) | (uint32_t) ~(i0 + j);
        n += __popcll(pass[j]);
      }
      if (n > kBuf - 64 * E) {             // uniform: the next tile might not fit (kBuf - 64 E >= kMaxK + kSlack)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        const uint32_t im = cut(buf, n, K, kSlack, lane);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        full = true;
        least = im == 0xffffffffu ? __builtin_nanf("") : value_of(im);
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  if (n > K) cut(buf, n, K, 0, lane);
  if (lane == 0) held[wave] = n;
  __syncthreads();

  // all waves' lists side by side, padded with zeros (below every key) to a power of two, sorted falling
  int Kp = 1;
  while (Kp < K) Kp <<= 1;
  const int S = W * max(Kp, 64);           // 1, 2 or 4 keys a thread
  uint64_t mine[4];
  const int cnt = S / blockDim.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = tid + j * blockDim.x;
    mine[j] = 0ull;
    if (j < cnt) {
      const int w = i / Kp, r = i % Kp;
      if (w < W && r < held[w]) mine[j] = keys[w * kBuf + r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < cnt) keys[tid + j * blockDim.x] = mine[j];
  __syncthreads();
  for (int size = 2; size <= S; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = tid; i < S / 2; i += blockDim.x) {
        const int lo = 2 * i - (i & (step - 1)), up = lo + step;
        const uint64_t x = keys[lo], y = keys[up];
        if ((x < y) == ((lo & size) == 0)) {
          keys[lo] = y;
          keys[up] = x;
        }
      }
      __syncthreads();
    }
  for (int j = tid; j < K; j += blockDim.x) {
    const int i = (int)~(uint32_t)keys[j];
    values[(int64_t)blockIdx.x * K + j] = row[i];
    tokens[(int64_t)blockIdx.x * K + j] = i;
  }
}

// ---- rows held in registers -----------------------------------------------------------------------------------------
constexpr int kCap = 4096;                 // keys in LDS

// The row's whole aligned 16-byte pieces, thread t those of t, t + nt, ... (nt threads, NP pieces each at most), and what
// stands before the first and behind the last of them, up to 2 (E - 1) logits, one each with the first threads.
template <typename T, int NP>
__global__ __launch_bounds__(1024, sizeof(T) == 2 ? 8 : 4) void held_kernel(const T* logits, int64_t stride, int V, int K,
                                                                            T* values, int64_t* tokens) {
  constexpr int E = 16 / sizeof(T);
  __shared__ uint64_t keys[kCap];
  __shared__ uint32_t images[1024], firsts[1024];
  __shared__ uint32_t bound[2];            // image; least complement of a token at that image
  __shared__ int count, part[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nt = blockDim.x;
  const T* row = logits + (int64_t)blockIdx.x * stride;
  const int head = min((int)((16u - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / (int)sizeof(T), V);
  const char* base = reinterpret_cast<const char*>(row + head);
  const int pieces = (V - head) / E, tail = V - head - pieces * E;
  auto piece = [&](int p) { return *reinterpret_cast<const uint4*>(base + (uint32_t)p * 16u); };
  const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;            // -inf
  uint32_t w[NP][4];
#pragma unroll
  for (int u = 0; u < NP; ++u) {
    uint4 q = make_uint4(none, none, none, none);
    if (u * nt + tid < pieces) q = piece(u * nt + tid);
    w[u][0] = q.x;
    w[u][1] = q.y;
    w[u][2] = q.z;
    w[u][3] = q.w;
  }
  const int extra = tid < head ? tid : tid < head + tail ? V - tail + (tid - head) : -1;   // token of the single logit
  const float ex = extra >= 0 ? Elem<T>::load(row + extra) : -INFINITY;
  auto token_of = [&](int u, int j) { return head + (u * nt + tid) * E + j; };
  auto key = [](float x, int token) { return ((uint64_t)image_of(x) << 32) | ~(uint32_t)token; };
  if (tid == 0) count = 0;
  // (w opaque from one use to the next: the unpacked values of one are not worth the registers until the other)
  auto opaque = [&]() {
#pragma unroll
    for (int u = 0; u < NP; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(w[u][j]));
  };
  const int held = max(0, (pieces - tid + nt - 1) / nt);       // pieces of this thread
  // the thread's keys from memory, for the slow paths
  auto each = [&](auto&& f) {
    if (extra >= 0) f(key(ex, extra));
#pragma unroll 1
    for (int u = 0; u < held; ++u) {
      const uint4 q = piece(u * nt + tid);
      const uint32_t v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < E; ++j) f(key(element<T>(v, j), token_of(u, j)));
    }
  };

  // the thread's largest value; a NaN is above it
  opaque();
  float most = ex;
  bool nan = ex != ex;
#pragma unroll
  for (int u = 0; u < NP; ++u)
#pragma unroll
    for (int j = 0; j < E; j += 2) {
      const float x = element<T>(w[u], j), y = element<T>(w[u], j + 1);
      most = fmaxf(fmaxf(x, y), most);
      nan |= __builtin_isunordered(x, y);
    }
  const bool some = held > 0 || extra >= 0;                    // (a thread that holds nothing has no part in this)
  const uint32_t mine = !some ? 0u : nan ? 0xffffffffu : image_of(most);
  images[tid] = mine;
  for (int i = nt + tid; i < 1024; i += nt) images[i] = 0u;
  __syncthreads();

  if (wave == 0) {
    uint32_t im[16];
    uint32_t a = 0xffffffffu, b = 0u;
    int at_least = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      im[j] = images[j * 64 + lane];
      a = min(a, im[j] - 1u);                                  // (0, nothing, becomes the largest)
      b = max(b, im[j]);
      at_least += __popcll(__ballot(im[j] != 0u));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      a = min(a, (uint32_t)__shfl_xor((int)a, o));
      b = max(b, (uint32_t)__shfl_xor((int)b, o));
    }
    a = __builtin_amdgcn_readfirstlane(a) + 1u;
    b = __builtin_amdgcn_readfirstlane(b);
    if (at_least < K) {                                        // every element may be one of the K
      a = 1u;
    } else {
      while (a < b && at_least > K + kSlack) {
        const uint32_t mid = a + ((b - a) >> 1) + ((b - a) & 1u);
        int c = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) c += __popcll(__ballot(im[j] >= mid));
        if (c >= K) {
          a = mid;
          at_least = c;
        } else {
          b = mid - 1u;
        }
      }
    }
    if (lane == 0) {
      bound[0] = a;
      bound[1] = at_least > K + kSlack ? 1u : 0u;              // (1: ties to be cut)
    }
  }
  __syncthreads();
  const uint32_t a = bound[0];
  uint32_t t = 0u;
  if (bound[1]) {                          // uniform: more threads than K + kSlack have their largest value there
    // as composites of value and lowest token: the K-th largest of the threads'
    uint32_t first = 0u;
    if (mine == a)
      each([&](uint64_t k) {
        if ((uint32_t)(k >> 32) == a) first = max(first, (uint32_t)k);
      });
    firsts[tid] = first;
    for (int i = nt + tid; i < 1024; i += nt) firsts[i] = 0u;
    __syncthreads();
    if (wave == 0) {
      uint32_t fi[16];
      int above = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        fi[j] = firsts[j * 64 + lane];                         // (0 unless the thread's value is the bound)
        above += __popcll(__ballot(images[j * 64 + lane] > a));
      }
      const int need = K - above;          // >= 1: the bisection ended with fewer than K above a
      uint32_t lo = 0u, hi = 0xffffffffu;
      while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1) + ((hi - lo) & 1u);
        int c = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) c += __popcll(__ballot(fi[j] >= mid));
        if (c >= need) lo = mid; else hi = mid - 1u;
      }
      if (lane == 0) bound[1] = lo;
    }
    __syncthreads();
    t = bound[1];
  }

  // the keys at or above the bound
  const uint64_t least = ((uint64_t)a << 32) | t;
  const float value = a == 0xffffffffu || a == 1u ? -INFINITY : value_of(a);   // (a key below `least` may pass this one)
  auto append = [&](uint64_t k) {
    if (k >= least) {
      const int at = atomicAdd(&count, 1);
      if (at < kCap) keys[at] = k;
    }
  };
  opaque();
  uint32_t which = 0u;                     // pieces with a value that passes in some lane
#pragma unroll
  for (int u = 0; u < NP; ++u) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < E; ++j) any |= !(element<T>(w[u], j) < value);
    if (__ballot(any && u < held)) which |= 1u << u;
  }
  while (which) {                          // uniform
    const int u = __builtin_ctz(which);
    which &= which - 1u;
    uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (i == u) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = w[i][j];
      }
    if (u < held) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float x = element<T>(v, j);
        if (!(x < value)) append(key(x, token_of(u, j)));
      }
    }
  }
  if (extra >= 0) append(key(ex, extra));
  __syncthreads();
  int n = count;
  if (n > kCap) {                          // uniform: the exact K-th largest key of the whole row
    uint64_t lo = least, hi = ~0ull;
    while (lo < hi) {
      const uint64_t mid = lo + ((hi - lo) >> 1) + ((hi - lo) & 1u);
      int c = 0;
      each([&](uint64_t k) { c += k >= mid; });
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
      __syncthreads();
      if (lane == 0) part[wave] = c;
      __syncthreads();
      c = 0;
      for (int v = 0; v < nt / 64; ++v) c += part[v];
      if (c >= K) lo = mid; else hi = mid - 1ull;
    }
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
    each([&](uint64_t k) {
      if (k >= lo) keys[atomicAdd(&count, 1)] = k;             // K of them: keys differ
    });
    __syncthreads();
    n = K;
  }
  for (int i = tid; i < n; i += nt) {
    const uint64_t k = keys[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += keys[j] > k;
    if (rank < K) {
      const int at = (int)~(uint32_t)k;
      values[(int64_t)blockIdx.x * K + rank] = row[at];
      tokens[(int64_t)blockIdx.x * K + rank] = at;
    }
  }
}

// waves a row: 4096 waves (16 a CU) over the rows, one to sixteen
int waves_of(int64_t rows) {
  int w = 1;
  while (w < 16 && rows * w * 2 <= 4096) w *= 2;
  return w;
}

template <typename T>
int launch(const void* logits, int64_t stride, int64_t rows, int V, int K, void* values, int64_t* tokens, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const T* x = (const T*)logits;
  T* out = (T*)values;
  const int pieces = (V + E - 1) / E;                          // at least those of a row at any alignment
  const dim3 grid((unsigned)rows);
  if (V <= 65536) {
    // threads: a piece each, up to 1024
    const dim3 block((unsigned)(pieces >= 1024 ? 1024 : (pieces + 63) / 64 * 64));
    const int np = (pieces + (int)block.x - 1) / (int)block.x;
    if (np <= 1) held_kernel<T, 1><<<grid, block, 0, s>>>(x, stride, V, K, out, tokens);
    else if (np <= 2) held_kernel<T, 2><<<grid, block, 0, s>>>(x, stride, V, K, out, tokens);
    else if (np <= 4) held_kernel<T, 4><<<grid, block, 0, s>>>(x, stride, V, K, out, tokens);
    else if (np <= 8) held_kernel<T, 8><<<grid, block, 0, s>>>(x, stride, V, K, out, tokens);
    else if constexpr (sizeof(T) == 4) held_kernel<T, 16><<<grid, block, 0, s>>>(x, stride, V, K, out, tokens);
    return dh_check_launch("dh_top_logits");
  }
  const int W = waves_of(rows);
  const size_t lds = (size_t)W * kBuf * sizeof(uint64_t);
  if (lds > 65536 - 256) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&stream_kernel<T>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return dh_fail(DH_ERR_LAUNCH_FAILED, "dh_top_logits: %zu bytes of LDS: %s", lds, hipGetErrorString(e));
  }
  stream_kernel<T><<<grid, dim3(64 * W), lds, s>>>(x, stride, V, K, out, tokens);
  return dh_check_launch("dh_top_logits");
}

}  // namespace

extern "C" int dh_top_logits(int dtype, const void* logits, int64_t row_stride, int64_t rows, int V, int K, void* values,
                             int64_t* tokens, void* stream) {
  const char* who = "dh_top_logits";
  DH_REQUIRE(dtype == DH_F32 || dtype == DH_BF16, DH_ERR_UNSUPPORTED_DTYPE, "%s: dtype %d", who, dtype);
  DH_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 22) && V >= 1 && V <= (1 << 24), DH_ERR_UNSUPPORTED_SHAPE,
             "%s: rows=%lld V=%d", who, (long long)rows, V);
  DH_REQUIRE(K >= 1 && K <= kMaxK && K <= V, DH_ERR_UNSUPPORTED_SHAPE, "%s: K=%d must be in [1, min(%d, V=%d)]", who, K,
             kMaxK, V);
  if (rows == 0) return 0;
  DH_REQUIRE(logits && values && tokens, DH_ERR_INVALID_ARG, "%s: null pointer argument", who);
  const size_t size = dtype == DH_BF16 ? 2 : 4;
  DH_REQUIRE((uintptr_t)logits % size == 0 && (uintptr_t)values % size == 0 && (uintptr_t)tokens % 8 == 0, DH_ERR_INVALID_ARG,
             "%s: operands not aligned to their elements", who);
  hipStream_t s = (hipStream_t)stream;
  return dtype == DH_BF16 ? launch<bf16_t>(logits, row_stride, rows, V, K, values, tokens, s)
                          : launch<float>(logits, row_stride, rows, V, K, values, tokens, s);
}
