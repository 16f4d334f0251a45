// The K largest logits of every row and their tokens, for gfx950: a teacher's targets for distillation.
//   values[r, 0 .. K) = the K largest of logits[r], falling;  tokens[r, j] = where they stand, the lower token first where
//   values are equal (0.0 and -0.0 are), NaN above every number.
//
// A value and its token make one 64-bit key, different for every element: an order-preserving 32-bit image of the value
// above the complement of the token. The K largest keys are the answer, with no case for ties.
//
// One pass over the row (V bytes of logits read once; compares only, so the read bounds it): a wave streams its part of the
// row in 16-byte loads and keeps, in LDS, every element above the value of the K-th best so far. When the buffer could
// overflow within the next tile it is cut back to its K largest and that value rises: for values in no order, about
// K ln(V / K) elements enter after the first tiles, and the buffer is cut two to four times. Rows in ascending order cut it
// after every tile, slower but the same answer. Several waves share a row where the rows are too few to fill the card; their
// lists are sorted together.

#include "dh_common.h"

namespace {

constexpr int kBuf = 1024;                 // keys a wave holds: more than kMaxK plus a tile
constexpr int kMaxK = 256;
constexpr int kPer = kBuf / 64;
constexpr int kLoads = 4;                  // 16-byte loads in flight a lane

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

// Cuts the wave's keys buf[0, n) to their K largest (n > K), in no order; returns the smallest of them. The image of the
// K-th largest by bisection, then, among the keys of that image, the complement of its token.
__device__ __forceinline__ uint64_t cut(uint64_t* buf, int n, int K, int lane) {
  uint32_t hi[kPer], lo[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const uint64_t k = j * 64 + lane < n ? buf[j * 64 + lane] : 0ull;
    hi[j] = (uint32_t)(k >> 32);
    lo[j] = (uint32_t)k;
  }
  uint32_t a = 1u, b = 0xffffffffu;                            // the largest image v with count(hi >= v) >= K
  int at_least = n;                                            // count(hi >= a)
  while (a < b && at_least != K) {
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
  if (at_least != K) {                                         // ties at a: the lowest tokens of them
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
  uint64_t least = ~0ull;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const bool keep = hi[j] != 0u && (hi[j] > a || (hi[j] == a && lo[j] >= t));
    const uint64_t mask = __ballot(keep);
    const uint64_t k = ((uint64_t)hi[j] << 32) | lo[j];
    if (keep) {
      buf[at + below_me(mask)] = k;
      least = k < least ? k : least;
    }
    at += __popcll(mask);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor((unsigned long long)least, o);
    least = u < least ? u : least;
  }
  return least;
}

// W waves a row (a workgroup). mis: elements between the 16-byte boundary at or below the row and the row.
template <typename T>
__global__ __launch_bounds__(1024) void top_kernel(const T* logits, int64_t stride, int V, int K, T* values, int64_t* tokens) {
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
  bool full = false;                       // K elements seen: only larger values matter (a later token loses a tie)
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
      float x[E];
      uint64_t pass[E];
      uint64_t any = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if constexpr (sizeof(T) == 2)
          x[j] = __uint_as_float((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
        else
          x[j] = __uint_as_float(w[j]);
        const bool in = i0 + j >= 0 && i0 + j < V;
        pass[j] = __ballot(in && (!full || !(x[j] <= least)));
        any |= pass[j];
      }
      if (any == 0) continue;              // uniform
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if ((pass[j] >> lane) & 1)
          buf[n + below_me(pass[j])] = ((uint64_t)image_of(x[j]) << 32) | (uint32_t) ~(i0 + j);
        n += __popcll(pass[j]);
      }
      if (n > kBuf - 64 * E) {             // uniform: the next tile might not fit (kBuf - 64 E >= K)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        const uint64_t k = cut(buf, n, K, lane);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        n = K;
        full = true;
        const uint32_t im = (uint32_t)(k >> 32);
        least = im == 0xffffffffu ? __builtin_nanf("") : value_of(im);
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  if (n > K) {
    cut(buf, n, K, lane);
    n = K;
  }
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

// waves a row: 4096 waves (16 a CU) over the rows, one to sixteen
int waves_of(int64_t rows) {
  int w = 1;
  while (w < 16 && rows * w * 2 <= 4096) w *= 2;
  return w;
}

template <typename T>
int launch(const void* logits, int64_t stride, int64_t rows, int V, int K, void* values, int64_t* tokens, hipStream_t s) {
  const int W = waves_of(rows);
  const size_t lds = (size_t)W * kBuf * sizeof(uint64_t);
  if (lds > 65536 - 256) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&top_kernel<T>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return dh_fail(DH_ERR_LAUNCH_FAILED, "dh_top_logits: %zu bytes of LDS: %s", lds, hipGetErrorString(e));
  }
  top_kernel<T><<<dim3((unsigned)rows), dim3(64 * W), lds, s>>>((const T*)logits, stride, V, K, (T*)values, tokens);
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
