// The K largest logits of every row and their tokens, for gfx950: a teacher's targets for distillation.
//   values[r, 0 .. K) = the K largest of logits[r], falling;  tokens[r, j] = where they stand, the lower token first where
//   values are equal (0.0 and -0.0 are), NaN above every number.
//
// A value and its token make one 64-bit key, different for every element: an order-preserving 32-bit image of the value
// above the complement of the token. The K largest keys are the answer, with no case for ties.
//
// One workgroup a row, of up to 1024 threads, which read the row once and go back to a few per cent of it:
//   - each thread keeps the largest of its values (a half instruction a value, and another half for NaN);
//   - the K-th largest of those, or a value slightly below it, is a lower bound of the K-th largest logit: bisection over their
//     images by one wave, ended once K to K + kSlack threads are at least there;
//   - those threads' 16-byte pieces are read again, by the whole workgroup, and the logits at the bound or above (K and a few
//     tens more: a thread rarely holds two) go to LDS as keys;
//   - a key's rank is the number of larger keys; ranks below K write their value and token.
// Ties at the bound (masked vocabularies, constant rows) take the lower tokens first. Rows whose large values all stand where
// few threads read them, more than LDS holds, are bisected as a whole, slowly. The first pass is bound by its read, and its
// two workgroups a CU fill each other's other steps. (Rows kept in registers instead of read again: 130 us in place of
// TOPUS at 4096 x 50257 bf16, the search for the large values in 64 registers a thread being most of it; a wave a row with a
// running bound: 219 us.)

#include "dh_common.h"

namespace {

constexpr int kMaxK = 256;
constexpr int kSlack = 32;                 // threads more than K that end the bisection
constexpr int kCap = 9 * kMaxK;            // keys in LDS: ties leave up to E K of them, and K above
constexpr int kMany = 512;                 // rows from which a row gets 512 threads
constexpr int kU = 8;                      // 16-byte loads in flight a thread

__device__ __forceinline__ uint32_t image_of(float x) {        // a < b  <=>  image(a) < image(b); NaN above all
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);                // -0.0 as 0.0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, int token) { return ((uint64_t)image_of(x) << 32) | ~(uint32_t)token; }

template <typename T>
__device__ __forceinline__ float element(const uint32_t (&w)[4], int j) {      // element j of 16 bytes
  if constexpr (sizeof(T) == 2)
    return __uint_as_float((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
  else
    return __uint_as_float(w[j]);
}

// The largest v in [lo, hi] with count(v) >= need, given count(lo) >= need; ends early once the count is at most `enough`.
// got: the count at the result. All uniform in the wave.
template <typename V, typename F>
__device__ __forceinline__ V bisect(V lo, V hi, int need, int enough, int& got, F&& count) {
  while (lo < hi && got > enough) {
    const V mid = lo + ((hi - lo) >> 1) + ((hi - lo) & 1);
    const int c = count(mid);
    if (c >= need) {
      lo = mid;
      got = c;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// The row's whole aligned 16-byte pieces, thread t those of t, t + nt, ... (nt threads), and what stands before the first and
// behind the last of them, up to 2 (E - 1) logits, one each with the first threads.
template <typename T, int NT>
__global__ __launch_bounds__(NT, 8) void top_kernel(const T* logits, int64_t stride, int V, int K, T* values,
                                                      int64_t* tokens) {
  constexpr int E = 16 / sizeof(T);
  __shared__ uint64_t keys[kCap];
  __shared__ uint32_t images[NT], firsts[NT];
  __shared__ uint16_t list[NT];            // the threads at or above the bound
  __shared__ uint32_t bound[2];            // image; least complement of a token at that image
  __shared__ int count, listed, part[NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nt = blockDim.x;
  const T* row = logits + (int64_t)blockIdx.x * stride;
  const int head = min((int)((16u - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / (int)sizeof(T), V);
  const char* base = reinterpret_cast<const char*>(row + head);
  const int pieces = (V - head) / E, tail = V - head - pieces * E;
  auto piece = [&](int p, uint32_t (&w)[4]) {
    const uint4 q = *reinterpret_cast<const uint4*>(base + (uint32_t)p * 16u);
    w[0] = q.x;
    w[1] = q.y;
    w[2] = q.z;
    w[3] = q.w;
  };
  const int extra = tid < head ? tid : tid < head + tail ? V - tail + (tid - head) : -1;   // token of the single logit
  const float ex = extra >= 0 ? Elem<T>::load(row + extra) : -INFINITY;
  // all keys of this thread, from memory, for the slow paths
  auto each = [&](auto&& f) {
    if (extra >= 0) f(key_of(ex, extra));
#pragma unroll 1
    for (int p = tid; p < pieces; p += nt) {
      uint32_t w[4];
      piece(p, w);
#pragma unroll
      for (int j = 0; j < E; ++j) f(key_of(element<T>(w, j), head + p * E + j));
    }
  };
  if (tid == 0) count = listed = 0;

  // the thread's largest value; a NaN is above it
  float most = ex;
  bool nan = ex != ex;
  for (int p = tid; p < pieces; p += nt * kU) {
    uint32_t w[kU][4];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int k = p + u * nt;
      piece(k < pieces ? k : p, w[u]);     // (behind the row: the first piece again, which changes no maximum)
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int j = 0; j < E; j += 2) {
        const float x = element<T>(w[u], j), y = element<T>(w[u], j + 1);
        most = fmaxf(fmaxf(x, y), most);
        nan |= __builtin_isunordered(x, y);
      }
  }
  const bool some = tid < pieces || extra >= 0;                // (a thread that holds nothing has no part in this)
  const uint32_t mine = !some ? 0u : nan ? 0xffffffffu : image_of(most);
  images[tid] = mine;
  for (int i = nt + tid; i < NT; i += nt) images[i] = 0u;
  __syncthreads();

  if (wave == 0) {
    uint32_t im[NT / 64];
    uint32_t a = 0xffffffffu, b = 0u;
    int got = 0;
#pragma unroll
    for (int j = 0; j < NT / 64; ++j) {
      im[j] = images[j * 64 + lane];
      a = min(a, im[j] - 1u);                                  // (0, nothing, becomes the largest)
      b = max(b, im[j]);
      got += __popcll(__ballot(im[j] != 0u));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      a = min(a, (uint32_t)__shfl_xor((int)a, o));
      b = max(b, (uint32_t)__shfl_xor((int)b, o));
    }
    a = __builtin_amdgcn_readfirstlane(a) + 1u;
    b = __builtin_amdgcn_readfirstlane(b);
    if (got < K) {
      a = 1u;                                                  // every element may be one of the K
    } else {
      a = bisect(a, b, K, K + kSlack, got, [&](uint32_t v) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < NT / 64; ++j) c += __popcll(__ballot(im[j] >= v));
        return c;
      });
    }
    if (lane == 0) {
      bound[0] = a;
      bound[1] = got > K + kSlack ? 1u : 0u;                   // (1: ties to be cut)
    }
  }
  __syncthreads();
  const uint32_t a = bound[0];
  uint32_t t = 0u, first = 0u;
  if (bound[1]) {                          // uniform: more threads than K + kSlack have their largest value there
    // as composites of value and lowest token: the K-th largest of the threads'
    if (mine == a)
      each([&](uint64_t k) {
        if ((uint32_t)(k >> 32) == a) first = max(first, (uint32_t)k);
      });
    firsts[tid] = first;
    for (int i = nt + tid; i < NT; i += nt) firsts[i] = 0u;
    __syncthreads();
    if (wave == 0) {
      uint32_t fi[NT / 64];
      int above = 0, got = NT;
#pragma unroll
      for (int j = 0; j < NT / 64; ++j) {
        fi[j] = firsts[j * 64 + lane];                         // (0 unless the thread's value is the bound)
        above += __popcll(__ballot(images[j * 64 + lane] > a));
      }
      // (fewer than K are above a: the bisection ended there)
      const uint32_t lo = bisect(0u, 0xffffffffu, K - above, K - above, got, [&](uint32_t v) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < NT / 64; ++j) c += __popcll(__ballot(fi[j] >= v));
        return c;
      });
      if (lane == 0) bound[1] = lo;
    }
    __syncthreads();
    t = bound[1];
  }
  const uint64_t least = ((uint64_t)a << 32) | t;
  if (((uint64_t)mine << 32 | first) >= least) list[atomicAdd(&listed, 1)] = (uint16_t)tid;
  auto append = [&](uint64_t k) {
    if (k >= least) {
      const int at = atomicAdd(&count, 1);
      if (at < kCap) keys[at] = k;
    }
  };
  if (extra >= 0) append(key_of(ex, extra));
  __syncthreads();

  // the pieces of the listed threads: 2^lg threads a turn of the list, the others on their further pieces
  int lg = 0;
  while ((1 << lg) < min(listed, nt)) ++lg;
  const float value = a == 0xffffffffu || a == 1u ? -INFINITY   // (a key below `least` may pass this one)
                                                  : __uint_as_float((a & 0x80000000u) ? (a & 0x7fffffffu) : ~a);
  const int step = max(nt >> lg, 1);       // (threads past step << lg, of which there are too few for a turn, stay out)
  if ((tid >> lg) < step && (tid & ((1 << lg) - 1)) < listed) {
    const int who = list[tid & ((1 << lg) - 1)];
    for (int p = (tid >> lg) * nt + who; p < pieces; p += step * nt) {
      uint32_t w[4];
      piece(p, w);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float x = element<T>(w, j);
        if (!(x < value)) append(key_of(x, head + p * E + j));
      }
    }
  }
  __syncthreads();
  int n = count;
  if (n > kCap) {                          // uniform: the exact K-th largest key of the whole row
    int got = n;
    const uint64_t lo = bisect(least, (uint64_t)~0ull, K, K, got, [&](uint64_t v) {
      int c = 0;
      each([&](uint64_t k) { c += k >= v; });
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
      __syncthreads();
      if (lane == 0) part[wave] = c;
      __syncthreads();
      c = 0;
      for (int i = 0; i < nt / 64; ++i) c += part[i];
      return c;
    });
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

template <typename T>
int launch(const void* logits, int64_t stride, int64_t rows, int V, int K, void* values, int64_t* tokens, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const int need = ((V + E - 1) / E + 63) / 64 * 64;           // a piece a thread, or more
  const dim3 grid((unsigned)rows);
  if (rows < kMany)
    top_kernel<T, 1024><<<grid, dim3((unsigned)(need < 1024 ? need : 1024)), 0, s>>>((const T*)logits, stride, V, K,
                                                                                    (T*)values, tokens);
  else
    top_kernel<T, 512><<<grid, dim3((unsigned)(need < 512 ? need : 512)), 0, s>>>((const T*)logits, stride, V, K, (T*)values,
                                                                                  tokens);
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
