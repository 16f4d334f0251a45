// The K largest logits of every row and their tokens, for gfx950: a teacher's targets for distillation.
//   values[r, 0 .. K) = the K largest of logits[r], falling;  tokens[r, j] = where they stand, the lower token first where
//   values are equal (0.0 and -0.0 are), NaN above every number.
//
// A value and its token make one 64-bit key, different for every element: an order-preserving 32-bit image of the value
// above the complement of the token. The K largest keys are the answer, with no case for ties; below the token a bit says
// which zero it was, so that a key has its value whole (NaN apart).
//
// One workgroup a row, which reads the row once and goes back to a part of it, about (K + kSlack) of its groups (a fifth of a
// long row at K 64 with 512 groups, half of it at K 256):
//   - the largest value of every group of logits, one group a thread: its own 16-byte pieces or, in long rows, one 128-byte
//     line of each eight pieces that it read with its seven neighbours (whole lines, so that going back costs no more than
//     the groups themselves hold);
//   - the K-th largest of those, or a value slightly below it, is a lower bound of the K-th largest logit: bisection over their
//     images by one wave, ended once K to K + kSlack groups are at least there;
//   - those groups are read again, by the whole workgroup, and the logits at the bound or above (K and a few tens more: a
//     group rarely holds two) go to LDS as keys;
//   - a key's rank is the number of larger keys; ranks below K write their value and token.
// Ties at the bound take the lower tokens first. Where more keys pass than LDS holds (masked vocabularies and constant rows,
// whose ties fill whole lines; large values in few groups), the K-th largest of the keys that it does hold is the next bound
// and the row is read again, nearly always once: 1024 x 50257, masked to 40 tokens, bf16 K 64 211 us where bisecting the row
// took 3916, fp32 K 256 420 where it took 6512, beside 27 and 56 of ordinary rows. Rows with a NaN are bisected, slowly.
// The first pass is bound by its read. 4096 x 50257 bf16, K 64: 79 us, 5.2 TB/s. (Rows kept in registers instead of read
// again: 130 us; a wave a row with a running bound: 219 us; groups of pieces from eight lines each, which going back reads
// whole: 106 us.)

#include <type_traits>

#include "dh_common.h"

namespace {

constexpr int kMaxK = 256;
constexpr int kSlack = 32;                 // threads more than K that end the bisection
constexpr int kCap = 9 * kMaxK;            // keys in LDS: where groups are pieces, ties leave up to E K of them, and K above
constexpr int kTurns = 4;                  // reads of a row whose keys do not fit, each by a higher bound, before the bisection
// Rows from which a row of fewer than kLong pieces gets 512 threads in place of 1024, so that four rows share a CU (K 64, in a
// graph; bf16, V 50257: 85 against 95 us at 4096 rows, 29 against 33 at 1024, 19 against 20 at 512; V 8000, 4096 rows: 38
// against 73; 16000 pieces, 1024 rows: 56 against 50; fp32, V 50257, 1024 rows: 48 against 43).
constexpr int kMany = 512, kLong = 8192;
constexpr int kFew = 128;                  // keys up to which a thread ranks one (K 64: 95 keys or so, 256: 330)
constexpr int kU = 4;                      // 16-byte loads in flight a thread
// Groups are lines where there are kLines times as many lines as the bisection may leave, or one for every thread: with few more
// groups than that the bound falls to the lowest of their maxima, and the whole row is above it.
// Lines and, by this rule, pieces, 2048 rows of bf16, K 256, us: 256 lines 614 and 53, 320 lines 94 and 55, 448 lines 61 and 58;
// K 160, 256 lines 42 and 33, 320 lines 40 and 35.
constexpr int kLines = 2;

__device__ __forceinline__ uint32_t image_of(float x) {        // a < b  <=>  image(a) < image(b); NaN above all
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);                // -0.0 as 0.0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t image) {
  return __uint_as_float((image & 0x80000000u) ? (image & 0x7fffffffu) : ~image);
}
__device__ __forceinline__ uint64_t key_of(float x, int token) {               // token < 2^24
  return ((uint64_t)image_of(x) << 32) | (~(uint32_t)token << 8) | (__float_as_uint(x) == 0x80000000u ? 1u : 0u);
}
__device__ __forceinline__ int token_of(uint64_t key) { return (int)(~(uint32_t)key >> 8); }

template <typename T>
__device__ __forceinline__ float element(const uint32_t (&w)[4], int j) {      // element j of 16 bytes
  if constexpr (sizeof(T) == 2)
    return __uint_as_float((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
  else
    return __uint_as_float(w[j]);
}

// The larger one, NaN if one is: v_maximum3_f32 takes a pair more, and asks for no canonical input.
__device__ __forceinline__ float larger(float x, float y) { return __builtin_elementwise_maximum(x, y); }

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

// The row's whole aligned 16-byte pieces, thread t reads those of t, t + nt, ... (nt threads), and what stands before the first
// and behind the last of them, up to 2 (E - 1) logits, one each with the first threads' groups. Groups of thread t: the pieces
// it reads, or (lines) of each stretch of 8 nt pieces the eight from line(t) nt + 8 floor(t / 8).
template <typename T, int NT>
__global__ __launch_bounds__(NT, 8) void top_kernel(const T* logits, int64_t stride, int V, int K, T* values,
                                                      int64_t* tokens) {
  constexpr int E = 16 / sizeof(T);
  __shared__ uint64_t keys[kCap];
  __shared__ uint32_t images[NT], firsts[NT];
  __shared__ uint16_t list[NT];            // the threads at or above the bound
  __shared__ uint32_t bound[2];            // image; least complement of a token at that image
  __shared__ int count, listed, nans, part[NT / 64];
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
  const bool lines = pieces >= 4 * nt && (pieces >= 8 * nt || pieces / 8 >= kLines * (K + kSlack));
  // which of a stretch's eight pieces is on the line of thread t, as the exchange below leaves them
  auto line = [](int t) { return (t & 1) << 2 | (t & 4) >> 1 | (t & 2) >> 1; };
  const int first_piece = lines ? line(tid) * nt + (tid & ~7) : tid;           // of the thread's group
  // all keys of the thread's group, for the slow paths
  auto each = [&](auto&& f) {
    if (extra >= 0) f(key_of(ex, extra));
#pragma unroll 1
    for (int p = first_piece; p < pieces; p += lines ? 8 * nt : nt)
#pragma unroll 1
      for (int i = 0; i < (lines ? min(8, pieces - p) : 1); ++i) {
        uint32_t w[4];
        piece(p + i, w);
#pragma unroll
        for (int j = 0; j < E; ++j) f(key_of(element<T>(w, j), head + (p + i) * E + j));
      }
  };
  if (tid == 0) count = listed = nans = 0;
  for (int i = nt + tid; i < NT; i += nt) images[i] = firsts[i] = 0u;

  // the group's largest value (NaN where it has one: the maxima propagate it)
  float most = ex;
  bool odd = false;                        // of a stretch's eight pieces: the first or the last four
  auto four = [&](int p, auto whole) {     // whole: none of the wave's four pieces is behind the last
    uint32_t w[kU][4];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      constexpr uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;    // -inf
      if constexpr (whole) {
        piece(p + u * nt, w[u]);
      } else {
        w[u][0] = w[u][1] = w[u][2] = w[u][3] = none;
        if (p + u * nt < pieces) piece(p + u * nt, w[u]);
      }
    }
    float top[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      top[u] = larger(element<T>(w[u], 0), element<T>(w[u], 1));
#pragma unroll
      for (int j = 2; j < E; j += 2) top[u] = larger(larger(element<T>(w[u], j), element<T>(w[u], j + 1)), top[u]);
    }
    if (lines) {                           // uniform: each lane gives away what it is not to keep, four values in three steps
      const bool b2 = lane & 4, b1 = lane & 2;
      const float x = larger(b2 ? top[2] : top[0], dpp_move<0x141, 0xf>(b2 ? top[0] : top[2]));    // row_half_mirror
      const float y = larger(b2 ? top[3] : top[1], dpp_move<0x141, 0xf>(b2 ? top[1] : top[3]));
      float z = larger(b1 ? y : x, dpp_move<0x4e, 0xf>(b1 ? x : y));           // quad_perm(2,3,0,1)
      z = larger(z, dpp_move<0xb1, 0xf>(z));                                   // quad_perm(1,0,3,2)
      if ((bool)(lane & 1) == odd) most = larger(most, z);
    } else {
      most = larger(larger(larger(top[0], top[1]), larger(top[2], top[3])), most);
    }
    odd = !odd;
  };
  static_assert(kU == 4, "");
  int at = tid;                            // (whole waves stay in the loops: the lanes exchange above)
  for (; at - lane + 63 + (kU - 1) * nt < pieces; at += nt * kU) four(at, std::true_type{});
  for (; at - lane < pieces; at += nt * kU) four(at, std::false_type{});
  const bool nan = most != most;
  const bool some = extra >= 0 || first_piece < pieces;        // (a thread whose group holds nothing has no part in this)
  const uint32_t mine = some ? image_of(most) : 0u;
  images[tid] = mine;
  firsts[tid] = 0u;
  if (nan) nans = 1;
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

  // the listed groups, eight threads each
  const float value = a == 1u ? -INFINITY : value_of(a);
  if (!nans) {
    constexpr int R = 4;                   // groups in flight
    const int eighth = nt >> 3, stretch = 8 * nt, heard = listed;
    // pairs of a group and a stretch (eight pieces of the group, one of them here), group by group in each stretch
    int i = tid >> 3, begin = 0;
    auto settle = [&] {
      while (i >= heard && begin < pieces) {
        i -= heard;
        begin += stretch;
      }
    };
    settle();
    while (__any(begin < pieces)) {        // (a wave's lanes leave together; nothing below waits for other waves)
      uint32_t w[R][4];
      int at[R];
#pragma unroll
      for (int u = 0; u < R; ++u) {
        at[u] = pieces;
        w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0u;
        if (begin < pieces) {
          const int t = list[i], j = tid & 7;
          at[u] = begin + (lines ? line(t) * nt + (t & ~7) + j : j * nt + t);
          if (at[u] < pieces) piece(at[u], w[u]);
        }
        i += eighth;
        settle();
      }
#pragma unroll
      for (int u = 0; u < R; ++u) {
        if (!__any(at[u] < pieces)) continue;                  // (often one or two of the four are taken)
        uint32_t pass = 0u;                // a bit an element: nearly always one of a wave's turns is enough for all lanes
#pragma unroll
        for (int j = 0; j < E; ++j) pass |= element<T>(w[u], j) >= value ? 1u << j : 0u;
        if (at[u] >= pieces) pass = 0u;
        while (pass) {
          const int j = __builtin_ctz(pass);
          pass &= pass - 1u;
          const int d = sizeof(T) == 2 ? j >> 1 : j;
          const uint32_t two = d & 2 ? (d & 1 ? w[u][3] : w[u][2]) : (d & 1 ? w[u][1] : w[u][0]);
          const float x = __uint_as_float(sizeof(T) == 4 ? two : (j & 1) ? two & 0xffff0000u : two << 16);
          append(key_of(x, head + at[u] * E + j));
        }
      }
    }
  }
  __syncthreads();
  int n = count;
  auto total = [&](int c) {                // over the workgroup
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
    __syncthreads();
    if (lane == 0) part[wave] = c;
    __syncthreads();
    c = 0;
    for (int i = 0; i < nt / 64; ++i) c += part[i];
    return c;
  };
  auto gather = [&](uint64_t lo) {         // the row's keys from lo on, or kCap of them; how many there are
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
    each([&](uint64_t k) {
      if (k < lo) return;
      const int at = atomicAdd(&count, 1);
      if (at < kCap) keys[at] = k;
    });
    __syncthreads();
    return count;
  };
  // more keys than LDS holds: the K-th largest of those that it does is a higher bound
  uint64_t lo = nans ? (uint64_t)1 : least;
  for (int turn = 0; turn < kTurns && n > kCap && !nans; ++turn) {             // uniform
    int got = kCap;
    lo = bisect(lo, (uint64_t)~0ull, K, K, got, [&](uint64_t v) {
      int c = 0;
      for (int i = tid; i < kCap; i += nt) c += keys[i] >= v;
      return total(c);
    });
    n = gather(lo);
  }
  if (n > kCap || nans) {                  // uniform: the exact K-th largest key of the whole row; keys differ
    int got = V;
    lo = bisect(lo, (uint64_t)~0ull, K, K, got, [&](uint64_t v) {
      int c = 0;
      each([&](uint64_t k) { c += k >= v; });
      return total(c);
    });
    n = gather(lo);
  }
  // ranks, eight threads each; four keys a thread where there are many, so that a key read serves four
  auto ranks = [&](auto many) {
    constexpr int R = many ? 4 : 1;
    for (int i = (tid >> 3) * R; i < n; i += (nt >> 3) * R) {
      uint64_t k[R];
      int rank[R];
#pragma unroll
      for (int u = 0; u < R; ++u) {
        k[u] = keys[min(i + u, n - 1)];
        rank[u] = 0;
      }
#pragma unroll 4
      for (int j = tid & 7; j < n; j += 8) {
        const uint64_t other = keys[j];
#pragma unroll
        for (int u = 0; u < R; ++u) rank[u] += other > k[u];
      }
#pragma unroll
      for (int u = 0; u < R; ++u) {
        rank[u] += __shfl_xor(rank[u], 1);
        rank[u] += __shfl_xor(rank[u], 2);
        rank[u] += __shfl_xor(rank[u], 4);
        if (rank[u] < K && i + u < n && (tid & 7) == u) {
          const int token = token_of(k[u]);
          T* out = values + (int64_t)blockIdx.x * K + rank[u];
          if (nans)
            *out = row[token];
          else
            Elem<T>::store(out, (k[u] & 1u) ? -0.0f : value_of((uint32_t)(k[u] >> 32)));
          tokens[(int64_t)blockIdx.x * K + rank[u]] = token;
        }
      }
    }
  };
  if (n > kFew)
    ranks(std::true_type{});
  else
    ranks(std::false_type{});
}

template <typename T>
int launch(const void* logits, int64_t stride, int64_t rows, int V, int K, void* values, int64_t* tokens, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const int pieces = (V + E - 1) / E, need = (pieces + 63) / 64 * 64;          // a piece a thread, or more
  const dim3 grid((unsigned)rows);
  if (rows < kMany || pieces >= kLong)
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
