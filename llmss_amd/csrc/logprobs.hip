// Log-probabilities of tokens: of a given token a row with its rank, and of the row's n likeliest tokens.
//
//   lp(t) = x_t - M - log sum_j exp(x_j - M),  M = max_j x_j;   rank = 1 + #{j: x_j > x_token};   equal logits: the lower token first
//
// Bound by memory: the logits are read once. A workgroup owns a run of a row's tokens in registers and leaves its maximum, its sum
// of exponentials, how many of its tokens are ahead of the given one, and its own n likeliest in order; a second launch joins a row's
// runs. The n likeliest of a run: a number that at least n tokens reach is found from the lanes' own maxima (a binary search over the
// bits of an order-preserving key, by ballots), and the few tokens that reach it are ranked by counting. Keys carry the token behind the
// value, so no two are equal and a run of equal logits makes no list overflow. A NaN counts as no candidate, and makes its row's
// log-probabilities NaN; a row of nothing but -inf has log-probabilities of -inf.
#include "common.h"

#include <type_traits>

namespace {

constexpr int kMostTop = 64;
typedef unsigned long long u64;

// ascending with the value and, among equal values, with falling token; 0 for what is not there, above it for every number (-inf too)
__device__ __forceinline__ u64 key_of(float x, int t) {
  const unsigned u = __float_as_uint(x + 0.f);  // (-0 as 0)
  const unsigned k = x != x ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return k == 0u ? 0ull : (u64)k << 32 | (unsigned)~t;
}
__device__ __forceinline__ float value_of(u64 k) {
  const unsigned u = (unsigned)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

template <typename T>
__device__ __forceinline__ float at(const T* p) {
  if constexpr (sizeof(T) == 2) return bf2f(*p);
  else return *p;
}

// NT threads, PACKS x 8 tokens a thread. Partial results of run c of row b: part[b][c] = (m, s, ahead, -), top[b][c][n] keys.
template <typename T, int NT, int PACKS, bool VEC>
__global__ __launch_bounds__(NT) void logprobs_runs_kernel(const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ tokens, int V,
                                                           int n, float* __restrict__ part, u64* __restrict__ top) {
  constexpr int NW = NT / 64, RUN = NT * PACKS * 8;
  const int b = blockIdx.y, c = blockIdx.x, runs = gridDim.x, lo = c * RUN;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const T* row = logits + (int64_t)b * ld;
  __shared__ float red[NW], reds[NW];
  __shared__ int redn[NW];
  __shared__ u64 low[NW];
  __shared__ int found;
  extern __shared__ __attribute__((aligned(16))) u64 list[];  // at most n threads of a wave reach the number, 8 PACKS keys each
  const int64_t tok = tokens ? tokens[b] : -1;
  const bool given = tok >= 0 && tok < V;
  const float mine = given ? at(row + tok) : INFINITY;
  float x[PACKS][8];
#pragma unroll
  for (int k = 0; k < PACKS; ++k) {
    const int t = lo + (k * NT + threadIdx.x) * 8;
    if (VEC && t + 8 <= V) {
      if constexpr (sizeof(T) == 2) {
        const u16x8 v = *reinterpret_cast<const u16x8*>(row + t);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = bf2f(v[i]);
      } else {
        const f32x4 p = *reinterpret_cast<const f32x4*>(row + t), q = *reinterpret_cast<const f32x4*>(row + t + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[k][i] = p[i];
          x[k][4 + i] = q[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k][i] = t + i < V ? at(row + t + i) : -INFINITY;
    }
  }
  float m = -INFINITY;
  int ahead = 0;
#pragma unroll
  for (int k = 0; k < PACKS; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m = fmaxf(m, x[k][i]);
      ahead += x[k][i] > mine;
    }
  // the run's maximum, sum and count
  float wm = warp_max(m);
  if (lane == 0) red[w] = wm;
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  float M = red[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) M = fmaxf(M, red[i]);
  const float base = M == -INFINITY ? 0.f : M;
  constexpr float kL2e = 1.4426950408889634f;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < PACKS; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) s += __builtin_amdgcn_exp2f((x[k][i] - base) * kL2e);
  s = warp_sum(s);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ahead += __shfl_xor(ahead, o, 64);
  if (lane == 0) {
    reds[w] = s;
    redn[w] = ahead;
  }
  // a number that n of the wave's lanes reach with their best token (0: fewer have one)
  if (n > 0) {
    u64 best = 0;
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = lo + (k * NT + threadIdx.x) * 8 + i;
        const u64 q = t < V ? key_of(x[k][i], t) : 0ull;
        best = q > best ? q : best;
      }
    u64 reach = 0;
#pragma unroll 1
    for (int bit = 63; bit >= 0; --bit) {
      const u64 want = reach | 1ull << bit;
      if (__popcll(__ballot(best >= want)) >= n) reach = want;
    }
    if (lane == 0) low[w] = reach;
    __syncthreads();
    u64 line = low[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) line = low[i] > line ? low[i] : line;
    if (line == 0) line = 1;
    if (best >= line) {
#pragma unroll
      for (int k = 0; k < PACKS; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int t = lo + (k * NT + threadIdx.x) * 8 + i;
          const u64 q = t < V ? key_of(x[k][i], t) : 0ull;
          if (q >= line) list[atomicAdd(&found, 1)] = q;
        }
    }
  }
  __syncthreads();
  if (n > 0) {
    const int have = found;
    u64* mine_top = top + ((int64_t)b * runs + c) * n;
    for (int i = threadIdx.x; i < have; i += NT) {
      const u64 q = list[i];
      int rank = 0;
      for (int j = 0; j < have; ++j) rank += list[j] > q;
      if (rank < n) mine_top[rank] = q;
    }
    for (int i = have + threadIdx.x; i < n; i += NT) mine_top[i] = 0;
  }
  if (threadIdx.x == 0) {
    float S = 0.f;
    int A = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      S += reds[i];
      A += redn[i];
    }
    float* o = part + ((int64_t)b * runs + c) * 4;
    o[0] = M;
    o[1] = S;
    o[2] = __int_as_float(A);
  }
}

// One workgroup a row: the row's sum, then every run's n likeliest are placed by how many of each run are ahead of them.
template <typename T>
__global__ __launch_bounds__(256) void logprobs_join_kernel(const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ tokens, int V, int n,
                                                            int runs, const float* __restrict__ part, const u64* __restrict__ top,
                                                            float* __restrict__ lp, int64_t* __restrict__ rank,
                                                            int64_t* __restrict__ top_ids, float* __restrict__ top_lp) {
  extern __shared__ __attribute__((aligned(16))) u64 keys[];
  __shared__ float red[32];
  const int b = blockIdx.x;
  const float* p = part + (int64_t)b * runs * 4;
  for (int i = threadIdx.x; i < runs * n; i += 256) keys[i] = top[(int64_t)b * runs * n + i];
  float m = -INFINITY;
  for (int i = threadIdx.x; i < runs; i += 256) m = fmaxf(m, p[4 * i]);
  const float M = block_max(m, red);
  constexpr float kL2e = 1.4426950408889634f;
  float s = 0.f;
  int ahead = 0;
  for (int i = threadIdx.x; i < runs; i += 256) {
    const float mi = p[4 * i];
    // (a run of -inf alone gives nothing; its sum may be NaN, which stays)
    s += mi == -INFINITY ? (p[4 * i + 1] != p[4 * i + 1] ? NAN : 0.f) : p[4 * i + 1] * __builtin_amdgcn_exp2f((mi - M) * kL2e);
    ahead += __float_as_int(p[4 * i + 2]);
  }
  const f32x2 both = block_sum2(s, 0.f, red);
  int there = 0;
  for (int i = threadIdx.x; i < runs * n; i += 256) there += keys[i] != 0;
  const f32x2 counts = block_sum2((float)ahead, (float)there, red);  // (below 2^24: exact)
  const float ls = M == -INFINITY && both[0] == 0.f ? 0.f : logf(both[0]);
  const float base = M == -INFINITY ? 0.f : M;
  if (threadIdx.x == 0) {
    const int64_t tok = tokens ? tokens[b] : -1;
    const bool given = tok >= 0 && tok < V;
    lp[b] = given ? at(logits + (int64_t)b * ld + tok) - base - ls : 0.f;
    rank[b] = given ? (int64_t)counts[0] + 1 : 0;
  }
  for (int i = (int)counts[1] + threadIdx.x; i < n; i += 256) {  // (a row of so many NaN that there are no n others)
    top_ids[(int64_t)b * n + i] = -1;
    top_lp[(int64_t)b * n + i] = NAN;
  }
  for (int i = threadIdx.x; i < runs * n; i += 256) {
    const u64 q = keys[i];
    if (q == 0) continue;
    const int own = i / n;
    int place = i - own * n;
    for (int c = 0; c < runs; ++c) {
      if (c == own) continue;
      int lo = 0, hi = n;  // keys of run c above q
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (keys[c * n + mid] > q) lo = mid + 1;
        else hi = mid;
      }
      place += lo;
      if (place >= n) break;
    }
    if (place < n) {
      top_ids[(int64_t)b * n + place] = (int)~(unsigned)q;
      top_lp[(int64_t)b * n + place] = value_of(q) - base - ls;
    }
  }
}

constexpr int kNT = 256;

// 8-token packs of a thread: four, or one while those would fill the chip less than twice; two where the lists of the likeliest grow.
int packs_of(int B, int V, int n) {
  if (n > 32) return 2;
  return V > (1 << 18) || (int64_t)B * ((V + 4 * 8 * kNT - 1) / (4 * 8 * kNT)) >= 512 ? 4 : 1;
}

}  // namespace

int logprobs_runs(int B, int V, int n) {
  const int run = kNT * 8 * packs_of(B, V, n);
  return (V + run - 1) / run;
}

void launch_logprobs(const void* logits, int64_t ld, bool fp32, const void* tokens, int B, int V, int n, void* part, void* top, void* lp,
                     void* rank, void* top_ids, void* top_lp, hipStream_t st) {
  if (B == 0) return;
  if (B > 65535) throw std::runtime_error("token_logprobs: at most 65535 rows");
  if (n < 0 || n > kMostTop || n > V) throw std::runtime_error("token_logprobs: top_n must be between 0 and min(64, vocab)");
  const int packs = packs_of(B, V, n), runs = logprobs_runs(B, V, n);
  const size_t join = (size_t)runs * n * 8;
  if (V >= 1 << 24 || join > 60 * 1024) throw std::runtime_error("token_logprobs: vocabulary too large");
  const bool vec = (uintptr_t)logits % 16 == 0 && ld * (fp32 ? 4 : 2) % 16 == 0;
  const dim3 grid(runs, B);
#define LK(T_, P_, V_)                                                                                                  \
  logprobs_runs_kernel<T_, kNT, P_, V_><<<grid, kNT, std::min((size_t)n * 4, (size_t)kNT) * P_ * 8 * 8, st>>>((const T_*)logits, ld, (const int64_t*)tokens, V, n, \
                                                                                (float*)part, (u64*)top)
#define LP(T_)                                                                                                          \
  do {                                                                                                                  \
    if (packs == 4) {                                                                                                   \
      if (vec) LK(T_, 4, true);                                                                                         \
      else LK(T_, 4, false);                                                                                            \
    } else if (packs == 2) {                                                                                            \
      if (vec) LK(T_, 2, true);                                                                                         \
      else LK(T_, 2, false);                                                                                            \
    } else {                                                                                                            \
      if (vec) LK(T_, 1, true);                                                                                         \
      else LK(T_, 1, false);                                                                                            \
    }                                                                                                                   \
    HIP_CHECK_LAUNCH();                                                                                                 \
    logprobs_join_kernel<T_><<<B, 256, join, st>>>((const T_*)logits, ld, (const int64_t*)tokens, V, n, runs, (const float*)part, \
                                                   (const u64*)top, (float*)lp, (int64_t*)rank, (int64_t*)top_ids, (float*)top_lp); \
  } while (0)
  if (fp32) LP(float);
  else LP(bf16_t);
#undef LP
#undef LK
  HIP_CHECK_LAUNCH();
}
