// Log-probabilities of tokens: of a given token a row with its rank, and of the row's n likeliest tokens.
//
//   lp(t) = x_t - M - log sum_j exp(x_j - M),  M = max_j x_j;   rank = 1 + #{j: x_j > x_token};   equal logits: the lower token first
//
// Bound by memory: the logits are read once. A workgroup owns a run of a row's tokens in registers and leaves its maximum, its sum
// of exponentials, how many of its tokens are ahead of the given one, and its own n likeliest in order; a second launch joins a row's
// runs. The n likeliest of a run: a number that at least n tokens reach is found from the lanes' own maxima (a binary search over the
// upper bits of an order-preserving key, by ballots), and the few tokens that reach it are ranked by counting. Keys carry the token behind
// the value, so no two are equal: where a run of equal logits has more than the list takes, the search goes on over all bits. A NaN
// counts as no candidate, and makes its row's log-probabilities NaN; a row of nothing but -inf has log-probabilities of -inf. Few rows of
// ordinary vocabularies take one launch, a workgroup a row.
// One row of 32000 bf16 tokens 8.0 us, a chain of waits (tokens, maximum, sum, search, list); 64 of 50257 13.3, as they are one compute
// unit's each; 256 of 131071 fp32 tokens with 20 likeliest 28.6 + 6.5, the first 4.7 TB/s. Rows that do not start on 16 bytes are read a token
// at a time: 64 of 50257 bf16 tokens 23.5 us, 256 24.9 (aligned 13.3, 16.4).
#include "common.h"

#include <type_traits>

namespace {

constexpr int kMostTop = 64;
constexpr float kL2e = 1.4426950408889634f;
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

// A log-probability is x - base - log, from the row's maximum and its sum against it.
__device__ __forceinline__ float base_of(float M) { return M == -INFINITY ? 0.f : M; }
__device__ __forceinline__ float log_of(float M, float S) { return M == -INFINITY && S == 0.f ? 0.f : logf(S); }

template <typename T>
__device__ __forceinline__ float at(const T* p) {
  if constexpr (sizeof(T) == 2) return bf2f(*p);
  else return *p;
}

struct Answers {
  float* lp;
  int64_t *rank, *top_ids;
  float* top_lp;
};

// NT threads, up to PACKS x 8 tokens a thread, len a run. Partial results of run c of row b: part[b][c] = (m, s, ahead, -), top[b][c][n]
// keys. ALONE: a row is one run, and its results are the row's.
template <typename T, int NT, int PACKS, bool VEC, bool ALONE>
__global__ __launch_bounds__(NT) void logprobs_runs_kernel(const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ tokens, int V,
                                                           int n, int len, int cap, float* __restrict__ part, u64* __restrict__ top,
                                                           const Answers to) {
  constexpr int NW = NT / 64;
  const int b = blockIdx.y, c = blockIdx.x, runs = gridDim.x, lo = c * len, end = min(V, lo + len);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const T* row = logits + (int64_t)b * ld;
  __shared__ float red[NW], reds[NW], line[NW];
  __shared__ int redn[NW], redc[NW], found;
  extern __shared__ __attribute__((aligned(16))) u64 list[];  // cap keys
  const int64_t tok = tokens ? tokens[b] : -1;
  float x[PACKS][8];
#pragma unroll
  for (int k = 0; k < PACKS; ++k) {
    const int t = lo + (k * NT + threadIdx.x) * 8;
    if (VEC && t + 8 <= end) {
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
      for (int i = 0; i < 8; ++i) x[k][i] = t + i < end ? at(row + t + i) : -INFINITY;
    }
  }
  const bool given = tok >= 0 && tok < V;
  const float mine = given ? at(row + tok) : INFINITY;
  float m = -INFINITY;
  int ahead = 0;
#pragma unroll
  for (int k = 0; k < PACKS; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m = fmaxf(m, x[k][i]);
      ahead += x[k][i] > mine;
    }
  // the wave's maximum, and its sum against it (the waves' are joined at the end)
  const float wm = warp_max(m), base = base_of(wm);
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < PACKS; ++k) {  // (a pack's sum first: fewer roundings behind each other)
    float p = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) p += __builtin_amdgcn_exp2f((x[k][i] - base) * kL2e);
    s += p;
  }
  s = warp_sum(s);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ahead += __shfl_xor(ahead, o, 64);
  if (lane == 0) {
    red[w] = wm;
    reds[w] = s;
    redn[w] = ahead;
  }
  if (n > 0) {
    // a value that so many of the wave's lanes reach with their best (-inf: fewer do), to the upper 16 bits of its key
    const unsigned best = (unsigned)(key_of(m, 0) >> 32);
    auto reached_by = [&](int lanes) {
      unsigned reach = 0;
#pragma unroll
      for (int bit = 31; bit >= 16; --bit) {
        const unsigned want = reach | 1u << bit;
        if (__popcll(__ballot(best >= want)) >= lanes) reach = want;
      }
      return reach <= 0x007fffffu ? -INFINITY : value_of((u64)reach << 32);
    };
    // each wave's share of n, by the threads of it that have tokens: all of a share reach the least of the waves' values
    const int holders = min(NT, (end - lo + 7) / 8), held = min(max(holders - w * 64, 0), 64);
    const float part_of = held ? reached_by((n * held + holders - 1) / holders) : INFINITY;
    if (lane == 0) line[w] = part_of;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    float L = line[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) L = fminf(L, line[i]);
    if (holders < n) L = -INFINITY;
    if (m >= L) {  // (a thread without a token has -inf)
#pragma unroll
      for (int k = 0; k < PACKS; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int t = lo + (k * NT + threadIdx.x) * 8 + i;
          if (x[k][i] >= L && t < end) {
            const int p = atomicAdd(&found, 1);
            if (p < cap) list[p] = key_of(x[k][i], t);
          }
        }
    }
  }
  __syncthreads();
  float M = red[0], S = 0.f;
  int A = 0;
#pragma unroll
  for (int i = 1; i < NW; ++i) M = fmaxf(M, red[i]);
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    // (a wave of -inf alone gives nothing; its sum may be NaN, which stays)
    S += red[i] == -INFINITY ? reds[i] : reds[i] * __builtin_amdgcn_exp2f((red[i] - M) * kL2e);
    A += redn[i];
  }
  auto give = [&](int place, u64 q) {  // (0: a row of so many NaN that there are no n others)
    if constexpr (ALONE) {
      to.top_ids[(int64_t)b * n + place] = q ? (int)~(unsigned)q : -1;
      to.top_lp[(int64_t)b * n + place] = q ? value_of(q) - base_of(M) - log_of(M, S) : NAN;
    } else {
      top[((int64_t)b * runs + c) * n + place] = q;
    }
  };
  if (n > 0) {
    int have = found;
    if (have > cap) {  // (ties, or a run with few numbers: the same in every thread)
      // the exact way: keys that hold the token too are never equal, so n threads and no more reach the line with their best, or all
      // that have a token where those are fewer
      u64 best = 0;
#pragma unroll
      for (int k = 0; k < PACKS; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int t = lo + (k * NT + threadIdx.x) * 8 + i;
          const u64 q = t < end ? key_of(x[k][i], t) : 0ull;
          best = q > best ? q : best;
        }
      u64 l = 0;
#pragma unroll 1
      for (int bit = 63; bit >= 0; --bit) {
        const u64 want = l | 1ull << bit;
        const int mine = __popcll(__ballot(best >= want));
        __syncthreads();  // (the counts of the bit before are read)
        if (lane == 0) redc[w] = mine;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) all += redc[i];
        if (all >= n) l = want;
      }
      if (threadIdx.x == 0) found = 0;
      if (l == 0) l = 1;
      __syncthreads();
      if (best >= l) {
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int t = lo + (k * NT + threadIdx.x) * 8 + i;
            const u64 q = t < end ? key_of(x[k][i], t) : 0ull;
            if (q >= l) list[atomicAdd(&found, 1)] = q;
          }
      }
      __syncthreads();
      have = found;
    }
    for (int i = threadIdx.x; i < have; i += NT) {
      const u64 q = list[i];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < have; ++j) place += list[j] > q;
      if (place < n) give(place, q);
    }
    for (int i = have + threadIdx.x; i < n; i += NT) give(i, 0);
  }
  if (threadIdx.x == 0) {
    if constexpr (ALONE) {
      to.lp[b] = given ? mine - base_of(M) - log_of(M, S) : 0.f;
      to.rank[b] = given ? (int64_t)A + 1 : 0;
    } else {
      *reinterpret_cast<f32x4*>(part + ((int64_t)b * runs + c) * 4) = f32x4{M, S, __int_as_float(A), 0.f};
    }
  }
}

// One workgroup a row: the row's sum, then the runs' likeliest are ranked. Every run's keys stand in order, so of n keys that are wanted
// none lies below the j-th of each run with j = n / runs, nor below any run's n-th: what is left is ranked by counting.
template <typename T>
__global__ __launch_bounds__(256) void logprobs_join_kernel(const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ tokens, int V, int n,
                                                            int runs, const float* __restrict__ part, const u64* __restrict__ top,
                                                            float* __restrict__ lp, int64_t* __restrict__ rank,
                                                            int64_t* __restrict__ top_ids, float* __restrict__ top_lp) {
  extern __shared__ __attribute__((aligned(16))) u64 keys[];  // runs x n, and as many that are left
  __shared__ float redm[4], reds[4];
  __shared__ int reda[4], redt[4], left;
  __shared__ u64 redj[4], redn[4];
  const int b = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  u64* const kept = keys + (int64_t)runs * n;
  const int64_t tok = tokens ? tokens[b] : -1;
  const bool given = tok >= 0 && tok < V;
  const float mine = given ? at(logits + (int64_t)b * ld + tok) : 0.f;
  const int j = n > 0 ? min((n + runs - 1) / runs, n) : 0;
  float m = -INFINITY, s = 0.f;
  int ahead = 0, there = 0;
  u64 least = ~0ull, most = 0;  // of the runs' j-th keys, of their n-th ones
  for (int i = threadIdx.x; i < runs; i += 256) {
    const f32x4 p = *reinterpret_cast<const f32x4*>(part + ((int64_t)b * runs + i) * 4);
    const float t = fmaxf(m, p[0]);
    // (a run of -inf alone gives nothing; its sum may be NaN, which stays)
    s = (m == -INFINITY ? s : s * __builtin_amdgcn_exp2f((m - t) * kL2e)) + (p[0] == -INFINITY ? p[1] : p[1] * __builtin_amdgcn_exp2f((p[0] - t) * kL2e));
    m = t;
    ahead += __float_as_int(p[2]);
    if (n > 0) {
      const u64 kj = top[((int64_t)b * runs + i) * n + j - 1], kn = top[((int64_t)b * runs + i) * n + n - 1];
      least = kj < least ? kj : least;
      most = kn > most ? kn : most;
    }
  }
  for (int i = threadIdx.x; i < runs * n; i += 256) {
    const u64 q = top[(int64_t)b * runs * n + i];
    keys[i] = q;
    there += q != 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64), t = fmaxf(m, m2);
    s = (m == -INFINITY ? s : s * __builtin_amdgcn_exp2f((m - t) * kL2e)) + (m2 == -INFINITY ? s2 : s2 * __builtin_amdgcn_exp2f((m2 - t) * kL2e));
    m = t;
    ahead += __shfl_xor(ahead, o, 64);
    there += __shfl_xor(there, o, 64);
    const u64 l2 = __shfl_xor(least, o, 64), n2 = __shfl_xor(most, o, 64);
    least = l2 < least ? l2 : least;
    most = n2 > most ? n2 : most;
  }
  if (lane == 0) {
    redm[w] = m;
    reds[w] = s;
    reda[w] = ahead;
    redt[w] = there;
    redj[w] = least;
    redn[w] = most;
  }
  if (threadIdx.x == 0) left = 0;
  __syncthreads();
  float M = redm[0], S = 0.f;
  int A = 0, all = 0;
  u64 line = 0, lj = ~0ull;
#pragma unroll
  for (int i = 1; i < 4; ++i) M = fmaxf(M, redm[i]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    S += redm[i] == -INFINITY ? reds[i] : reds[i] * __builtin_amdgcn_exp2f((redm[i] - M) * kL2e);
    A += reda[i];
    all += redt[i];
    lj = redj[i] < lj ? redj[i] : lj;
    line = redn[i] > line ? redn[i] : line;
  }
  line = lj > line ? lj : line;
  if (line == 0) line = 1;
  const float base = base_of(M), ls = log_of(M, S);
  if (threadIdx.x == 0) {
    lp[b] = given ? mine - base - ls : 0.f;
    rank[b] = given ? (int64_t)A + 1 : 0;
  }
  if (n == 0) return;
  for (int i = threadIdx.x; i < runs * n; i += 256) {
    const u64 q = keys[i];
    if (q >= line) kept[atomicAdd(&left, 1)] = q;
  }
  for (int i = all + threadIdx.x; i < n; i += 256) {  // (a row of so many NaN that there are no n others)
    top_ids[(int64_t)b * n + i] = -1;
    top_lp[(int64_t)b * n + i] = NAN;
  }
  __syncthreads();
  const int have = left;
  for (int i = threadIdx.x; i < have; i += 256) {
    const u64 q = kept[i];
    int place = 0;
#pragma unroll 8
    for (int c = 0; c < have; ++c) place += kept[c] > q;
    if (place < n) {
      top_ids[(int64_t)b * n + place] = (int)~(unsigned)q;
      top_lp[(int64_t)b * n + place] = value_of(q) - base - ls;
    }
  }
}

// Threads and 8-token packs of a thread where a row is several runs. (Runs of one pack, for few rows: 2 rows of 131071 with the
// likeliest token 14.7 us and 15.1, 20 rows with 5 14.1 and 14.9, but 2 rows with 20 22.4 and 14.7: one form does for all.)
constexpr int kNT = 256, kPacks = 4;
constexpr int kAlone = 1024;  // threads where a row is one run

// Whether a row is one workgroup's, of 1024 threads with 2, 4 or 8 packs: while there is a compute unit for each (two workgroups
// with 2 packs share one). It saves the second launch and the partial results. The calls in one launch and in two, with the host's steps
// and from a captured graph, bf16: one row of 32000 11.7 and 15.6 us, captured 8.2 and 11.0; 128 rows of 32000 11.4 and 15.7, captured 10.2
// and 11.9; 512 of 9000 13.1 and 15.9, captured 12.7 and 14.1; 256 of 50257 16.4 and 19.6, captured 16.3 and 19.4; beyond, 300 rows of 32000
// 18.6 and 17.1, captured 18.4 and 16.3, 512 of 50257 29.7 and 27.3, captured 29.9 and 27.2. Few rows of 8 packs are the exception: 64 of
// 50257 take 13.9 us and 15.7 with the host's steps, but 13.3 and 12.1 captured (8 rows 12.4 and 11.4): the second launch costs a graph
// less than three quarters of the chip.
bool alone(int B, int V) { return V <= kAlone * 8 * 2 ? B <= 512 : V <= kAlone * 8 * 8 && B <= 256; }

// Keys that a run's list holds: several times what is found as a rule, and what the exact way may need.
int list_of(int n, int packs) { return n == 0 ? 0 : std::max(512, n * packs * 8); }

}  // namespace

int logprobs_runs(int B, int V) {
  if (alone(B, V)) return 0;
  constexpr int run = kNT * 8 * kPacks;
  return (V + run - 1) / run;
}

void launch_logprobs(const void* logits, int64_t ld, bool fp32, const void* tokens, int B, int V, int n, void* part, void* top, void* lp,
                     void* rank, void* top_ids, void* top_lp, hipStream_t st) {
  if (B == 0) return;
  if (B > 65535) throw std::runtime_error("token_logprobs: at most 65535 rows");
  if (n < 0 || n > kMostTop || n > V) throw std::runtime_error("token_logprobs: top_n must be between 0 and min(64, vocab)");
  const bool vec = (uintptr_t)logits % 16 == 0 && ld * (fp32 ? 4 : 2) % 16 == 0;
  const Answers to = {(float*)lp, (int64_t*)rank, (int64_t*)top_ids, (float*)top_lp};
#define LK(T_, NT_, P_, V_, A_)                                                                                            \
  logprobs_runs_kernel<T_, NT_, P_, V_, A_><<<grid, NT_, (size_t)list_of(n, P_) * 8, st>>>(                                \
      (const T_*)logits, ld, (const int64_t*)tokens, V, n, len, list_of(n, P_), (float*)part, (u64*)top, to)
#define LT(NT_, P_, A_)                                              \
  do {                                                               \
    if (fp32 && vec) LK(float, NT_, P_, true, A_);                   \
    else if (fp32) LK(float, NT_, P_, false, A_);                    \
    else if (vec) LK(bf16_t, NT_, P_, true, A_);                     \
    else LK(bf16_t, NT_, P_, false, A_);                             \
    HIP_CHECK_LAUNCH();                                              \
  } while (0)
  if (alone(B, V)) {
    const dim3 grid(1, B);
    const int len = V;
    if (V <= kAlone * 8 * 2) LT(kAlone, 2, true);
    else if (V <= kAlone * 8 * 4) LT(kAlone, 4, true);
    else LT(kAlone, 8, true);
    return;
  }
  const int runs = logprobs_runs(B, V);
  const int len = ((V + runs - 1) / runs + 7) / 8 * 8;  // (runs of a row as long as each other: a short last one has no better line)
  const size_t join = (size_t)runs * n * 8;
  if (V >= 1 << 24 || join > 30 * 1024) throw std::runtime_error("token_logprobs: vocabulary too large");
  const dim3 grid(runs, B);
  LT(kNT, kPacks, false);
#define LJ(T_)                                                                                                                \
  logprobs_join_kernel<T_><<<B, 256, 2 * join, st>>>((const T_*)logits, ld, (const int64_t*)tokens, V, n, runs, (const float*)part, \
                                                     (const u64*)top, to.lp, to.rank, to.top_ids, to.top_lp)
  if (fp32) LJ(float);
  else LJ(bf16_t);
#undef LJ
#undef LT
#undef LK
  HIP_CHECK_LAUNCH();
}
