// Rules on the logits in front of the sampler: penalties for tokens that were there before, biases of single tokens, and the mask
// of a grammar's state.
//
//   seen(t) = t among the row's known tokens, c(t) = how often among those behind the prompt
//   y = x;  seen: y = y > 0 ? y / r : y r;   y -= c f;   c > 0: y -= p;   y += the biases of t, in their order;   not allowed: -inf
//
// Bound by memory: each logit is read and written once. A workgroup owns a run of CH tokens of a row; it walks the row's known tokens and
// biases (from the caches: they are few beside the logits) and keeps what concerns its run in LDS - a counter a token, of 16 bits (two
// in a word) up to 32767 known tokens and 32 beyond, with a bit for "seen"; the run's biases as a list in their order. The logits are
// asked for first and come meanwhile; then the run goes through with 16-byte accesses, and only tokens whose counter is not zero cost more
// than a copy. Biased tokens are written once more at the end, by a thread each (found in the stream, by a table of them in LDS, 300
// biases a row cost 256 x 131071 fp32 logits 27 us beside 48, written once more 6). Integer counts, and biases summed in the order of the
// list: the result does not depend on the order in which threads run.
// 256 rows of 131071 fp32 logits 48 us as they are (5.6 TB/s), with up to 8000 known tokens, 300 biases and a mask 67; 64 of 50257 in bf16 with
// up to 1000 known tokens 9.6, one of 32000 3.9, a chain of waits. Rows that do not start on 16 bytes go a token at a time: 64 of 50257 in bf16
// 12.4 us, 256 31.7 (aligned 9.5, 21.8).
#include "common.h"

#include <type_traits>

namespace {

constexpr int kThreads = 512, kPacks = 4, kMostRun = kThreads * kPacks * 8;
constexpr int kMostBiases = 1024;

struct LogitRules {
  const void* x;
  int64_t ldx;
  void* y;
  int64_t ldy;
  const void* ids;
  int64_t ldi;
  int most;  // columns of ids
  const int *lens, *prompts;
  const float *rep, *pres, *freq;
  const int* bias_ids;
  const float* bias;
  int64_t ldb;
  int biases;
  const unsigned* mask;
  int64_t ldm;
  const int* mask_rows;
  int masks, V, wide;  // wide: ids of 64 bits
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const u16x8 x = *reinterpret_cast<const u16x8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf2f(x[i]);
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    u16x8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f2bf(v[i]);
    *reinterpret_cast<u16x8*>(p) = x;
  } else {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
}
template <typename T>
__device__ __forceinline__ float load1(const T* p) {
  if constexpr (sizeof(T) == 2) return bf2f(*p);
  else return *p;
}
template <typename T>
__device__ __forceinline__ void store1(T* p, float v) {
  if constexpr (sizeof(T) == 2) *p = f2bf(v);
  else *p = v;
}

// W: 16-bit counters, else 32. VEC: rows of both sides on 16 bytes.
template <typename TI, typename TO, bool W16, bool VEC>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(const LogitRules a, int CH) {
  extern __shared__ __attribute__((aligned(16))) unsigned lds[];
  const int b = blockIdx.y, lo = blockIdx.x * CH, n = min(CH, a.V - lo);
  constexpr unsigned kSeen = W16 ? 0x8000u : 0x80000000u, kCount = kSeen - 1;
  unsigned* cnt = lds;
  const int words = W16 ? CH / 2 : CH;
  int* list_t = (int*)(lds + words);  // the run's biases: tokens, values
  float* list_v = (float*)(list_t + a.biases);
  __shared__ int waves[2][kThreads / 64];
  const TI* x = (const TI*)a.x + (int64_t)b * a.ldx + lo;
  TO* y = (TO*)a.y + (int64_t)b * a.ldy + lo;

  const float r = a.rep ? a.rep[b] : 1.f, p = a.pres ? a.pres[b] : 0.f, f = a.freq ? a.freq[b] : 0.f;
  const int len = a.lens && (a.rep || a.pres || a.freq) ? min(max(a.lens[b], 0), a.most) : 0;
  const int mrow = a.mask ? (a.mask_rows ? a.mask_rows[b] : b) : -1;
  const unsigned* mask = mrow >= 0 && mrow < a.masks ? a.mask + (int64_t)mrow * a.ldm : nullptr;
  const bool marks = len > 0;
  // (each thread's one or two entries; they are placed below)
  static_assert(kMostBiases == 2 * kThreads, "two entries a thread");
  int bt[2] = {-1, -1};
  float bv[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = k * kThreads + threadIdx.x;
    if (i < a.biases) {
      bt[k] = a.bias_ids[(int64_t)b * a.ldb + i];
      bv[k] = a.bias[(int64_t)b * a.ldb + i];
    }
  }
  // the logits themselves are asked for first: they come while the known tokens are walked
  float v[VEC ? kPacks : 1][8];
  const int n8 = n & ~7;
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int t = (k * kThreads + threadIdx.x) * 8;
      if (t < n8) load8(x + t, v[k]);
    }
  }
  auto mark = [&](int t, unsigned v, bool add) {
    unsigned* c = W16 ? cnt + (t >> 1) : cnt + t;
    if (W16 && (t & 1)) v <<= 16;
    if (add) atomicAdd(c, v);
    else atomicOr(c, v);
  };
  if (marks) {
    for (int i = threadIdx.x * 4; i < words; i += kThreads * 4) *reinterpret_cast<u32x4*>(cnt + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    const int prompt = a.prompts ? min(max(a.prompts[b], 0), len) : 0;
    for (int i0 = threadIdx.x; i0 < len; i0 += 4 * kThreads) {
      int64_t t[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = min(i0 + k * kThreads, len - 1);
        t[k] = a.wide ? ((const int64_t*)a.ids)[b * a.ldi + i] : (int64_t)((const int*)a.ids)[b * a.ldi + i];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + k * kThreads;
        t[k] -= lo;
        if (i >= len || t[k] < 0 || t[k] >= n) continue;
        if (i >= prompt) mark((int)t[k], 1u, true);
        else mark((int)t[k], kSeen, false);
      }
    }
    __syncthreads();
  }
  auto rules = [&](float v, unsigned c) {
    const unsigned times = c & kCount;
    if (times || (c & kSeen)) v = v > 0.f ? v / r : v * r;
    if (times) v = __fsub_rn(__fsub_rn(v, __fmul_rn((float)times, f)), p);
    return v;
  };
  auto counter = [&](int t) { return W16 ? (cnt[t >> 1] >> (t & 1 ? 16 : 0)) & 0xffffu : cnt[t]; };
  auto masked = [&](int t) { return mask && !(mask[(lo + t) >> 5] >> ((lo + t) & 31) & 1); };
  auto one = [&](int t) {
    float v = load1(x + t);
    if (marks) {
      const unsigned c = counter(t);
      if (c) v = rules(v, c);
    }
    store1(y + t, masked(t) ? -INFINITY : v);
  };
  // the run's biases as a list in their order; each entry's token is the first entry's, whose thread sums it and writes the token at
  // the end, from the logit that it takes before any is overwritten
  int mine[2] = {-1, -1}, found = 0;
  float was[2], add[2];
  if (a.biases > 0) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned long long in[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      in[k] = __ballot(bt[k] >= lo && bt[k] < lo + n);
      if (lane == 0) waves[k][w] = __popcll(in[k]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int at = found + __popcll(in[k] & ((1ull << lane) - 1));
      for (int i = 0; i < kThreads / 64; ++i) {
        at += i < w ? waves[k][i] : 0;
        found += waves[k][i];
      }
      if (in[k] >> lane & 1) {
        list_t[at] = bt[k] - lo;
        list_v[at] = bv[k];
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = k * kThreads + threadIdx.x;
      if (e >= found) continue;
      const int t = list_t[e];
      was[k] = load1(x + t);
      float sum = 0.f;
      bool first = true, any = false;
      for (int j = 0; j < found; ++j) {
        if (list_t[j] != t) continue;
        if (j < e) first = false;
        sum = any ? sum + list_v[j] : list_v[j];
        any = true;
      }
      add[k] = sum;
      if (first) mine[k] = t;
    }
    __syncthreads();
  }
  if constexpr (!VEC) {
    for (int t = threadIdx.x; t < n; t += kThreads) one(t);
  } else {
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int t = (k * kThreads + threadIdx.x) * 8;
      if (t >= n8) break;
      unsigned open = 0xff;
      if (mask) open = mask[(lo + t) >> 5] >> ((lo + t) & 31);
      if (marks) {
        unsigned c[8], any = 0;
        if constexpr (W16) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(cnt + t / 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            c[2 * i] = w[i] & 0xffffu;
            c[2 * i + 1] = w[i] >> 16;
            any |= w[i];
          }
        } else {
          const u32x4 w0 = *reinterpret_cast<const u32x4*>(cnt + t), w1 = *reinterpret_cast<const u32x4*>(cnt + t + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            c[i] = w0[i];
            c[4 + i] = w1[i];
            any |= w0[i] | w1[i];
          }
        }
        if (any) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c[i]) v[k][i] = rules(v[k][i], c[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = open >> i & 1 ? v[k][i] : -INFINITY;
      store8(y + t, v[k]);
    }
    for (int t = n8 + threadIdx.x; t < n; t += kThreads) one(t);
  }
  if (a.biases > 0) {
    __syncthreads();  // (what was written above is there)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (mine[k] < 0) continue;
      float v = was[k];
      if (marks) {
        const unsigned c = counter(mine[k]);
        if (c) v = rules(v, c);
      }
      store1(y + mine[k], masked(mine[k]) ? -INFINITY : v + add[k]);
    }
  }
}

template <typename TI, typename TO>
void launch_rules(const LogitRules& a, int B, bool w16, hipStream_t st) {
  const bool vec = ((uintptr_t)a.x | (uintptr_t)a.y) % 16 == 0 && a.ldx * sizeof(TI) % 16 == 0 && a.ldy * sizeof(TO) % 16 == 0;
  // Runs as long as 1024 workgroups or more are left: a run's workgroup walks all that is known of the row (64 rows of 50257 with 500
  // known tokens 12.0 us, with 256 workgroups 12.6, with 4096 14.9; 256 of 131071 52.6, with 256 52.8, with 4096 51.0).
  int CH = 1024;
  while (CH < (w16 ? kMostRun : kMostRun / 2) && (int64_t)B * ((a.V + CH - 1) / CH) > 1024) CH *= 2;
  const dim3 grid((a.V + CH - 1) / CH, B);
  const size_t lds = (size_t)(w16 ? CH * 2 : CH * 4) + (size_t)a.biases * 8;
#define LR(W_, V_) adjust_logits_kernel<TI, TO, W_, V_><<<grid, kThreads, lds, st>>>(a, CH)
  if (w16) {
    if (vec) LR(true, true);
    else LR(true, false);
  } else {
    if (vec) LR(false, true);
    else LR(false, false);
  }
#undef LR
}

}  // namespace

void launch_adjust_logits(const void* x, int64_t ldx, bool x32, void* y, int64_t ldy, bool y32, int B, int V, const void* ids, int64_t ldi,
                          int most, bool ids64, const void* lens, const void* prompts, const void* rep, const void* pres,
                          const void* freq, const void* bias_ids, const void* bias, int64_t ldb, int biases, const void* mask,
                          int64_t ldm, const void* mask_rows, int masks, hipStream_t st) {
  if (B == 0 || V == 0) return;
  if (B > 65535) throw std::runtime_error("adjust_logits: at most 65535 rows");
  if (biases > kMostBiases) throw std::runtime_error("adjust_logits: at most 1024 biases a row");
  LogitRules a;
  a.x = x;
  a.ldx = ldx;
  a.y = y;
  a.ldy = ldy;
  a.ids = ids;
  a.ldi = ldi;
  a.most = most;
  a.lens = (const int*)lens;
  a.prompts = (const int*)prompts;
  a.rep = (const float*)rep;
  a.pres = (const float*)pres;
  a.freq = (const float*)freq;
  a.bias_ids = (const int*)bias_ids;
  a.bias = (const float*)bias;
  a.ldb = ldb;
  a.biases = bias_ids ? biases : 0;
  a.mask = (const unsigned*)mask;
  a.ldm = ldm;
  a.mask_rows = (const int*)mask_rows;
  a.masks = masks;
  a.V = V;
  a.wide = ids64;
  const bool w16 = most < 0x8000;
  if (x32) launch_rules<float, float>(a, B, w16, st);
  else if (y32) launch_rules<bf16_t, float>(a, B, w16, st);
  else launch_rules<bf16_t, bf16_t>(a, B, w16, st);
  HIP_CHECK_LAUNCH();
}
