// Attention of a batch whose sequences share a long prefix: the prefix's keys and values are read once for all rows, not once
// a sequence.
//
// Row t (sequence b, position p) attends positions 0 .. p. The first P positions of every context lie in the pages of ONE
// table, the others in pages of the sequence's own:
//   s_j = scale q . k_j,   o = sum_j exp(s_j - M) v_j / sum_j exp(s_j - M)
// A softmax over two sets of keys is joined from the sets' own maxima, sums and unnormalised outputs:
//   M = max_i m_i,   o = sum_i e^(m_i - M) o_i / sum_i e^(m_i - M) l_i
// so the prefix (all rows of the batch against a run of its keys a workgroup) and the own parts are worked on apart, each leaving
// (m, l, o) in fp32. The prefix's share is bound by matrix instructions and what they are fed from LDS from some 200 rows a key head on,
// the own parts by memory.
//
// Both kinds take (row, query head of the key head's group) pairs as "slots", the columns of swapped products
//   S^T[key][slot] = K Q^T,   O^T[dim][slot] += V^T P^T
// so that a lane owns a slot's softmax (lane & 15) and P^T is made in the registers that the second product takes it from.
// Two forms of a workgroup:
//  rows by waves - many slots: each wave has 16 NS slots of its own, all four share tiles of keys and values in LDS (two places:
//    the next tile is fetched while one is computed). A fragment from LDS feeds NS matrix instructions; two of them ask LDS for all that it
//    gives, 128 bytes a cycle, so one group cannot pass half of the matrix rate.
//  keys by waves - up to 16 slots (single tokens' own parts, a few rows behind a prefix): the waves walk different keys of the same
//    slots, without a barrier, keys straight into registers, and meet at the end. One slot of 16 may be real: 64 keys of 128
//    numbers cost a wave about 1000 cycles, memory takes 3500 to bring a compute unit's share of them. Few registers and 38 KB of LDS, so
//    that four workgroups share a compute unit.
// Together they make three kinds of call (`shared_plan`): both parts in one launch of either form and a launch that joins, or the prefix
// by rows and then own parts by keys, which join the prefix's results themselves.
//
// Measured: 128 rows of 64 heads in 8 groups behind 16381 positions 83 us for the prefix (830 TFLOP/s; 256 rows
// behind 16384 135 us, 1.0 PFLOP/s), 39 for own parts of up to 500; 64 rows of 32 heads behind 2048 positions 12 + 28 (own parts at
// 4 TB/s); 16 heads of 256 with 24 questions behind 1777 positions 101 - 106 (530 TFLOP/s, near what one group a fragment allows) + 17 for the
// join.
//
// Keys that a slot does not see weigh nothing whatever lies there: scores are replaced, not multiplied; and where a tile that is masked
// for some slots holds values that are not finite, they are kept from the slots that do not see them (see `add_values`). In place of rows past
// the last visible key a row that the cache has is loaded: the last visible one again or, by keys, one of a page that was asked for before
// the length was known.
// fp8 cache rows: e4m3 numbers are exact in bf16, a row's scale multiplies its score and its weight.
#include "common.h"

#include <cfloat>
#include <type_traits>

namespace {

constexpr float kLog2eS = 1.4426950408889634f;
constexpr float kFloor = -FLT_MAX;  // a maximum before any key was seen
constexpr int kTail = 16;           // bytes behind the numbers of an fp8 cache row, the first four its scale

struct SharedAttn {
  const bf16_t* q;
  int64_t q_stride;
  const void *kc, *vc;
  const int* prefix_table;
  const int* bt;
  int64_t bt_stride;
  const int* cu;   // null: row t is sequence t
  const int* ctx;  // positions of a sequence's context, its new ones among them
  float *po, *pml;
  bf16_t* out;
  int64_t out_stride;
  int parts, finish;  // partial results of a (row, head); whether the own parts' launch joins them itself
  unsigned page_bytes;
  int T, B, nh, nkv, G, bs, shift, pages, P, own_cap;  // shift: log2 of bs where it is a power of two
  int pre_items, pre_tiles, pre_split, pre_keys, pre_few;
  int own_tiles, own_split, own_keys, own_few;
  float scale_log2;
};

// The sequence of a row, or -1: the last one that begins at or before it (so one with rows, where several begin there).
__device__ __forceinline__ int seq_of(const SharedAttn& a, int t) {
  if (!a.cu) return t < a.B ? t : -1;
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return t >= a.cu[lo] && t < a.cu[lo + 1] ? lo : -1;
}

// Positions that a row sees.
__device__ __forceinline__ int seen_by(const SharedAttn& a, int t) {
  const int b = seq_of(a, t);
  if (b < 0) return 0;
  const int left = a.cu ? a.cu[b + 1] - 1 - t : 0;  // rows of the sequence behind this one
  return max(0, a.ctx[b] - left);
}

// What a workgroup works on: slots [first, slots) in rows from row0 on, keys [begin, stop) of a table's.
struct Item {
  const int* table;
  int row0, slots, first, kvh, begin, stop, part, own;
};

__device__ __forceinline__ int slot_limit(const SharedAttn& a, const Item& it, int slot) {
  const int n = seen_by(a, it.row0 + slot / a.G);
  return it.own ? min(max(n - a.P, 0), a.own_cap) : min(n, a.P);
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (that m0, which `to_lds` names as changed, is none of the registers the compiler gives out)
// Where the cache rows of a tile of 16 KT keys lie, in bytes. Pages of 16, 32, 64 .. positions (BY16): a lane asks for the page of one
// run of 16 keys, a tile ahead (a vector load, which the wait in front of the next tile covers: a scalar one would have the reads of
// LDS wait for it); a run's address is formed in scalar registers, a lane adds 32 bits. Others: each row asks for its own page where
// it is needed. RB: bytes of a cache row.
template <bool BY16, int KT, int RB>
struct Rows {
  const SharedAttn& a;
  const Item& it;
  int ids = 0;
  // a page's first byte of this key head; one that the cache does not have counts as the first
  __device__ __forceinline__ int64_t start(int page) const {
    const unsigned p = (unsigned)page < (unsigned)a.pages ? (unsigned)page : 0u;
    return (int64_t)((uint64_t)p * a.page_bytes) + (int64_t)it.kvh * a.bs * RB;
  }
  __device__ __forceinline__ int base(int kv0, int run) const { return min(kv0 + 16 * run, (it.stop - 1) & ~15); }
  __device__ __forceinline__ void ask(int kv0) {  // (in front of other accesses to memory: else it is moved to where its answer is used)
    if constexpr (BY16) ids = it.table[min(kv0 + 16 * (int)(threadIdx.x % KT), it.stop - 1) >> a.shift];
  }
  // what was asked for: the bytes in front of each run of the tile, a run a lane
  __device__ __forceinline__ int64_t asked(int kv0) const {
    return BY16 ? start(ids) + (base(kv0, threadIdx.x % KT) & (a.bs - 1)) * RB : 0;
  }
  // the bytes in front of a lane's own row of the tile
  __device__ __forceinline__ int64_t own_row(int64_t runs, int kv0, int row) const {
    if constexpr (BY16) return __shfl(runs, row >> 4, 64) + min(row & 15, it.stop - 1 - base(kv0, row >> 4)) * RB;
    else return alone(kv0 + row);
  }
  __device__ __forceinline__ int64_t of_run(int64_t runs, int run) const {
    return (int64_t)((uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(runs >> 32), run) << 32 | (unsigned)__builtin_amdgcn_readlane((int)runs, run));
  }
  // row r < 16 of run `run` of a tile, the same run in every lane; keys past the last stand for the last
  __device__ __forceinline__ unsigned row_at(int kv0, int run, int r) const { return min(r, it.stop - 1 - base(kv0, run)) * RB; }
  __device__ __forceinline__ int64_t alone(int k) const {
    k = min(k, it.stop - 1);
    const int i = k / a.bs;
    return start(it.table[i]) + (k - i * a.bs) * RB;
  }
  template <typename V>
  __device__ __forceinline__ V load(const void* cache, int64_t run_at, int kv0, int run, int r, unsigned more) const {
    if constexpr (BY16) return *reinterpret_cast<const V*>((const char*)cache + run_at + (row_at(kv0, run, r) + more));
    else return *reinterpret_cast<const V*>((const char*)cache + alone(kv0 + 16 * run + r) + more);
  }
  // 16 bytes a lane from memory into LDS (lane l at `at` + 16 l, the same `at` in every lane). Through inline assembly, so that the compiler does not hold reads
  // of other places in LDS back until it has landed: every use stands behind a wait for vmcnt(0) of its own. The compiler does not see into it: it is told
  // that m0 changes, and the base is written again by a scalar move (which also is what has to stand between a write of m0 and the load), as one that a
  // vector instruction wrote (a spilled one's v_readlane) may not be read by a load within five instructions.
  __device__ __forceinline__ void to_lds(const char* p, unsigned off, unsigned at) const {  // (all of a run's rows: p the run's, off a lane's)
    asm volatile("s_mov_b32 m0, %2\n\ts_mov_b64 %0, %0\n\tglobal_load_lds_dwordx4 %1, %0" : "+s"(p) : "v"(off), "s"(at) : "memory", "m0");
  }
  __device__ __forceinline__ void to_lds(const void* cache, int64_t run_at, int kv0, int run, int r, unsigned more, unsigned at) const {
    if constexpr (BY16) {
      to_lds((const char*)cache + run_at, row_at(kv0, run, r) + more, at);
    } else {
      const char* p = (const char*)cache + alone(kv0 + 16 * run + r) + more;
      asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(at) : "memory", "m0");
    }
  }
};
#pragma clang diagnostic pop

// Has the compiler wait for what was loaded into x: a first use inside a loop would be waited for in every turn, and with it
// for the loads into LDS that it does not count.
__device__ __forceinline__ void landed(s16x8& x) { asm volatile("" : "+v"(x)); }

__device__ __forceinline__ s16x8 fp8_to_bf16(unsigned lo, unsigned hi) {
  const u32x4 o = {__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                   __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                   __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                   __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
  return __builtin_bit_cast(s16x8, o);
}

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// The order of a block's reads of LDS and matrix instructions: AHEAD reads first, then after every M matrix instructions R reads more,
// until N are made. Left alone the compiler reads one fragment ahead, and every product waits most of a read's time.
template <int N, int AHEAD, int R, int M>
__device__ __forceinline__ void read_ahead() {
  constexpr int kRead = 0x100, kMfma = 0x8;
  __builtin_amdgcn_sched_group_barrier(kRead, AHEAD, 0);
#pragma unroll
  for (int i = AHEAD; i < N; i += R) {
    __builtin_amdgcn_sched_group_barrier(kMfma, M, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, R, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMfma, AHEAD / R * M, 0);
}

// 16-byte chunk c of row r in an LDS image of unpadded rows: rows of 16 reads and of transposing reads fall on different banks.
template <int D>
__device__ __forceinline__ int swz(int c, int r) {
  return D >= 128 ? c ^ ((r & 7) << 1) : c ^ (r & 7);
}

// V^T fragment of 32 keys (from row r32 of the image on) and 16 dims.
template <int D>
__device__ __forceinline__ s16x8 v_fragment(const char* img, int r32, int dt, int g, int li) {
  const int tq = li >> 2, tp = li & 3;
  const int r0 = r32 + 4 * g + tq, r1 = r0 + 16, c = 2 * dt + (tp >> 1);
  const char* a0 = img + r0 * D * 2 + (swz<D>(c, r0) << 4) + (tp & 1) * 8;
  const char* a1 = img + r1 * D * 2 + (swz<D>(c, r1) << 4) + (tp & 1) * 8;
  const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(a0));
  const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(a1));
  return s16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
}

// The scale of row `r` of an fp8 tile of N rows, and its reciprocal behind the N scales. Scales below 2^-100 count as that (their rows hold
// nothing above 4e-28); a reciprocal of what is not finite is 0, as such a scale may belong to a row that is not seen.
template <int N>
__device__ __forceinline__ void keep_scale(float* at, int r, float scale) {
  if (fabsf(scale) < 0x1p-100f) scale = 0x1p-100f;
  at[r] = scale;
  const float inv = fabsf(scale) < INFINITY ? __builtin_amdgcn_rcpf(scale) : 0.f;
  bf16_t* const two = reinterpret_cast<bf16_t*>(at + N);
  const bf16_t hi = f2bf(inv);
  two[r] = hi;
  two[N + r] = f2bf(inv - bf2f(hi));
}

// A maximum whose steps are 2 or more (not the one before any key was seen).
__device__ __forceinline__ bool far_off(float m) { return fabsf(m) >= 0x1p24f && m != kFloor; }

// Scores of 16 KT keys and NS groups of slots become weights: the running maximum of a slot moves only where its own has grown by
// more than 8 (weights stay below 2^8), so most tiles exchange nothing between lanes and rescale nothing. Weights are rounded to
// bf16 for the second product (half a step of 2^-8, as any bf16 operand); their sum is taken of the rounded ones, by a product with
// ones, so that they add up to 1 as they are used. fp8 rows: a weight times its row's scale (vscale) is what is rounded, so in place of the
// ones stand the scales' reciprocals, in two bf16 numbers that hold 16 bits of them (behind the scales, see `keep_scale`). Against 64 bits
// 0.0019; with a sum of the weights as they were, 0.0024 and for peaked rows 0.0027. lim: keys [.., lim) are seen, counted from the tile's first.
// An exponent is s scale - m in one rounding, while m is the rounded product: off by up to half a step of m, the same for every key of the
// slot, so that it cancels, but from 2^31 on it would take the weights out of range. From 2^24 on (`far`, the same for all lanes of the wave, looked
// at where a maximum moves) the product is rounded first, and the largest key's exponent is 0.
template <int D, int KT, int NS, bool MASK, bool KV8>
__device__ __forceinline__ void soften(f32x4 (&s)[NS][KT], const int (&lim)[NS], float scale_log2, int g, float (&m)[NS], int& far,
                                       f32x4 (&lsum)[NS], f32x4 (&o)[NS][D / 16], s16x8 (&pf)[NS][KT / 2], const float* vscale) {
  float mx[NS];
  bool grew = false;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    mx[n] = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (MASK) s[n][kt][i] = kt * 16 + 4 * g + i < lim[n] ? s[n][kt][i] : -INFINITY;
        mx[n] = fmaxf(mx[n], s[n][kt][i]);
      }
    mx[n] *= scale_log2;
    grew |= mx[n] > m[n] + 8.f;
  }
  if (__ballot(grew || far)) {
    bool any = false;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const float top = xor32_max(xor16_max(mx[n]));
      const bool up = top > m[n] + 8.f;
      const float alpha = up ? __builtin_amdgcn_exp2f(m[n] - top) : 1.f;
      if (up) m[n] = top;
      any |= far_off(m[n]);
#pragma unroll
      for (int i = 0; i < 4; ++i) lsum[n][i] *= alpha;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] *= alpha;
    }
    far = __ballot(any) != 0;
    if (far) {  // (slots near 0 beside them keep their one rounding)
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float p = s[n][kt][i] * scale_log2;
            asm("" : "+v"(p));  // (or the difference is taken in one rounding with it)
            s[n][kt][i] = far_off(m[n]) ? p - m[n] : fmaf(s[n][kt][i], scale_log2, -m[n]);
          }
    }
  }
  const float by = far ? 1.f : scale_log2;
  const s16x8 ones = {0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80};
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const float nm = far ? 0.f : -m[n];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      f32x4 v;
      if constexpr (KV8) v = *reinterpret_cast<const f32x4*>(vscale + kt * 16 + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[n][kt][i], by, nm));
        short w;
        if constexpr (KV8) {
          w = (short)f2bf(p * v[i]);
          if (MASK && p == 0.f) w = 0;  // (a key that is not seen: its scale may be anything)
        } else {
          w = (short)f2bf(p);
        }
        pf[n][kt >> 1][(kt & 1) * 4 + i] = w;
      }
    }
#pragma unroll
    for (int k = 0; k < KT / 2; ++k) {
      if constexpr (KV8) {
        const short* const two = reinterpret_cast<const short*>(vscale + 16 * KT) + 32 * k + 4 * g;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const s16x4 x = *reinterpret_cast<const s16x4*>(two + h * 16 * KT), y = *reinterpret_cast<const s16x4*>(two + h * 16 * KT + 16);
          lsum[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, pf[n][k], lsum[n], 0, 0, 0);
        }
      } else {
        lsum[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[n][k], lsum[n], 0, 0, 0);
      }
    }
  }
}

// O^T += V^T P^T. Where a tile that is masked for some slots holds values that are not finite, the products would give them to every
// slot (0 times such a value is NaN): there the weights go through `own_lds` (16 slots of 16 KT keys, the wave's own) and each slot
// takes the keys that it sees one after the other. Rare, so kept small.
template <int D, int KT, int NS, bool FEW>
__device__ __forceinline__ void add_values(bool masked, const char* img, bf16_t* own_lds, const int (&lim)[NS], int g_, int li_,
                                           const s16x8 (&pf)[NS][KT / 2], f32x4 (&o)[NS][D / 16]) {
  if (masked) {
    int g = g_, li = li_;
    asm volatile("" : "+v"(g), "+v"(li));  // (the rare path's addresses are formed in it and hold no registers outside)
    unsigned bad = 0;
#pragma unroll
    for (int k = 0; k < KT / 2; ++k)
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        const u32x4 x = __builtin_bit_cast(u32x4, v_fragment<D>(img, 32 * k, dt, g, li));
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= (x[i] & 0x7f807f80u) + 0x00800080u;  // (an exponent of ones carries into bit 15)
        if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    if (__ballot((bad & 0x80008000u) != 0)) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const s16x8& p = pf[n][kt >> 1];
          const int h = (kt & 1) * 4;
          *reinterpret_cast<s16x4*>(own_lds + li * 16 * KT + kt * 16 + 4 * g) = s16x4{p[h], p[h + 1], p[h + 2], p[h + 3]};
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int last = min(lim[n], 16 * KT);
#pragma unroll 1
        for (int k = 0; k < last; ++k) {
          const float p = bf2f(own_lds[li * 16 * KT + k]);
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            const u16x4 v = *reinterpret_cast<const u16x4*>(img + k * D * 2 + (swz<D>(2 * dt + (g >> 1), k) << 4) + (g & 1) * 8);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][dt][i] = fmaf(p, bf2f(v[i]), o[n][dt][i]);
          }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < KT / 2; ++k)
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const s16x8 vf = v_fragment<D>(img, 32 * k, dt, g_, li_);
#pragma unroll
      for (int n = 0; n < NS; ++n) o[n][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n][k], o[n][dt], 0, 0, 0);
      if (FEW && dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (second form: no registers for more reads ahead)
    }
  if constexpr (!FEW) read_ahead<KT / 2 * (D / 16) * 2, 8, 2, NS>();
}

// A sum of no weights is left as -0, one of weights of zero (keys of -inf) as +0, so that a row that sees nothing gets zeros and one that
// sees keys of -inf alone, and has no softmax, 0 / 0.
constexpr unsigned kNone = 0x80000000u;

// A softmax over several sets of keys from the sets' (m, l) and four of their outputs.
struct Joined {
  float top = kFloor, l = 0.f;
  unsigned none = kNone;  // (as long as every set's sum is -0)
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(f32x2 ml, f32x4 x) {
    none &= __float_as_uint(ml[1]);
    if (ml[1] == 0.f) return;  // (a set without a visible key; its outputs may be anything)
    const float t = fmaxf(top, ml[0]), f = __builtin_amdgcn_exp2f(top - t), h = __builtin_amdgcn_exp2f(ml[0] - t);
    top = t;
    l = l * f + ml[1] * h;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * f + x[e] * h;
  }
  // parts first, first + step, .. < n, N asked for at a time
  template <int D, int N>
  __device__ __forceinline__ void add_parts(const float* ml, const float* x, int first, int step, int n) {
    for (int p = first; p < n; p += N * step) {
      f32x2 b[N];
      f32x4 v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int q = min(p + i * step, n - 1);
        b[i] = *reinterpret_cast<const f32x2*>(ml + 2 * q);
        v[i] = *reinterpret_cast<const f32x4*>(x + (int64_t)q * D);
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (p + i * step < n) add(b[i], v[i]);
    }
  }
  __device__ __forceinline__ float sum() const { return l == 0.f ? __uint_as_float(none) : l; }
  __device__ __forceinline__ void store(bf16_t* out) const {
    const float inv = __float_as_uint(sum()) == kNone ? 0.f : 1.f / l;
    u16x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = f2bf(o[e] * inv);
    *reinterpret_cast<u16x4*>(out) = r;
  }
};

// Parts first, first + step, .. < n of a slot join what its lanes hold of it (x: the lane's first dims of the first part).
template <int D>
__device__ __forceinline__ void add_parts(const float* ml, const float* x, int first, int step, int n, f32x4 (&o)[D / 16], float& m, f32x4& lsum) {
  f32x4 v[D / 16];
  f32x2 b = {kFloor, 0.f};
  auto load = [&](int p) {
    b = *reinterpret_cast<const f32x2*>(ml + 2 * p);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) v[dt] = *reinterpret_cast<const f32x4*>(x + (int64_t)p * D + dt * 16);
  };
  if (first < n) load(first);
  unsigned none = kNone;
#pragma unroll 1
  for (int p = first; p < n; p += step) {
    f32x4 w[D / 16];
    const f32x2 c = b;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) w[dt] = v[dt];
    if (p + step < n) load(p + step);
    none &= __float_as_uint(c[1]);
    if (c[1] == 0.f) continue;  // (a part without a visible key; its outputs may be anything)
    const float t = fmaxf(m, c[0]), f = __builtin_amdgcn_exp2f(m - t), h = __builtin_amdgcn_exp2f(c[0] - t);
    m = t;
#pragma unroll
    for (int e = 0; e < 4; ++e) lsum[e] = lsum[e] * f + c[1] * h;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[dt][e] = o[dt][e] * f + w[dt][e] * h;
  }
  if (lsum[0] == 0.f) lsum[0] = __uint_as_float(__float_as_uint(lsum[0]) & none);
}

template <int D>
__device__ __forceinline__ void leave(const SharedAttn& a, const Item& it, int slot, int g, const f32x4 (&o)[D / 16], float m, float l) {
  const int64_t pi = ((int64_t)(it.row0 + slot / a.G) * a.nh + it.kvh * a.G + slot % a.G) * a.parts + it.part;
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<f32x4*>(a.po + pi * D + dt * 16 + 4 * g) = o[dt];
  if (g == 0) {
    a.pml[pi * 2] = m;
    a.pml[pi * 2 + 1] = l;
  }
}

// ------------------------------------------------------------------------------------------------------ rows by waves
// Keys of a tile: 64, of wide heads 32 (two places of keys and values: 64 KB either way, two workgroups a compute unit).
constexpr int tile_keys(int D) { return D == 256 ? 32 : 64; }

template <int D, bool KV8, int NS, bool BY16>
__device__ __forceinline__ void rows_by_waves(const SharedAttn& a, Item it, char* smem, float* scales, bf16_t* apart, int* red) {
  constexpr int BKV = tile_keys(D), KT = BKV / 16;
  constexpr int CH = D / 8;          // 16-byte chunks of an LDS row
  constexpr int TILE = BKV * D * 2;  // bytes of a tile of keys, and of values
  // (a lane's number as something new each time: what follows from it is formed where it is used and holds no registers in between)
  auto anew = [&]() {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
  };
  const int lane = anew(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  int slot[NS], lim[NS];
  int lo = INT_MAX, hi = 0;
  unsigned blind = 0;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    slot[n] = it.first + (w * NS + n) * 16 + li;
    lim[n] = slot[n] < it.slots ? slot_limit(a, it, slot[n]) : 0;
    if (lim[n] > it.begin) {
      lo = min(lo, lim[n]);
      hi = max(hi, lim[n]);
    } else {
      // a slot behind the last, or one that sees none of the keys (of an idle row): no reason for a mask, its sum is made zero at the
      // end (128 rows, three of them idle, behind 16381 positions: with masks their workgroups hold the launch up, 103 us and not 84)
      lim[n] = INT_MAX;
      blind |= 1u << n;
    }
  }
  const int wave_lo = wave_min(lo), wave_hi = wave_max(hi);
  __syncthreads();  // (a workgroup may have had an item before)
  if (lane == 0) red[w] = wave_hi;
  __syncthreads();
  it.stop = __builtin_amdgcn_readfirstlane(min(it.stop, max(max(red[0], red[1]), max(red[2], red[3]))));

  f32x4 o[NS][D / 16], lsum[NS];
  float m[NS];
  int far = 0;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    m[n] = kFloor;
    lsum[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (it.stop > it.begin) {
    s16x8 qf[NS][D / 32];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int sl = min(slot[n], it.slots - 1);
      const bf16_t* qp = a.q + (int64_t)(it.row0 + sl / a.G) * a.q_stride + (int64_t)(it.kvh * a.G + sl % a.G) * D + 8 * g;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) qf[n][ks] = *reinterpret_cast<const s16x8*>(qp + 32 * ks);
    }
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) landed(qf[n][ks]);
    Rows<BY16, KT, KV8 ? D + kTail : 2 * D> rows{a, it};
    const int ntiles = (it.stop - it.begin + BKV - 1) / BKV;

    // bf16: 16 bytes a lane straight into LDS, a wave's instruction covers RPI rows
    constexpr int RPI = 64 / CH, LPW = BKV / RPI / 4;
    // fp8: 16 numbers a thread and piece, through registers
    constexpr int PIECES = BKV * (D / 16) / 256;
    u32x4 k8[KV8 ? PIECES : 1], v8[KV8 ? PIECES : 1];
    float sc = 0.f;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(LDS_AS char*)smem);
    const int lane_row = (D == 256 ? w * RPI : w * RPI & 15) + lane / CH;
    const unsigned lane_off = lane_row * 2 * D + (swz<D>(lane % CH, lane_row) << 4);
    auto fetch = [&](int j) {
      const int lane = anew();
      const int kv0 = it.begin + j * BKV;
      const unsigned sl = lds0 + (j & 1) * 2 * TILE;
      if constexpr (KV8) {
        const int64_t runs = rows.asked(kv0), at = rows.own_row(runs, kv0, threadIdx.x % BKV);
        int64_t pg[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; ++i)  // (16 rows of 4, 8 or 16 pieces: a wave's rows lie within one run of 16)
          pg[i] = rows.of_run(runs, __builtin_amdgcn_readfirstlane((threadIdx.x + i * 256) / D));
        rows.ask(kv0 + BKV);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int c = threadIdx.x + i * 256, r = c / (D / 16), run = __builtin_amdgcn_readfirstlane(c / D);
          k8[i] = rows.template load<u32x4>(a.kc, pg[i], kv0, run, r & 15, (c % (D / 16)) * 16);
          v8[i] = rows.template load<u32x4>(a.vc, pg[i], kv0, run, r & 15, (c % (D / 16)) * 16);
        }
        if (threadIdx.x < 2 * BKV)
          sc = *reinterpret_cast<const float*>((const char*)(threadIdx.x < BKV ? a.kc : a.vc) + at + D);
      } else {
        const int64_t runs = rows.asked(kv0);
        int64_t pg[LPW];
#pragma unroll
        for (int i = 0; i < LPW; ++i) pg[i] = rows.of_run(runs, (i * 4 + w) * RPI / 16);
        rows.ask(kv0 + BKV);
        if (BY16 && kv0 + BKV <= it.stop) {  // (a lane's row in its run and its chunk are the same for every instruction but for 8 rows)
#pragma unroll
          for (int i = 0; i < LPW; ++i) {
            const int inst = i * 4 + w;
            const int64_t at = pg[i] + (D == 256 ? (i & 1) * 8 * 2 * D : 0);
            rows.to_lds((const char*)a.kc + at, lane_off, sl + inst * 1024);
            rows.to_lds((const char*)a.vc + at, lane_off, sl + TILE + inst * 1024);
          }
          return;
        }
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
          const int inst = i * 4 + w, r = inst * RPI + lane / CH;
          rows.to_lds(a.kc, pg[i], kv0, inst * RPI / 16, r & 15, swz<D>(lane % CH, r) << 4, sl + inst * 1024);
          rows.to_lds(a.vc, pg[i], kv0, inst * RPI / 16, r & 15, swz<D>(lane % CH, r) << 4, sl + TILE + inst * 1024);
        }
      }
    };
    auto put = [&](int j) {  // (fp8) the pieces fetched last
      char* sk = smem + (j & 1) * 2 * TILE;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int c = threadIdx.x + i * 256, r = c / (D / 16), c0 = (c % (D / 16)) * 2;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = r * D * 2 + (swz<D>(c0 + h, r) << 4);
          *reinterpret_cast<s16x8*>(sk + at) = fp8_to_bf16(k8[i][2 * h], k8[i][2 * h + 1]);
          *reinterpret_cast<s16x8*>(sk + TILE + at) = fp8_to_bf16(v8[i][2 * h], v8[i][2 * h + 1]);
        }
      }
      if (threadIdx.x < BKV) scales[(j & 1) * 3 * BKV + threadIdx.x] = sc;
      else if (threadIdx.x < 2 * BKV) keep_scale<BKV>(scales + (j & 1) * 3 * BKV + BKV, threadIdx.x - BKV, sc);
    };
    auto tile = [&](int j, auto mask_c) {
      constexpr bool MASK = decltype(mask_c)::value;
      const int kv0 = it.begin + j * BKV;
      const char* sk = smem + (j & 1) * 2 * TILE;
      f32x4 s[NS][KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int n = 0; n < NS; ++n) s[n][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        s16x8 kf[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const int r = kt * 16 + li;
          kf[kt] = *reinterpret_cast<const s16x8*>(sk + r * D * 2 + (swz<D>(4 * ks + g, r) << 4));
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int n = 0; n < NS; ++n) s[n][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kt], qf[n][ks], s[n][kt], 0, 0, 0);
      }
      read_ahead<KT * (D / 32), 6, 1, NS>();
      __builtin_amdgcn_sched_barrier(0);
      const float* vs = nullptr;
      if constexpr (KV8) {
        const float* ks_ = scales + (j & 1) * 3 * BKV;
        vs = ks_ + BKV;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const f32x4 f = *reinterpret_cast<const f32x4*>(ks_ + kt * 16 + 4 * g);
#pragma unroll
          for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][kt][i] *= f[i];
        }
      }
      int left[NS];
#pragma unroll
      for (int n = 0; n < NS; ++n) left[n] = MASK ? min(lim[n], it.stop) - kv0 : BKV;
      s16x8 pf[NS][KT / 2];
      soften<D, KT, NS, MASK, KV8>(s, left, a.scale_log2, g, m, far, lsum, o, pf, vs);
      add_values<D, KT, NS, false>(MASK, sk + TILE, apart + w * 16 * BKV, left, g, li, pf, o);
    };
    // tiles that every slot of the wave sees whole come first, in a loop without masks
    const int whole = min(max(0, (min(wave_lo, it.stop) - it.begin) / BKV), ntiles);
    rows.ask(it.begin);
    fetch(0);
    if constexpr (KV8) {
      put(0);
      if (ntiles > 1) fetch(1);
    }
    auto next = [&](int j) {  // tile j is there for every wave; the place of tile j - 1 is free
      if constexpr (KV8) {
        __syncthreads();
        if (j + 1 < ntiles) {
          put(j + 1);
          if (j + 2 < ntiles) fetch(j + 2);
        }
      } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (j + 1 < ntiles) fetch(j + 1);
      }
    };
    int j = 0;
    for (; j < whole; ++j) {
      next(j);
      tile(j, std::false_type{});
    }
    for (; j < ntiles; ++j) {
      next(j);
      if (it.begin + j * BKV < wave_hi) tile(j, std::true_type{});
    }
  }
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const int l = anew(), slot = it.first + (w * NS + n) * 16 + (l & 15);
    if (slot < it.slots) leave<D>(a, it, slot, l >> 4, o[n], m[n], blind >> n & 1 ? -0.f : lsum[n][0]);
  }
}

// ------------------------------------------------------------------------------------------------------ keys by waves
// A wave takes every fourth run of 32 keys and asks for a run's keys and values together. Keys come straight into the first product's registers (fp8: 16 numbers a lane, so that
// a pair of products shares them: dims 64 m + 16 g + 8 h of the query's row stand beside them), values through LDS places of
// the wave's own.
template <int D, bool KV8, bool BY16>
__device__ __forceinline__ void keys_by_waves(const SharedAttn& a, Item it, char* smem, float* scales, bf16_t* apart) {
  constexpr int KT = 2, BK = 32, CH = D / 8;
  constexpr int TILE = BK * D * 2;
  // (a lane's number as something new each time: what follows from it is formed where it is used and holds no registers in between)
  auto anew = [&]() {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
  };
  const int lane = anew(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int slot = it.first + li;
  const bool real = slot < it.slots;
  Rows<BY16, KT, KV8 ? D + kTail : 2 * D> rows{a, it};
  const int step = 4 * BK;
  int kv0 = it.begin + w * BK;
  if (it.begin < it.stop) rows.ask(kv0);  // (beside the context's length: a page past it is not used)
  int lim[1] = {INT_MAX}, lo, hi;
  if (it.own && it.slots == a.G) {  // one token: a limit for all
    lim[0] = lo = hi = __builtin_amdgcn_readfirstlane(slot_limit(a, it, 0));
  } else {
    if (real) lim[0] = slot_limit(a, it, slot);
    lo = wave_min(it.own || lim[0] > it.begin ? lim[0] : INT_MAX);  // (of the prefix's parts those with a sum of zero are not looked at)
    hi = wave_max(real ? lim[0] : 0);
  }
  it.stop = min(it.stop, hi);

  f32x4 o[1][D / 16], lsum[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
  float m[1] = {kFloor};
  int far = 0;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) o[0][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  __syncthreads();  // (a workgroup may have had an item before: the places below are free)
  if (kv0 < it.stop) {
    s16x8 qf[D / 32];
    {
      const int sl = min(slot, it.slots - 1);
      const bf16_t* qp = a.q + (int64_t)(it.row0 + sl / a.G) * a.q_stride + (int64_t)(it.kvh * a.G + sl % a.G) * D;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
        qf[ks] = *reinterpret_cast<const s16x8*>(qp + (KV8 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g));
    }
    char* const img = smem + w * TILE;
    const unsigned img_at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(LDS_AS char*)img);
    float* const fac = scales + w * 3 * BK;  // (fp8) scales of the keys, of the values, what is kept behind those
    s16x8 kf[KT][KV8 ? 1 : D / 32];
    u32x4 k8[KT][KV8 ? D / 64 : 1];
    constexpr int RPI = 64 / CH, INS = BK / RPI, PIECES = BK * (D / 16) / 64;
    u32x4 v8[KV8 ? PIECES : 1];
    float sc = 0.f;
    int64_t scale_at = 0;
    auto keys = [&](int kv0, const int64_t (&pg)[KT]) {
      const int l = anew(), li = l & 15, g = l >> 4;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        if constexpr (KV8) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c) k8[kt][c] = rows.template load<u32x4>(a.kc, pg[kt], kv0, kt, li, 64 * c + 16 * g);
        } else {
#pragma unroll
          for (int ks = 0; ks < D / 32; ++ks) kf[kt][ks] = rows.template load<s16x8>(a.kc, pg[kt], kv0, kt, li, 64 * ks + 16 * g);
        }
      }
      if constexpr (KV8) sc = *reinterpret_cast<const float*>((const char*)(lane < BK ? a.kc : a.vc) + scale_at);
    };
    auto values = [&](int kv0, const int64_t (&pg)[KT]) {
      const int lane = anew();
      if constexpr (KV8) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int c = lane + i * 64, r = c / (D / 16);
          const int run = i * 64 / D;  // (16 rows are D pieces)
          v8[i] = rows.template load<u32x4>(a.vc, pg[run], kv0, run, r & 15, (c % (D / 16)) * 16);
        }
      } else {
#pragma unroll
        for (int i = 0; i < INS; ++i) {
          const int r = i * RPI + lane / CH;
          rows.to_lds(a.vc, pg[i * RPI / 16], kv0, i * RPI / 16, r & 15, swz<D>(lane % CH, r) << 4, img_at + i * 1024);
        }
      }
    };
    int64_t pg[KT];
    auto pages = [&](int kv0) {  // those asked for, and what lies a turn behind them is asked for
      const int64_t runs = rows.asked(kv0);
      if constexpr (KV8) scale_at = rows.own_row(runs, kv0, threadIdx.x % BK) + D;
#pragma unroll
      for (int i = 0; i < KT; ++i) pg[i] = rows.of_run(runs, i);
      rows.ask(kv0 + step);
    };
#pragma unroll 1
    for (; kv0 < it.stop; kv0 += step) {
      pages(kv0);
      keys(kv0, pg);
      values(kv0, pg);
      __builtin_amdgcn_sched_barrier(0);  // (no product, and no wait for its keys, between the loads)
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (KV8) {
        const int lane = anew();
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int c = lane + i * 64, r = c / (D / 16), c0 = (c % (D / 16)) * 2;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<s16x8*>(img + r * D * 2 + (swz<D>(c0 + h, r) << 4)) = fp8_to_bf16(v8[i][2 * h], v8[i][2 * h + 1]);
        }
        if (lane < BK) fac[lane] = sc;
        else keep_scale<BK>(fac + BK, lane - BK, sc);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      f32x4 s[1][KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) s[0][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          s16x8 f;
          if constexpr (KV8) f = fp8_to_bf16(k8[kt][ks >> 1][2 * (ks & 1)], k8[kt][ks >> 1][2 * (ks & 1) + 1]);
          else f = kf[kt][ks];
          s[0][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, qf[ks], s[0][kt], 0, 0, 0);
        }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (KV8) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const f32x4 f = *reinterpret_cast<const f32x4*>(fac + kt * 16 + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[0][kt][i] *= f[i];
        }
      }
      const float* vs = KV8 ? fac + BK : nullptr;
      s16x8 pf[1][1];
      const int left[1] = {min(lim[0], it.stop) - kv0};
      soften<D, KT, 1, true, KV8>(s, left, a.scale_log2, g, m, far, lsum, o, pf, vs);
      const int l = anew();
      add_values<D, KT, 1, true>(kv0 + BK > min(lo, it.stop), img, apart + w * 16 * BK, left, l >> 4, l & 15, pf, o);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the place is read)
    }
  }
  if (lim[0] <= it.begin) lsum[0][0] = -0.f;
  const bool finish = it.own && a.finish;
  if (finish) {  // the own part is one workgroup's: the prefix's parts, left by the launch before, join it here, every fourth a wave
    const int l = anew(), slot = it.first + (l & 15), g = l >> 4;
    const int sl = min(slot, it.slots - 1);
    const int64_t pi = ((int64_t)(it.row0 + sl / a.G) * a.nh + it.kvh * a.G + sl % a.G) * a.parts;
    add_parts<D>(a.pml + pi * 2, a.po + pi * D + 4 * g, w, 4, a.pre_split, o[0], m[0], lsum[0]);
  }
  // the waves meet: outputs [wave][slot][D] and (m, l)
  __syncthreads();
  float* const so = reinterpret_cast<float*>(smem);
  constexpr int LDO = D + 4;
  {
    const int l = anew(), li = l & 15, g = l >> 4;
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<f32x4*>(so + (w * 16 + li) * LDO + dt * 16 + 4 * g) = o[0][dt];
  if (g == 0) {
    scales[(w * 16 + li) * 2] = m[0];
    scales[(w * 16 + li) * 2 + 1] = lsum[0][0];
  }
  }
  __syncthreads();
#pragma unroll 1
  for (int c = w * 64 + anew(); c < 16 * (D / 4); c += 256) {
    const int sl = c / (D / 4), d4 = c % (D / 4);
    if (it.first + sl >= it.slots) continue;
    Joined j;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      j.add(*reinterpret_cast<const f32x2*>(scales + (i * 16 + sl) * 2), *reinterpret_cast<const f32x4*>(so + (i * 16 + sl) * LDO + d4 * 4));
    const int s_ = it.first + sl;
    const int64_t row = it.row0 + s_ / a.G, head = it.kvh * a.G + s_ % a.G;
    if (finish) {
      j.store(a.out + row * a.out_stride + head * D + d4 * 4);
    } else {
      const int64_t pi = (row * a.nh + head) * a.parts + it.part;
      *reinterpret_cast<f32x4*>(a.po + pi * D + d4 * 4) = j.o;
      if (d4 == 0) *reinterpret_cast<f32x2*>(a.pml + pi * 2) = f32x2{j.top, j.sum()};
    }
  }
}

enum Form { ROWS, KEYS };

// Items [0, pre_items) are the prefix's, the others own parts. The second form is bound by memory and takes few registers and little LDS:
// more of its workgroups share a compute unit.
template <int D, bool KV8, int NS, int FORM, bool BY16>
__global__ __launch_bounds__(256, FORM == KEYS && D < 256 ? 4 : 2) void attn_shared_kernel(const SharedAttn a) {
  constexpr int PLACES = FORM == ROWS ? 2 * 2 * tile_keys(D) * D * 2 : 4 * 32 * D * 2;  // tiles; each wave's values
  constexpr int MEET = FORM == ROWS ? 0 : 4 * 16 * (D + 4) * 4;                         // the second form's outputs
  __shared__ __attribute__((aligned(16))) char smem[PLACES > MEET ? PLACES : MEET];
  __shared__ __attribute__((aligned(16))) float scales[FORM == ROWS ? (KV8 ? 2 * 3 * tile_keys(D) : 4) : 4 * 3 * 32];
  __shared__ __attribute__((aligned(16))) bf16_t apart[4 * 16 * (FORM == KEYS ? 32 : tile_keys(D))];
  __shared__ int red[4];
  constexpr int per = FORM == KEYS ? 16 : 64 * NS;
  Item it;
  int id = blockIdx.x, tile, tiles;
  if (id < a.pre_items) {  // (key head, run of keys, tile of slots), the tiles of a run on one die
    id = xcd_remap(id, a.pre_items);
    const int run = id / a.pre_tiles;
    tile = id % a.pre_tiles;
    tiles = INT_MAX / 1024;  // (one turn)
    it.own = 0;
    it.table = a.prefix_table;
    it.row0 = 0;
    it.slots = a.T * a.G;
    it.kvh = run / a.pre_split;
    it.part = run % a.pre_split;
    it.begin = it.part * a.pre_keys;
    it.stop = min(a.P, it.begin + a.pre_keys);
  } else {
    id -= a.pre_items;
    const int run = id % a.own_split;
    tile = id / a.own_split % a.own_tiles;
    tiles = a.own_tiles;
    it.own = 1;
    it.kvh = id / a.own_split / a.own_tiles % a.nkv;
    const int b = id / a.own_split / a.own_tiles / a.nkv;
    it.table = a.bt + b * a.bt_stride;
    it.row0 = a.cu ? min(max(a.cu[b], 0), a.T) : b;
    it.slots = (a.cu ? max(min(a.cu[b + 1], a.T) - it.row0, 0) : 1) * a.G;
    it.part = a.pre_split + run;
    it.begin = run * a.own_keys;
    it.stop = run + 1 < a.own_split ? min(a.own_cap, it.begin + a.own_keys) : a.own_cap;
  }
  // (the grid is sized for the longest portion and own part that the caller names: longer ones take more turns)
  for (; tile < (it.slots + per - 1) / per; tile += tiles) {
    it.first = tile * per;
    if constexpr (FORM == ROWS) rows_by_waves<D, KV8, NS, BY16>(a, it, smem, scales, apart, red);
    else keys_by_waves<D, KV8, BY16>(a, it, smem, scales, apart);
    if (!it.own) break;
  }
}

// Groups of D / 4 threads, four numbers a thread. TOGETHER: so many of them, a workgroup, take a (row, head)'s parts in turn and meet in
// LDS, where there are more than 12 (the calls, a group alone and together: one row of 32 heads behind 120000 positions 61 us and 32, 10
// rows behind 4000 15.1 and 13.6, 33 rows of 48 heads behind 7990 26.3 and 25.2; with up to 12, 180 rows of 32 heads 30.2 and 32.5).
template <int D, int TOGETHER>
__global__ __launch_bounds__(256) void attn_shared_join_kernel(const SharedAttn a) {
  constexpr int PER = D / 4, EACH = PER * TOGETHER;
  const int64_t i = (int64_t)blockIdx.x * (256 / EACH) + threadIdx.x / EACH;
  const int grp = threadIdx.x % EACH / PER, d = threadIdx.x % PER * 4;
  const int t = i / a.nh, h = i % a.nh;
  const bool there = i < (int64_t)a.T * a.nh && seq_of(a, t) >= 0;  // (a row of no sequence stays as it was)
  Joined j;
  if (there) {
    const float *ml = a.pml + i * a.parts * 2, *x = a.po + i * a.parts * D + d;
    if (TOGETHER > 1) j.add_parts<D, 4>(ml, x, grp, TOGETHER, a.parts);
    else if (a.parts <= 2) j.add_parts<D, 2>(ml, x, 0, 1, a.parts);
    else j.add_parts<D, 8>(ml, x, 0, 1, a.parts);
  }
  if constexpr (TOGETHER > 1) {
    __shared__ __attribute__((aligned(16))) f32x4 so[256];
    __shared__ f32x2 sml[256];
    so[threadIdx.x] = j.o;
    sml[threadIdx.x] = f32x2{j.top, j.sum()};
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int k = 1; k < TOGETHER; ++k) j.add(sml[threadIdx.x + k * PER], so[threadIdx.x + k * PER]);
  }
  if (there) j.store(a.out + (int64_t)t * a.out_stride + (int64_t)h * D + d);
}

struct Plan {
  int ns, pre_tiles, pre_split, pre_keys, pre_few, own_tiles, own_split, own_keys, own_few;
};

int up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// The prefix's cut for ns groups of slots a wave, and what it takes in us: two workgroups a compute unit and all of them at once, so that
// no second round has to be waited for (one key head, 1584 slots behind 7990 positions: 525 workgroups 45 us, 500 33), each of 256 keys or
// more. A tile of 64 keys takes 2.0 us with one group (64 slots a workgroup), 3.3 with two (128) while two workgroups share a compute
// unit; the partial results are written and read once, at 4.5 TB/s. Two groups halve what LDS is read for, but twice the cuts fill the
// chip with them (the calls, with one and two: 128 rows of 64 heads in 8 groups behind 16381 positions 130 us and 115, 128 rows of 32 key
// heads behind 8000 66 and 75, one key head as above 27 and 29). Heads of 64 take one: three of their workgroups share a compute unit
// (128 rows of 32 heads in 8 groups behind 16000 37 us, with two 41). fp8 rows take as long either way (their conversion is the tile's)
// and heads of 256 have no registers for two.
double cut_prefix(Plan& p, int ns, int64_t slots, int nkv, int D, int P) {
  const int tile = tile_keys(D);
  p.ns = ns;
  p.pre_tiles = up(slots, 64 * ns);
  const int64_t pairs = (int64_t)p.pre_tiles * nkv;
  const int runs = (int)std::max<int64_t>(1, std::min<int64_t>(512 / pairs, up(P, 256)));
  p.pre_keys = up(up(P, runs), tile) * tile;
  p.pre_split = up(P, p.pre_keys);
  const double rounds = std::max(1.0, (double)pairs * p.pre_split / 512);
  return rounds * p.pre_keys / 64 * (ns == 2 ? 3.3 : 2.0) + 2.0 * slots * nkv * (D + 2) * 4 * p.pre_split / 4.5e6;
}

// Which form takes what (the calls among others; heads of 128 as 32 in 8 groups where nothing else is said):
//  up to 16 slots in the whole batch: both parts by keys (one row behind 2000 positions 9.4 us from a captured graph, the prefix by rows
//   11.5, either 15 with the host's steps; 2 rows behind 16000 19.5 and 21.7, of fp8 16.9 and 21.0; 4 rows behind 30000 27.9 and 27.0, of fp8
//   22.4 and 25.8).
//  own parts by keys in a launch of their own, after the prefix's, where up to 16 slots a sequence and at least 512 (sequence, key
//   head) pairs fill the chip: each pair is then one workgroup's, and no third launch joins (64 rows of 32 key heads behind 2048 39.7 us,
//   in one launch with the prefix by rows 42.4, of fp8 34.9 and 43.4; 128 rows of 64 heads in 8 behind 16381 119 and 122, of fp8 150 and 149; 100
//   rows behind 2000 29.4 and 29.6, of fp8 29.0 and 32.6).
//   Not where own parts are long beside the prefix, which then fill its gaps (64 rows of 8, 2000 and up to 3000 positions: 117 us apart,
//   112 together), and not for heads of 64 (equal, or 69 together and 74) and of 256 (30 and 40: by keys two workgroups share a compute
//   unit, not four).
//  everything else by rows in one launch (fewer pairs: 60 rows of one key head behind 4000 18.0 us, apart 25.8; 33 rows of 48 heads on
//   one key head behind 7990 26.1 and 31.7).
//  no prefix: own parts of up to 16 slots by keys (64 rows of up to 500 19.5 us, by rows 19.9; fp8 17.4 and 23.2).
// Own parts are cut until there are 256 workgroups by rows beside the prefix's (20 rows of 8 key heads with 4 tokens each 24.1 us, with 512
// 27.6, with 2048 33.3) and 512 by keys (2 rows of 8 with up to 8000 positions 15.5, with 256 19.6, with 2048 15.4).
Plan shared_plan(int T, int B, int nkv, int G, int D, int P, int max_qlen, int max_own, bool kv8) {
  Plan p;
  const int64_t slots = (int64_t)T * G;
  const int tile = tile_keys(D);
  p.pre_few = slots <= 16;
  p.ns = 1;
  p.pre_tiles = 1;
  p.pre_split = 0;
  p.pre_keys = tile;
  if (P > 0 && p.pre_few) {  // 32 keys a wave at a time, as many workgroups as there are keys for up to the chip's
    const int runs = std::max(1, std::min(512 / nkv, up(P, 128)));
    p.pre_keys = up(up(P, runs), 128) * 128;
    p.pre_split = up(P, p.pre_keys);
  } else if (P > 0) {
    const double one = cut_prefix(p, 1, slots, nkv, D, P);
    Plan two = p;
    if (!kv8 && D == 128 && slots > 64 && cut_prefix(two, 2, slots, nkv, D, P) < one) p = two;
  }
  const int64_t portion = (int64_t)std::max(1, max_qlen) * G;
  p.own_few = p.pre_few || (portion <= 16 && (P == 0 || (D == 128 && (int64_t)B * nkv >= 512 && max_own <= P / 2)));
  p.own_tiles = up(portion, p.own_few ? 16 : 64 * p.ns);
  const int unit = p.own_few ? 128 : tile;
  const int runs = up(p.own_few ? 512 : 256, (int64_t)B * nkv * p.own_tiles);
  const int want = std::max(1, std::min(runs, up(std::max(1, max_own), 2 * unit)));
  p.own_keys = up(up(std::max(1, max_own), want), unit) * unit;
  p.own_split = up(std::max(1, max_own), p.own_keys);
  return p;
}

}  // namespace

int attn_shared_parts(int T, int B, int nh, int nkv, int D, int P, int max_qlen, int max_own, bool kv8) {
  const Plan p = shared_plan(T, B, nkv, nh / nkv, D, P, max_qlen, max_own, kv8);
  return p.pre_split + p.own_split;
}

void launch_attn_shared(const void* q, int64_t q_stride, const void* kc, const void* vc, int pages, const void* prefix_table, int P,
                        const void* bt, int64_t bt_stride, int bt_width, const void* cu, const void* ctx, void* out, int64_t out_stride,
                        void* ws, int parts, int T, int B, int nh, int nkv, int D, int bs, int max_qlen, int max_own, float scale,
                        bool kv8, hipStream_t st) {
  if (nkv <= 0 || nh % nkv) throw std::runtime_error("attn_shared: nh must be a multiple of nkv");
  if (T == 0 || B == 0) return;
  const Plan p = shared_plan(T, B, nkv, nh / nkv, D, P, max_qlen, max_own, kv8);
  if (p.pre_split + p.own_split != parts) throw std::runtime_error("attn_shared: the workspace was made for another call");
  SharedAttn a;
  a.q = (const bf16_t*)q;
  a.q_stride = q_stride;
  a.kc = kc;
  a.vc = vc;
  a.prefix_table = (const int*)prefix_table;
  a.bt = (const int*)bt;
  a.bt_stride = bt_stride;
  a.cu = (const int*)cu;
  a.ctx = (const int*)ctx;
  a.po = (float*)ws;
  a.pml = a.po + (int64_t)T * nh * parts * D;
  a.T = T;
  a.B = B;
  a.nh = nh;
  a.nkv = nkv;
  a.G = nh / nkv;
  a.bs = bs;
  a.shift = __builtin_ctz(bs);
  const int64_t page_bytes = (int64_t)nkv * bs * (kv8 ? D + kTail : 2 * D);
  if (page_bytes > INT_MAX) throw std::invalid_argument("attn_shared: pages of 2 GiB and more");
  a.page_bytes = (unsigned)page_bytes;
  a.pages = pages;
  a.P = P;
  a.own_cap = (int)std::min<int64_t>((int64_t)bt_width * bs, INT_MAX / 2);
  a.pre_tiles = p.pre_tiles;
  a.pre_split = p.pre_split;
  a.pre_keys = p.pre_keys;
  a.pre_few = p.pre_few;
  a.own_tiles = p.own_tiles;
  a.own_split = p.own_split;
  a.own_keys = p.own_keys;
  a.own_few = p.own_few;
  a.scale_log2 = scale * kLog2eS;
  a.out = (bf16_t*)out;
  a.out_stride = out_stride;
  a.parts = parts;
  a.finish = 0;
  const int64_t pre = (int64_t)p.pre_tiles * nkv * p.pre_split, own = (int64_t)B * nkv * p.own_tiles * p.own_split;
  const int together = parts > 12 ? 1024 / D : 1;  // (see the join kernel)
  const int64_t join = ((int64_t)T * nh * (D / 4) * together + 255) / 256;
  constexpr int64_t kMostGroups = UINT32_MAX / 256;  // (a launch has fewer than 2^32 threads)
  if (pre + own > kMostGroups || join > kMostGroups || (int64_t)T * (nh / nkv) > INT_MAX / 2)
    throw std::invalid_argument("attn_shared: too many rows");
  // one launch for both parts where they take the same form; else the own parts', which follow, join the prefix's results themselves
  // (each is one workgroup's: there are 512 pairs or more)
  const bool apart = p.own_few && !p.pre_few && pre > 0;
  if (apart && p.own_split != 1) throw std::runtime_error("attn_shared: an own part of several workgroups cannot join the prefix's");
  const bool by16 = bs >= 16 && (bs & (bs - 1)) == 0;
#define SA(D_, KV8_, NS_, F_, N_)                                                                 \
  do {                                                                                            \
    if (by16) attn_shared_kernel<D_, KV8_, NS_, F_, true><<<(unsigned)(N_), 256, 0, st>>>(a); \
    else attn_shared_kernel<D_, KV8_, NS_, F_, false><<<(unsigned)(N_), 256, 0, st>>>(a);         \
    HIP_CHECK_LAUNCH();                                                                           \
  } while (0)
#define SF(D_, KV8_, NS_)                            \
  do {                                               \
    a.pre_items = (int)pre;                          \
    if (apart) {                                     \
      SA(D_, KV8_, NS_, ROWS, pre);                  \
      a.pre_items = 0;                               \
      a.finish = 1;                                  \
      SA(D_, KV8_, 1, KEYS, own);                    \
    } else if (p.own_few) SA(D_, KV8_, 1, KEYS, pre + own); \
    else SA(D_, KV8_, NS_, ROWS, pre + own);         \
  } while (0)
#define SD(D_)                                                                                    \
  do {                                                                                            \
    constexpr int TWO = D_ == 128 ? 2 : 1; /* (no such kernel for other heads) */                 \
    if (kv8) SF(D_, true, 1);                                                                     \
    else if (p.ns == 2) SF(D_, false, TWO);                                                       \
    else SF(D_, false, 1);                                                                        \
    if (a.finish) break;                                                                          \
    if (together > 1) attn_shared_join_kernel<D_, 1024 / D_><<<(unsigned)join, 256, 0, st>>>(a);  \
    else attn_shared_join_kernel<D_, 1><<<(unsigned)join, 256, 0, st>>>(a);                       \
  } while (0)
  switch (D) {
    case 64: SD(64); break;
    case 128: SD(128); break;
    case 256: SD(256); break;
    default: throw std::runtime_error("attn_shared: head_dim must be 64, 128 or 256");
  }
#undef SD
#undef SF
#undef SA
  HIP_CHECK_LAUNCH();
}
