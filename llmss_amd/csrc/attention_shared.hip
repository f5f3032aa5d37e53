// Attention of a batch whose sequences share a long prefix: the prefix's keys and values are read once for all rows, not once
// a sequence.
//
// Row t (sequence b, position p) attends positions 0 .. p. The first P positions of every context lie in the pages of ONE
// table, the others in pages of the sequence's own:
//   s_j = scale q . k_j,   o = sum_j exp(s_j - M) v_j / sum_j exp(s_j - M)
// A softmax over two sets of keys is joined from the sets' own maxima, sums and unnormalised outputs:
//   M = max_i m_i,   o = sum_i e^(m_i - M) o_i / sum_i e^(m_i - M) l_i
// so one launch has workgroups for the prefix (all rows of the batch against a run of its keys) and workgroups for the own
// parts, each leaving (m, l, o) in fp32, and a second launch joins them. The prefix's share is bound by matrix instructions from
// some 200 rows a key head on, the own parts by memory: in one launch they fill each other's gaps.
//
// Both kinds take (row, query head of the key head's group) pairs as "slots", the columns of swapped products
//   S^T[key][slot] = K Q^T,   O^T[dim][slot] += V^T P^T
// so that a lane owns a slot's softmax (lane & 15) and P^T is made in the registers that the second product takes it from.
// Two forms of a workgroup:
//  rows by waves - many slots: each wave has 16 NS slots of its own, all four share tiles of keys and values in LDS (two places:
//    the next tile is fetched while one is computed).
//  keys by waves - up to 16 slots (single tokens' own parts, a few rows behind a prefix): the waves walk different keys of the same
//    slots, without a barrier, keys straight into registers, and meet at the end. One slot of 16 may be real: 64 keys of 128
//    numbers cost a wave about 1000 cycles, memory takes 3500 to bring a compute unit's share of them.
//
// Keys that a slot does not see weigh nothing whatever lies there: scores are replaced, not multiplied; rows past the last visible
// key are never loaded (a visible one is, again); and where a tile that is masked for some slots holds values that are not finite,
// they are kept from the slots that do not see them (see `add_values`).
// fp8 cache rows: e4m3 numbers are exact in bf16, a row's scale multiplies its score and its weight.
#include "common.h"

#include <type_traits>

namespace {

constexpr float kLog2eS = 1.4426950408889634f;
constexpr float kFloor = -1.0e30f;  // a maximum before any key was seen
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
  int T, B, nh, nkv, G, bs, shift, pages, P, own_cap;  // shift: log2 of bs where it is a power of two, or -1
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

// The cache row of a key: pages of 16 m positions are asked once for 16 keys, by a scalar load.
template <bool BY16>
struct Rows {
  const SharedAttn& a;
  const Item& it;
  int64_t row_size;  // of one cache row, in cache elements
  __device__ __forceinline__ int64_t in_page(int k) const {
    const int i = a.shift >= 0 ? k >> a.shift : k / a.bs;
    const unsigned p = (unsigned)it.table[i];
    return (((int64_t)(p < (unsigned)a.pages ? p : 0) * a.nkv + it.kvh) * a.bs + (k - i * a.bs)) * row_size;
  }
  // key k16 + r, at most the last one; k16 the same in every lane and a multiple of 16, r < 16
  __device__ __forceinline__ int64_t at(int k16, int r) const {
    const int last = it.stop - 1;
    if constexpr (BY16) {
      const int base = __builtin_amdgcn_readfirstlane(min(k16, last & ~15));
      return in_page(base) + min(r, last - base) * row_size;
    } else {
      return in_page(min(k16 + r, last));
    }
  }
};

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

// Scores of 16 KT keys and NS groups of slots become weights: the running maximum of a slot moves only where its own has grown by
// more than 8 (weights stay below 2^8), so most tiles exchange nothing between lanes and rescale nothing. Weights are rounded to
// bf16 for the second product (half a step of 2^-8, as any bf16 operand); their sum is taken of the rounded ones, by a product with
// ones, so that they add up to 1 as they are used. lim: keys [.., lim) are seen, counted from the tile's first.
template <int D, int KT, int NS, bool MASK>
__device__ __forceinline__ void soften(f32x4 (&s)[NS][KT], const int (&lim)[NS], float scale_log2, int g, float (&m)[NS],
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
  if (__ballot(grew)) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const float top = xor32_max(xor16_max(mx[n]));
      const bool up = top > m[n] + 8.f;
      const float alpha = up ? __builtin_amdgcn_exp2f(m[n] - top) : 1.f;
      if (up) m[n] = top;
#pragma unroll
      for (int i = 0; i < 4; ++i) lsum[n][i] *= alpha;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] *= alpha;
    }
  }
  const s16x8 ones = {0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80};
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const float nm = -m[n];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        pf[n][kt >> 1][(kt & 1) * 4 + i] = (short)f2bf(__builtin_amdgcn_exp2f(fmaf(s[n][kt][i], scale_log2, nm)));
#pragma unroll
    for (int k = 0; k < KT / 2; ++k) lsum[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[n][k], lsum[n], 0, 0, 0);
    if (vscale) {  // (fp8 rows: the second rounding of a weight, to half a step again)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(vscale + kt * 16 + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // a key that weighs nothing is not seen, or as good as that: its scale may be anything
          const short p = pf[n][kt >> 1][(kt & 1) * 4 + i];
          pf[n][kt >> 1][(kt & 1) * 4 + i] = p ? (short)f2bf(__builtin_amdgcn_exp2f(fmaf(s[n][kt][i], scale_log2, nm)) * v[i]) : (short)0;
        }
      }
    }
  }
}

// O^T += V^T P^T. Where a tile that is masked for some slots holds values that are not finite, the products would give them to every
// slot (0 times such a value is NaN): there the weights go through `own_lds` (16 slots of 16 KT keys, the wave's own) and each slot
// takes the keys that it sees one after the other. Rare, so kept small.
template <int D, int KT, int NS, bool MASK>
__device__ __forceinline__ void add_values(const char* img, bf16_t* own_lds, const int (&lim)[NS], int g, int li,
                                           const s16x8 (&pf)[NS][KT / 2], f32x4 (&o)[NS][D / 16]) {
  if constexpr (MASK) {
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
      const s16x8 vf = v_fragment<D>(img, 32 * k, dt, g, li);
#pragma unroll
      for (int n = 0; n < NS; ++n) o[n][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n][k], o[n][dt], 0, 0, 0);
    }
}

template <int D>
__device__ __forceinline__ void leave(const SharedAttn& a, const Item& it, int slot, int g, const f32x4 (&o)[D / 16], float m, float l) {
  const int64_t pi = ((int64_t)(it.row0 + slot / a.G) * a.nh + it.kvh * a.G + slot % a.G) * (a.pre_split + a.own_split) + it.part;
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
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  int slot[NS], lim[NS];
  int lo = INT_MAX, hi = 0;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    slot[n] = it.first + (w * NS + n) * 16 + li;
    lim[n] = INT_MAX;  // (a slot behind the last: of no consequence, and no reason for a mask)
    if (slot[n] < it.slots) {
      lim[n] = slot_limit(a, it, slot[n]);
      lo = min(lo, lim[n]);
      hi = max(hi, lim[n]);
    }
  }
  const int wave_lo = wave_min(lo), wave_hi = wave_max(hi);
  __syncthreads();  // (a workgroup may have had an item before)
  if (lane == 0) red[w] = wave_hi;
  __syncthreads();
  it.stop = min(it.stop, max(max(red[0], red[1]), max(red[2], red[3])));

  f32x4 o[NS][D / 16], lsum[NS];
  float m[NS];
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
    const Rows<BY16> rows{a, it, KV8 ? D + kTail : D};
    const int ntiles = (it.stop - it.begin + BKV - 1) / BKV;

    // bf16: 16 bytes a lane straight into LDS, a wave's instruction covers RPI rows
    constexpr int RPI = 64 / CH, LPW = BKV / RPI / 4;
    // fp8: 16 numbers a thread and piece, through registers
    constexpr int PIECES = BKV * (D / 16) / 256;
    u32x4 k8[KV8 ? PIECES : 1], v8[KV8 ? PIECES : 1];
    float sc = 0.f;
    auto fetch = [&](int j) {
      const int kv0 = it.begin + j * BKV;
      char* sk = smem + (j & 1) * 2 * TILE;
      if constexpr (KV8) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int c = threadIdx.x + i * 256, r = c / (D / 16);
          // (16 rows of 4, 8 or 16 pieces: a wave's rows lie within one run of 16)
          const int64_t off = rows.at(kv0 + __builtin_amdgcn_readfirstlane(r & ~15), r & 15) + (c % (D / 16)) * 16;
          k8[i] = *reinterpret_cast<const u32x4*>((const unsigned char*)a.kc + off);
          v8[i] = *reinterpret_cast<const u32x4*>((const unsigned char*)a.vc + off);
        }
        if (threadIdx.x < 2 * BKV) {
          const Rows<false> one{a, it, D + kTail};
          const int64_t off = one.at(kv0, threadIdx.x % BKV) + D;
          sc = *reinterpret_cast<const float*>((const unsigned char*)(threadIdx.x < BKV ? a.kc : a.vc) + off);
        }
      } else {
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
          const int inst = i * 4 + w, r = inst * RPI + lane / CH;
          const int64_t off = rows.at(kv0 + (inst * RPI & ~15), r & 15) + swz<D>(lane % CH, r) * 8;
          __builtin_amdgcn_global_load_lds((const void*)((const bf16_t*)a.kc + off), (LDS_AS void*)(sk + inst * 1024), 16, 0, 0);
          __builtin_amdgcn_global_load_lds((const void*)((const bf16_t*)a.vc + off), (LDS_AS void*)(sk + TILE + inst * 1024), 16, 0, 0);
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
      if (threadIdx.x < 2 * BKV) scales[(j & 1) * 2 * BKV + threadIdx.x] = sc;
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
      __builtin_amdgcn_sched_barrier(0);
      const float* vs = nullptr;
      if constexpr (KV8) {
        const float* ks_ = scales + (j & 1) * 2 * BKV;
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
      soften<D, KT, NS, MASK>(s, left, a.scale_log2, g, m, lsum, o, pf, vs);
      add_values<D, KT, NS, MASK>(sk + TILE, apart + w * 16 * BKV, left, g, li, pf, o);
    };
    // tiles that every slot of the wave sees whole come first, in a loop without masks
    const int whole = min(max(0, (min(wave_lo, it.stop) - it.begin) / BKV), ntiles);
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
  for (int n = 0; n < NS; ++n)
    if (slot[n] < it.slots) leave<D>(a, it, slot[n], g, o[n], m[n], lsum[n][0]);
}

// ------------------------------------------------------------------------------------------------------ keys by waves
// A wave takes every fourth run of 32 keys. Keys come straight into the first product's registers (fp8: 16 numbers a lane, so that
// a pair of products shares them: dims 64 m + 16 g + 8 h of the query's row stand beside them), values through LDS places of
// the wave's own.
template <int D, bool KV8, bool BY16>
__device__ __forceinline__ void keys_by_waves(const SharedAttn& a, Item it, char* smem, float* scales, bf16_t* apart) {
  constexpr int KT = 2, BK = 32, CH = D / 8;
  constexpr int PLACES = D == 256 ? 1 : 2;  // of values: wide heads' would take all of LDS
  constexpr int TILE = BK * D * 2;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int slot = it.first + li;
  const bool real = slot < it.slots;
  int lim[1] = {INT_MAX};
  if (real) lim[0] = slot_limit(a, it, slot);
  const int lo = wave_min(lim[0]), hi = wave_max(real ? lim[0] : 0);
  it.stop = min(it.stop, hi);

  f32x4 o[1][D / 16], lsum[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
  float m[1] = {kFloor};
#pragma unroll
  for (int i = 0; i < D / 16; ++i) o[0][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  __syncthreads();  // (a workgroup may have had an item before: the places below are free)
  if (it.stop > it.begin) {
    s16x8 qf[D / 32];
    {
      const int sl = min(slot, it.slots - 1);
      const bf16_t* qp = a.q + (int64_t)(it.row0 + sl / a.G) * a.q_stride + (int64_t)(it.kvh * a.G + sl % a.G) * D;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
        qf[ks] = *reinterpret_cast<const s16x8*>(qp + (KV8 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g));
    }
    const Rows<BY16> rows{a, it, KV8 ? D + kTail : D};
    char* const mine = smem + w * PLACES * TILE;
    float* const fac = scales + w * 2 * BK;  // (fp8) scales of the keys, of the values
    s16x8 kf[KT][KV8 ? 1 : D / 32];
    u32x4 k8[KT][KV8 ? D / 64 : 1];
    constexpr int RPI = 64 / CH, INS = BK / RPI, PIECES = BK * (D / 16) / 64;
    u32x4 v8[KV8 ? PIECES : 1];
    float sc = 0.f;
    auto keys = [&](int kv0) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const int64_t off = rows.at(kv0 + kt * 16, li);
        if constexpr (KV8) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c) k8[kt][c] = *reinterpret_cast<const u32x4*>((const unsigned char*)a.kc + off + 64 * c + 16 * g);
        } else {
#pragma unroll
          for (int ks = 0; ks < D / 32; ++ks) kf[kt][ks] = *reinterpret_cast<const s16x8*>((const bf16_t*)a.kc + off + 32 * ks + 8 * g);
        }
      }
      if constexpr (KV8) {
        const Rows<false> one{a, it, D + kTail};
        sc = *reinterpret_cast<const float*>((const unsigned char*)(lane < BK ? a.kc : a.vc) + one.at(kv0, lane % BK) + D);
      }
    };
    auto values = [&](int kv0, int place) {
      if constexpr (KV8) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int c = lane + i * 64, r = c / (D / 16);
          const int64_t off = rows.at(kv0 + __builtin_amdgcn_readfirstlane(r & ~15), r & 15) + (c % (D / 16)) * 16;
          v8[i] = *reinterpret_cast<const u32x4*>((const unsigned char*)a.vc + off);
        }
      } else {
#pragma unroll
        for (int i = 0; i < INS; ++i) {
          const int r = i * RPI + lane / CH;
          const int64_t off = rows.at(kv0 + (i * RPI & ~15), r & 15) + swz<D>(lane % CH, r) * 8;
          __builtin_amdgcn_global_load_lds((const void*)((const bf16_t*)a.vc + off), (LDS_AS void*)(mine + place * TILE + i * 1024), 16, 0, 0);
        }
      }
    };
    const int step = 4 * BK;
    int kv0 = it.begin + w * BK, place = 0;
    if (kv0 < it.stop) {
      keys(kv0);
      values(kv0, 0);
    }
    for (; kv0 < it.stop; kv0 += step) {
      const int nx = kv0 + step;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this run's keys and values
      char* img = mine + place * TILE;
      if constexpr (KV8) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int c = lane + i * 64, r = c / (D / 16), c0 = (c % (D / 16)) * 2;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<s16x8*>(img + r * D * 2 + (swz<D>(c0 + h, r) << 4)) = fp8_to_bf16(v8[i][2 * h], v8[i][2 * h + 1]);
        }
        fac[lane] = sc;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      } else if constexpr (PLACES == 2) {
        if (nx < it.stop) values(nx, place ^ 1);
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
      if (nx < it.stop) {
        keys(nx);
        if constexpr (KV8) values(nx, 0);
      }
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
      if (kv0 + BK <= min(lo, it.stop)) {
        soften<D, KT, 1, false>(s, left, a.scale_log2, g, m, lsum, o, pf, vs);
        add_values<D, KT, 1, false>(img, apart + w * 16 * BK, left, g, li, pf, o);
      } else {
        soften<D, KT, 1, true>(s, left, a.scale_log2, g, m, lsum, o, pf, vs);
        add_values<D, KT, 1, true>(img, apart + w * 16 * BK, left, g, li, pf, o);
      }
      if constexpr (!KV8 && PLACES == 1) {
        if (nx < it.stop) values(nx, 0);  // (the reads of this run's were waited for by the products)
      }
      if constexpr (PLACES == 2) place ^= 1;
    }
  }
  // the waves meet: outputs [wave][slot][D] and (m, l)
  __syncthreads();
  float* const so = reinterpret_cast<float*>(smem);
  constexpr int LDO = D + 4;
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<f32x4*>(so + (w * 16 + li) * LDO + dt * 16 + 4 * g) = o[0][dt];
  if (g == 0) {
    scales[(w * 16 + li) * 2] = m[0];
    scales[(w * 16 + li) * 2 + 1] = lsum[0][0];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 16 * (D / 4); c += 256) {
    const int sl = c / (D / 4), d4 = c % (D / 4);
    if (it.first + sl >= it.slots) continue;
    float top = kFloor, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, scales[(i * 16 + sl) * 2]);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float li_ = scales[(i * 16 + sl) * 2 + 1];
      if (li_ == 0.f) continue;  // (this wave saw none of its keys)
      const float f = __builtin_amdgcn_exp2f(scales[(i * 16 + sl) * 2] - top);
      const f32x4 x = *reinterpret_cast<const f32x4*>(so + (i * 16 + sl) * LDO + d4 * 4);
      l += li_ * f;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += x[e] * f;
    }
    const int s_ = it.first + sl;
    const int64_t pi = ((int64_t)(it.row0 + s_ / a.G) * a.nh + it.kvh * a.G + s_ % a.G) * (a.pre_split + a.own_split) + it.part;
    *reinterpret_cast<f32x4*>(a.po + pi * D + d4 * 4) = sum;
    if (d4 == 0) {
      a.pml[pi * 2] = top;
      a.pml[pi * 2 + 1] = l;
    }
  }
}

// FORMS: which forms the items take, by waves' rows (r) or keys (k): the prefix's and the own parts'.
enum Forms { RR = 0, RK = 1, KK = 2 };

template <int D, bool KV8, int NS, int FORMS, bool BY16>
__global__ __launch_bounds__(256, 2) void attn_shared_kernel(const SharedAttn a) {
  constexpr int ROWS = 2 * 2 * tile_keys(D) * D * 2;                      // tiles of the first form
  constexpr int KEYS = 4 * (D == 256 ? 1 : 2) * 32 * D * 2;                // places of values of the second
  constexpr int MEET = 4 * 16 * (D + 4) * 4;                               // its outputs
  constexpr int SECOND = KEYS > MEET ? KEYS : MEET;
  constexpr int SIZE = FORMS == RR ? ROWS : FORMS == KK ? SECOND : ROWS > SECOND ? ROWS : SECOND;
  __shared__ __attribute__((aligned(16))) char smem[SIZE];
  __shared__ __attribute__((aligned(16))) float scales[4 * 2 * 64];
  __shared__ __attribute__((aligned(16))) bf16_t apart[4 * 16 * (FORMS == KK ? 32 : tile_keys(D))];
  __shared__ int red[4];
  Item it;
  int id = blockIdx.x;
  int tile, tiles, per;
  if (id < a.pre_items) {  // (key head, run of keys, tile of slots), the tiles of a run on one die
    id = xcd_remap(id, a.pre_items);
    const int run = id / a.pre_tiles;
    tile = id % a.pre_tiles;
    tiles = INT_MAX / 1024;
    per = FORMS == KK ? 16 : 64 * NS;
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
    per = FORMS == RR ? 64 * NS : 16;
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
    if constexpr (FORMS == RR) rows_by_waves<D, KV8, NS, BY16>(a, it, smem, scales, apart, red);
    else if constexpr (FORMS == KK) keys_by_waves<D, KV8, BY16>(a, it, smem, scales, apart);
    else if (it.own) keys_by_waves<D, KV8, BY16>(a, it, smem, scales, apart);
    else rows_by_waves<D, KV8, NS, BY16>(a, it, smem, scales, apart, red);
    if (!it.own) break;
  }
}

template <int D>
__global__ __launch_bounds__(256) void attn_shared_join_kernel(const SharedAttn a, bf16_t* __restrict__ out, int64_t out_stride) {
  constexpr int PER = D / 4;  // threads of a (row, head)
  const int np = a.pre_split + a.own_split;
  const int64_t i = (int64_t)blockIdx.x * (256 / PER) + threadIdx.x / PER;
  const int d = threadIdx.x % PER * 4;
  if (i >= (int64_t)a.T * a.nh) return;
  const int t = i / a.nh, h = i % a.nh;
  if (seq_of(a, t) < 0) return;  // a row of no sequence stays as it was
  const float* ml = a.pml + i * np * 2;
  const float* po = a.po + i * np * D + d;
  float top = kFloor, l = 0.f;
  for (int p = 0; p < np; ++p) top = fmaxf(top, ml[2 * p]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < np; ++p) {
    const float lp = ml[2 * p + 1];
    if (lp == 0.f) continue;  // (a part without a visible key)
    const float f = __builtin_amdgcn_exp2f(ml[2 * p] - top);
    const f32x4 x = *reinterpret_cast<const f32x4*>(po + (int64_t)p * D);
    l += lp * f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += x[e] * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  u16x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = f2bf(o[e] * inv);
  *reinterpret_cast<u16x4*>(out + (int64_t)t * out_stride + (int64_t)h * D + d) = r;
}

struct Plan {
  int ns, pre_tiles, pre_split, pre_keys, pre_few, own_tiles, own_split, own_keys, own_few;
};

int up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

Plan shared_plan(int T, int B, int nkv, int G, int D, int P, int max_qlen, int max_own) {
  Plan p;
  p.ns = 1;
  const int per = 64 * p.ns;
  const int64_t slots = (int64_t)T * G;
  p.pre_few = slots <= 16;
  p.pre_tiles = p.pre_few ? 1 : up(slots, per);
  const int tile = tile_keys(D);
  if (P > 0) {
    const int unit = p.pre_few ? 128 : tile;  // keys that a workgroup takes at a time
    const int runs = up(512, (int64_t)p.pre_tiles * nkv);
    const int want = std::max(1, std::min(runs, up(P, 2 * unit)));
    p.pre_keys = up(up(P, want), unit) * unit;
    p.pre_split = up(P, p.pre_keys);
  } else {
    p.pre_keys = tile;
    p.pre_split = 0;
  }
  const int64_t portion = (int64_t)std::max(1, max_qlen) * G;
  p.own_few = p.pre_few || portion <= 16 || max_qlen == 1;
  p.own_tiles = up(portion, p.own_few ? 16 : per);
  const int unit = p.own_few ? 128 : tile;
  const int runs = up(512, (int64_t)B * nkv * p.own_tiles);
  const int want = std::max(1, std::min(runs, up(std::max(1, max_own), 2 * unit)));
  p.own_keys = up(up(std::max(1, max_own), want), unit) * unit;
  p.own_split = up(std::max(1, max_own), p.own_keys);
  return p;
}

}  // namespace

int attn_shared_parts(int T, int B, int nh, int nkv, int D, int P, int max_qlen, int max_own) {
  const Plan p = shared_plan(T, B, nkv, nh / nkv, D, P, max_qlen, max_own);
  return p.pre_split + p.own_split;
}

void launch_attn_shared(const void* q, int64_t q_stride, const void* kc, const void* vc, int pages, const void* prefix_table, int P,
                        const void* bt, int64_t bt_stride, int bt_width, const void* cu, const void* ctx, void* out, int64_t out_stride,
                        void* ws, int parts, int T, int B, int nh, int nkv, int D, int bs, int max_qlen, int max_own, float scale,
                        bool kv8, hipStream_t st) {
  if (nkv <= 0 || nh % nkv) throw std::runtime_error("attn_shared: nh must be a multiple of nkv");
  if (T == 0 || B == 0) return;
  const Plan p = shared_plan(T, B, nkv, nh / nkv, D, P, max_qlen, max_own);
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
  a.shift = (bs & (bs - 1)) == 0 ? __builtin_ctz(bs) : -1;
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
  const int64_t pre = (int64_t)p.pre_tiles * nkv * p.pre_split, own = (int64_t)B * nkv * p.own_tiles * p.own_split;
  const int64_t join = ((int64_t)T * nh * (D / 4) + 255) / 256;
  if (pre + own > INT_MAX || join > INT_MAX || (int64_t)T * (nh / nkv) > INT_MAX / 2) throw std::runtime_error("attn_shared: too many rows");
  a.pre_items = (int)pre;
  const unsigned grid = (unsigned)(pre + own);
  const int forms = p.pre_few ? KK : p.own_few ? RK : RR;
#define SA(D_, KV8_, NS_, F_, BY_) attn_shared_kernel<D_, KV8_, NS_, F_, BY_><<<grid, 256, 0, st>>>(a)
#define SB(D_, KV8_, NS_, F_)                  \
  do {                                         \
    if (bs % 16 == 0) SA(D_, KV8_, NS_, F_, true); \
    else SA(D_, KV8_, NS_, F_, false);         \
  } while (0)
#define SF(D_, KV8_, NS_)                      \
  do {                                         \
    if (forms == RR) SB(D_, KV8_, NS_, RR);    \
    else if (forms == RK) SB(D_, KV8_, NS_, RK); \
    else SB(D_, KV8_, 1, KK);                  \
  } while (0)
#define SD(D_)                                                                                    \
  do {                                                                                            \
    if (kv8) SF(D_, true, 1);                                                                     \
    else SF(D_, false, 1);                                                                        \
    HIP_CHECK_LAUNCH();                                                                           \
    attn_shared_join_kernel<D_><<<(unsigned)join, 256, 0, st>>>(a, (bf16_t*)out, out_stride);     \
  } while (0)
  switch (D) {
    case 64: SD(64); break;
    case 128: SD(128); break;
    case 256: SD(256); break;
    default: throw std::runtime_error("attn_shared: head_dim must be 64, 128 or 256");
  }
#undef SD
#undef SF
#undef SB
#undef SA
  HIP_CHECK_LAUNCH();
}
