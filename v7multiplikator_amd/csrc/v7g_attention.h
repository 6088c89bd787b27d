// v7g_attention.h -- what the attention kernels share: their arguments, how the work is cut into units, and the
// two-part binary16 form of f32 operands.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <utility>

#include "v7g_device.h"

namespace v7g {

// One attention call.  Rows are (token, query head of the group) pairs: the G query heads that share a KV head lie
// next to each other in a token, so row r of a sequence and KV head hk is head hk*G + r%G of its token r/G, and a
// tile of rows reads each K/V row once for all of them.
struct AttnArgs {
  const float *q;
  float *out;
  long long q_stride, out_stride;  // f32 elements between tokens
  const uint16_t *k, *v;           // binary16; paged: page 0
  long long k_stride, v_stride;    // binary16 elements between tokens (paged: within a page)
  long long page_stride;           // paged: binary16 elements between pages
  const int32_t *table;            // paged: [n_seqs, table_width] page of each page_size tokens
  const int32_t *ctx;              // paged: tokens in the cache before this call's
  const int32_t *cu_q;             // [n_seqs + 1] first token of each sequence, or nullptr: token b is sequence b
  const int32_t *cu_k;             // packed: the same of the K/V rows
  const int64_t *mask;             // paged: per token mask_words words, bit j = attends to the sequence's new token j
  int mask_words;                  // 0: causal
  int table_width, page_shift, n_pages;
  int n_seqs, n_tokens, n_kv;  // n_kv: packed K/V rows
  int n_kv_heads, group;
  float scale_log2;  // the score scale times log2(e)
  int split_target;  // units per KV head aimed at; 0: no tile is split along the keys
  int units;         // per KV head, at most: what the grid and the partial results have room for
  float *part_o;     // [unit, KV head, tile row, head_dim]
  float *part_ml;    // [unit, KV head, tile row, 2]: running maximum (log2 domain) and sum
};

constexpr int kAttnRowShift = 4;    // 16 rows make a tile of the few-row kernel
constexpr int kAttnTileShift = 7;   // 128 rows one of the many-row kernel
constexpr int kAttnTileRows = 1 << kAttnTileShift;
constexpr int kAttnTileDims = 256;  // the many-row kernel's widest head
constexpr int kAttnUnits = 1024;    // units that fill the chip: four workgroups for each of 256 compute units
constexpr int kAttnMinChunk = 256;  // keys; shorter pieces cost more in joining than they save

// A sequence's tokens and keys.  Lengths and offsets come from device memory, so each is brought into the range of
// its buffer: a wrong one gives wrong rows, never an access outside.
struct AttnSeq {
  int q0, nq;   // its tokens in q
  int kv0, kv;  // its keys: packed rows kv0.., or positions 0.. of its pages
  int off;      // position of its token 0 among the keys
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// Keys that token `tok` of a sequence sees under the causal mask.
__device__ __forceinline__ int attn_limit(const AttnSeq &s, int tok) {
  const long long n = (long long)s.off + tok + 1;
  return n < 0 ? 0 : (n > s.kv ? s.kv : (int)n);
}

template <bool PAGED>
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs &a, int b) {
  AttnSeq s;
  if (a.cu_q) {
    s.q0 = clampi(a.cu_q[b], 0, a.n_tokens);
    s.nq = clampi(a.cu_q[b + 1], s.q0, a.n_tokens) - s.q0;
  } else {
    s.q0 = b;
    s.nq = 1;
  }
  if constexpr (PAGED) {
    const int cap = a.table_width << a.page_shift;  // below 2^31 (the entry's check)
    s.kv0 = 0;
    s.off = clampi(a.ctx[b], 0, cap);
    s.kv = s.nq > cap - s.off ? cap : s.off + s.nq;
  } else {
    if (a.cu_k) {
      s.kv0 = clampi(a.cu_k[b], 0, a.n_kv);
      s.kv = clampi(a.cu_k[b + 1], s.kv0, a.n_kv) - s.kv0;
    } else {  // as many K/V rows as tokens, at the same places
      s.kv0 = s.q0;
      s.kv = s.nq;
    }
    s.off = s.kv - s.nq;  // negative: the first tokens see nothing
  }
  return s;
}

// An entry of the block table, the same for the whole wave: through the scalar cache, so that waiting for it does not
// wait for the K and V rows on their way.
__device__ __forceinline__ int page_entry(const int32_t *table, long long i) {
  typedef const __attribute__((address_space(4))) int32_t *constant_p;
  return ((constant_p)(uintptr_t)table)[i];
}

// A unit of work: a tile of rows of a sequence and one piece of its keys.
struct AttnUnit {
  AttnSeq s;
  int seq, tile, piece, pieces, piece_keys;
};

// Sum over the wave's lanes.  Handed back through a scalar register, as every number here that all lanes share: the
// compiler then keeps what follows from it (pages, row addresses, loop bounds) out of the vector registers.
__device__ __forceinline__ int wave_sum(int v) {
  v += (int)dpp_u<DPP_QUAD_XOR1>((uint32_t)v);
  v += (int)dpp_u<DPP_QUAD_XOR2>((uint32_t)v);
  v += (int)dpp_u<DPP_ROW_HALF_MIRROR>((uint32_t)v);
  v += (int)dpp_u<DPP_ROW_MIRROR>((uint32_t)v);
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = (int)(a[0] + a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return __builtin_amdgcn_readfirstlane((int)(b[0] + b[1]));
}

// Tiles of 2^shift rows that a sequence has (tokens times heads stay below 2^31, the entry's check).
__device__ __forceinline__ int attn_tiles(const AttnSeq &s, int group, int shift) {
  return (int)(((unsigned)(s.nq * group) + (1u << shift) - 1) >> shift);
}

// Sequence b of the step of 64 that starts at b0; the first step is kept by the caller.
template <bool PAGED>
__device__ __forceinline__ AttnSeq attn_step(const AttnArgs &a, int b0, const AttnSeq &first) {
  AttnSeq s{0, 0, 0, 0, 0};
  if (b0 == 0)
    s = first;
  else if (b0 + (int)__lane_id() < a.n_seqs)
    s = attn_seq<PAGED>(a, b0 + __lane_id());
  return s;
}

// Keys per piece: the summed key counts of all tiles over the units aimed at, in whole blocks of 64.  Every
// workgroup derives the same number from the lengths, so the host needs none of them.
template <bool PAGED>
__device__ __forceinline__ int attn_piece_keys(const AttnArgs &a, int shift, const AttnSeq &first) {
  long long sum = 0;
  for (int b0 = 0; b0 < a.n_seqs; b0 += 64) {
    const AttnSeq s = attn_step<PAGED>(a, b0, first);
    sum += (long long)attn_tiles(s, a.group, shift) * s.kv;
  }
  // 24 bits at a time through the fast lane sums
  long long all = 0;
  for (int i = 0; i < 3; ++i) all += (long long)wave_sum((int)(sum >> (24 * i)) & 0xffffff) << (24 * i);
  sum = all;
  const long long keys = sum / a.split_target + 1;
  return __builtin_amdgcn_readfirstlane(
      keys < kAttnMinChunk ? kAttnMinChunk : (keys > 0x7fffff00 ? 0x7fffffff : ((int)keys + 63) & ~63));
}

__device__ __forceinline__ int attn_pieces(const AttnSeq &s, int piece_keys) {
  return s.kv <= piece_keys ? 1 : (int)(((unsigned)s.kv + (unsigned)piece_keys - 1) / (unsigned)piece_keys);
}

// What a workgroup does.  FIND_HEADS_LAST: `want` counts the KV heads fastest (workgroups that run together share a
// head's K/V rows in one L2, as the compute dies are dealt workgroups in turn); FIND_HEADS_FIRST: it counts units
// fastest, and comes back as the unit with the head in `hk`; FIND_ROW: the first piece's unit of row `hk` of token
// `want`.  False: past the last.  Every lane of the wave takes part.  Units go by sequences, tiles from the last (which
// sees the most keys) to the first, and pieces; where nothing is cut and one step of the wave's lanes holds all
// sequences, by tiles first, the longest of all sequences to the shortest.
enum { FIND_HEADS_LAST, FIND_HEADS_FIRST, FIND_ROW };

template <bool PAGED, int MODE>
__device__ __forceinline__ bool attn_find(const AttnArgs &a, int shift, int &want, int &hk, AttnUnit &u) {
  const int lane = __lane_id();
  AttnSeq first{0, 0, 0, 0, 0};
  if (lane < a.n_seqs) first = attn_seq<PAGED>(a, lane);
  u.piece_keys = a.split_target ? attn_piece_keys<PAGED>(a, shift, first) : 0x7fffffff;
  if constexpr (MODE == FIND_HEADS_LAST) {
    hk = (unsigned)want % (unsigned)a.n_kv_heads;
    want = (unsigned)want / (unsigned)a.n_kv_heads;
  }
  if constexpr (MODE == FIND_HEADS_FIRST) {
    int total = 0;
    for (int b0 = 0; b0 < a.n_seqs; b0 += 64) {
      const AttnSeq s = attn_step<PAGED>(a, b0, first);
      total += wave_sum(attn_tiles(s, a.group, shift) * attn_pieces(s, u.piece_keys));
    }
    if (total == 0) return false;
    hk = (unsigned)want / (unsigned)total;
    want -= hk * total;
    if (hk >= a.n_kv_heads) return false;
  }
  int base = 0;
  for (int b0 = 0; b0 < a.n_seqs; b0 += 64) {
    const AttnSeq s = attn_step<PAGED>(a, b0, first);
    const int tiles = attn_tiles(s, a.group, shift), pieces = attn_pieces(s, u.piece_keys);
    auto take = [&](int l) {
      u.seq = b0 + l;
      u.s.q0 = __builtin_amdgcn_readlane(s.q0, l);
      u.s.nq = __builtin_amdgcn_readlane(s.nq, l);
      u.s.kv0 = __builtin_amdgcn_readlane(s.kv0, l);
      u.s.kv = __builtin_amdgcn_readlane(s.kv, l);
      u.s.off = __builtin_amdgcn_readlane(s.off, l);
      u.pieces = __builtin_amdgcn_readlane(pieces, l);
    };
    if (MODE != FIND_ROW && !a.split_target && a.n_seqs > 1 && a.n_seqs <= 64) {
      // from(t): the units of tiles t and later, which come before all others
      auto from = [&](int t) { return wave_sum(tiles > t ? tiles - t : 0); };
      if (want >= from(0)) return false;
      int lo = 0, hi = 1;
      while (from(hi) > want) lo = hi, hi *= 2;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (from(mid) > want)
          lo = mid;
        else
          hi = mid;
      }
      const unsigned long long has = __ballot(tiles > lo);
      const int nth = want - from(lo + 1);
      const bool mine = tiles > lo && __popcll(has & ((1ull << lane) - 1)) == nth;
      take(__builtin_ctzll(__ballot(mine)));
      u.tile = lo;
      u.piece = 0;
      return true;
    }
    const int units = tiles * pieces;
    int incl = units;
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(incl, d);
      if (lane >= d) incl += o;
    }
    const bool mine = MODE == FIND_ROW ? (want >= s.q0 && want < s.q0 + s.nq)
                                       : (want >= base + incl - units && want < base + incl);
    const unsigned long long hit = __ballot(mine);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      take(l);
      const int begin = base + __builtin_amdgcn_readlane(incl - units, l);
      const int n = __builtin_amdgcn_readlane(tiles, l);
      if constexpr (MODE == FIND_ROW) {
        u.tile = ((want - u.s.q0) * a.group + hk) >> shift;
        u.piece = 0;
        want = begin + (n - 1 - u.tile) * u.pieces;
      } else {
        const int t = (int)((unsigned)(want - begin) / (unsigned)u.pieces);
        u.tile = n - 1 - t;
        u.piece = (want - begin) - t * u.pieces;
        // offsets that do not rise can add up past 32 bits: no tile then, rather than one of no sequence
        if ((unsigned)t >= (unsigned)n) return false;
      }
      return true;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// f(0), f(1), ... with the indices as constants.
template <int... I, class F>
__device__ __forceinline__ void each(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>{}), ...);
}

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));
// K/V rows are 8-byte aligned (what the K/V pack asks of them).
typedef v4u v4u_a8 __attribute__((aligned(8)));
typedef v2u v2u_a4 __attribute__((aligned(4)));
typedef v4f v4f_a16 __attribute__((aligned(16)));

// The f32 operands of the two products (q rows and softmax weights) enter the binary16 matrix instructions as
// x = hi + lo with hi = f16(x) and lo = f16(x - hi): 22 bits of x, so that the products with the binary16 K and V
// rows keep f32 accuracy; the accumulators are f32.  A q row is first scaled by the power of two that brings its
// largest element to [2^12, 2^13): neither part overflows, and lo's subnormals start 2^-36 below the row's largest.
__device__ __forceinline__ int q_row_exponent(float row_max) {
  const int e = (int)((__builtin_bit_cast(uint32_t, row_max) >> 23) & 255u);
  return (e == 0 || e == 255) ? 0 : 139 - e;
}

__device__ __forceinline__ void split8(const float (&x)[8], v8h &hi, v8h &lo) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const v2h h = __builtin_convertvector((v2f{x[i], x[i + 1]}), v2h);
    // x - h, exact, as fused multiply-adds that take their binary16 operand without a conversion (from the source
    // they become two instructions each)
    v2f d;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d[0]) : "v"(h), "v"(x[i]));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d[1]) : "v"(h), "v"(x[i + 1]));
    const v2h r = __builtin_convertvector(d, v2h);
    hi[i] = h[0], hi[i + 1] = h[1];
    lo[i] = r[0], lo[i + 1] = r[1];
  }
}

// Infinities and NaN among the binary16 elements of a V operand.  Rows that do not see such an element's key must not
// meet it as 0 * Inf, so where a mask cuts, these elements go as zeros into the product with the weights, and a second
// pair of products counts, per row and element, the +Inf and -Inf (NaN: both) among the keys that the row does see.
__device__ __forceinline__ bool nonfinite16(uint32_t x) {
  return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u;
}
__device__ __forceinline__ bool any_nonfinite(v8h v) {
  const v4u w = __builtin_bit_cast(v4u, v);
  return nonfinite16(w[0]) || nonfinite16(w[1]) || nonfinite16(w[2]) || nonfinite16(w[3]);
}
__device__ __forceinline__ v8h finite_part(v8h v) {
  v8h r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint16_t b = __builtin_bit_cast(uint16_t, (_Float16)v[i]);
    r[i] = (b & 0x7c00u) == 0x7c00u ? (_Float16)0.0f : (_Float16)v[i];
  }
  return r;
}
// 1 for an infinity of the sign and for NaN, else 0.
__device__ __forceinline__ v8h infinite_part(v8h v, bool negative) {
  v8h r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint16_t b = __builtin_bit_cast(uint16_t, (_Float16)v[i]);
    const bool on = b == (negative ? 0xfc00u : 0x7c00u) || (b & 0x7fffu) > 0x7c00u;
    r[i] = (_Float16)(on ? 1.0f : 0.0f);
  }
  return r;
}
// 1 for each of the lane's 8 keys whose bit is set.
__device__ __forceinline__ v8h seen_part(unsigned bits) {
  v8h r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (_Float16)((bits >> i) & 1 ? 1.0f : 0.0f);
  return r;
}

// Softmax weights are 2^(score - reference + 4): the reference follows the running maximum only when a score
// passes it by more than 8, so weights reach 2^12 at most and lo keeps its bits for weights near 1.
constexpr float kAttnWeightShift = 4.0f;
constexpr float kAttnLazy = 8.0f;

// Shapes and pointers are validated by the caller; tiles hold 2^shift rows (kAttnRowShift or kAttnTileShift), units: at
// most, per KV head, split: pieces have to be joined.
void launch_attention(const AttnArgs &a, int head_dim, bool paged, int shift, long long units, bool split,
                      hipStream_t stream);
void launch_attention_tiles(const AttnArgs &a, int head_dim, bool paged, unsigned grid, hipStream_t stream);

}  // namespace v7g
