// k_attention_tiles.hip -- attention of many rows, gfx950: whole prompts, and pieces of a prompt or trees of drafts
// over the paged cache.
//
// out = sum_j softmax_j(q . k_j * scale) v_j with an online softmax, bound by the matrix instructions.  A workgroup
// takes 128 rows (tokens times the query heads of one KV head), 32 to a wave, and walks the keys 32 at a time; K and V
// rows of the next 32 keys are on their way into LDS meanwhile (two buffers, one barrier per step), so each K/V row is
// read once per 128 rows.  As in the few-row kernel the products are transposed, S^T = K Q^T and O^T = V^T P^T, with
// 32x32x16 matrix instructions:
//   - a lane holds 16 scores of one row, the lane 32 further the other 16 of the block: the row's maximum is an
//     in-lane tree and one exchange, its sum one exchange at the very end;
//   - the scores' places are those of the second product's B operand if contraction index 8h+j (h = lane/32) means
//     key 4h+j (j < 4) or 8+4h+j-4 of each 16: the weights never move between lanes.  V^T's A operand in that order is
//     two transposing LDS reads of 4 keys each.
// LDS rows are padded so that no read meets itself on a bank: K by 16 bytes (the 8 rows of one pass of 16-byte reads
// start 16 bytes apart), V to an odd multiple of 64 bytes (4 rows of 64 bytes each in one pass of transposing reads).
// Counted at 8192 tokens: no conflict; with V rows padded by 32 bytes a quarter of the LDS cycles were, and trees of
// drafts took 3% longer.  The matrix units are busy 59% of the time there, at the 1.7 GHz that the power leaves.
#include "v7g_attention.h"
#include "v7g_internal.h"

namespace v7g {

namespace {

constexpr int kKeys = 32;  // keys of a step

template <int D>
struct TileLds {
  static constexpr int krow = D + 8, vrow = D % 64 ? D : D + 32;  // elements
  static constexpr int side = kKeys * (krow + vrow);
  // The widest heads leave no registers for the lower part of q: it waits in LDS, each wave's own.
  static constexpr bool q_low = D >= 224;
  static constexpr int bytes = 2 * side * 2 + (q_low ? kAttnTileRows * D * 2 : 0);
};

// Elements d0..d0+15 of 4 keys, transposed: lane i of 16 gets element d0+i of the 4 keys; it hands in the address of
// key i/4, elements 4*(i%4)...
__device__ __forceinline__ v4h read_transposed(const _Float16 *p) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s *lds_p;
  return __builtin_bit_cast(v4h, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(p)));
}

// The maximum with the lane 32 further.
__device__ __forceinline__ float max_halves(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// PAIR: eight waves, two groups of four that take the steps in turn, each with buffers of its own, and meet at the end.
// The same compute unit then works through one tile in half the time instead of through two side by side.
template <int D, bool PAGED, bool PAIR>
__global__ __launch_bounds__(PAIR ? 512 : 256, D <= 128 ? 2 : 1) void attention_tiles_kernel(AttnArgs a) {
  using L = TileLds<D>;
  constexpr int KS = D / 16, DT = D / 32, CR = D / 8;
  constexpr int kStride = PAIR ? 2 * kKeys : kKeys;  // keys between a group's steps
  constexpr int NL = (kKeys * CR + 255) / 256;  // 16-byte pieces of a K tile per thread
  constexpr auto pieces = std::make_integer_sequence<int, NL>{};
  extern __shared__ _Float16 lds[];
  const int lane = threadIdx.x & 63, tid = threadIdx.x & 255;
  const int group = PAIR ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
  _Float16 *tile_lds = lds + (PAIR ? group * 2 * L::side : 0);
  const int h = lane >> 5, c = lane & 31;
  int hk, unit = blockIdx.x;
  AttnUnit u;
  if (!attn_find<PAGED, FIND_HEADS_LAST>(a, kAttnTileShift, unit, hk, u) || unit >= a.units) return;
  const AttnSeq s = u.s;
  const int row0 = u.tile * kAttnTileRows + wave * 32;
  const int left = s.nq * a.group - row0;
  const int n_rows = left < 0 ? 0 : (left < 32 ? left : 32);  // of this wave
  const int row = row0 + (c < n_rows ? c : n_rows - 1);
  const int tok = n_rows ? row / a.group : 0, head = hk * a.group + (n_rows ? row % a.group : 0);
  const bool tree = PAGED && a.mask_words;
  const int64_t *words = a.mask + (long long)(s.q0 + tok) * a.mask_words;
  auto lim_of = [&](int r) { return attn_limit(s, r / a.group); };
  const int ctx = min(s.off, s.kv);
  const int lim = tree ? ctx : attn_limit(s, tok);
  // the wave's rows all see the keys below lim_min, and none from lim_max on
  const int lim_min = tree ? ctx : lim_of(row0);
  const int lim_max = n_rows == 0 ? 0 : (tree ? s.kv : lim_of(row0 + n_rows - 1));
  const int last_row = min(u.tile * kAttnTileRows + kAttnTileRows, s.nq * a.group) - 1;
  const int tile_max = tree ? s.kv : lim_of(last_row);
  const int key_lo = u.piece ? u.piece * u.piece_keys : 0;
  const int key_hi = u.piece + 1 < u.pieces ? min((u.piece + 1) * u.piece_keys, tile_max) : tile_max;

  v16f acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = v16f{};
  float m = -__builtin_inff(), l = 0.0f;

  const uint16_t *kbase = a.k + (long long)hk * D, *vbase = a.v + (long long)hk * D;
  // pages of a step's two 16-key halves, -1 where there is none
  auto pages_at = [&](int kb, int (&pg)[2]) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        pg[i] = -1;
        if (kb + 16 * i < key_hi) {
          const int p = page_entry(a.table, (long long)u.seq * a.table_width + ((kb + 16 * i) >> a.page_shift));
          pg[i] = (unsigned)p < (unsigned)a.n_pages ? p : -1;
        }
      }
    }
  };
  v4u kreg[NL], vreg[NL];
  // where a thread's pieces of the step to fetch next lie: packed rows are walked from step to step, paged ones
  // within 16 keys of a page
  long long ko[NL], vo[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int idx = tid + i * 256, r = idx / CR, ch = idx % CR;
    const long long first = PAGED ? (r & 15) : s.kv0 + key_lo + group * kKeys + r;
    ko[i] = first * a.k_stride + ch * 8;
    vo[i] = first * a.v_stride + ch * 8;
  }
  const long long kstep = kStride * a.k_stride, vstep = kStride * a.v_stride;
  // K and V rows of keys kb.. into registers; keys of no row or no page become zeros (read at the step's first row,
  // or in page 0)
  auto fetch = [&](int kb, const int (&pg)[2]) {
    const uint16_t *k0 = kbase, *k1 = kbase, *v0 = vbase, *v1 = vbase;
    if constexpr (PAGED) {
      const int in0 = kb & ((1 << a.page_shift) - 1), in1 = (kb + 16) & ((1 << a.page_shift) - 1);
      const long long p0 = max(pg[0], 0) * a.page_stride, p1 = max(pg[1], 0) * a.page_stride;
      k0 += p0 + in0 * a.k_stride;
      v0 += p0 + in0 * a.v_stride;
      k1 += p1 + in1 * a.k_stride;
      v1 += p1 + in1 * a.v_stride;
    }
    const bool whole = kb + kKeys <= key_hi && (!PAGED || (pg[0] >= 0 && pg[1] >= 0));
    each(pieces, [&](auto i) {
      const int idx = tid + i * 256, r = idx / CR, ch = idx % CR;
      const bool inside = kb + r < key_hi && (NL * 256 == kKeys * CR || r < kKeys);
      const uint16_t *kp = (PAGED && r >= 16 ? k1 : k0) + ko[i], *vp = (PAGED && r >= 16 ? v1 : v0) + vo[i];
      if (!inside) {
        kp = (PAGED ? k0 : k0 + ko[i] - r * a.k_stride) + (PAGED ? ch * 8 : 0);
        vp = (PAGED ? v0 : v0 + vo[i] - r * a.v_stride) + (PAGED ? ch * 8 : 0);
      }
      kreg[i] = *reinterpret_cast<const v4u_a8 *>(kp);
      vreg[i] = *reinterpret_cast<const v4u_a8 *>(vp);
      if constexpr (!PAGED) {
        ko[i] += kstep;
        vo[i] += vstep;
      }
    });
    if (!whole) {
      each(pieces, [&](auto i) {
        const int r = (tid + i * 256) / CR;
        const bool on = kb + r < key_hi && (!PAGED || (r < 16 ? pg[0] : pg[1]) >= 0);
        kreg[i] = on ? kreg[i] : v4u{0, 0, 0, 0};
        vreg[i] = on ? vreg[i] : v4u{0, 0, 0, 0};
      });
    }
  };
  auto store = [&](_Float16 *buf) {
    each(pieces, [&](auto i) {
      const int idx = tid + i * 256;
      const int r = idx / CR, ch = idx % CR;
      if (NL * 256 == kKeys * CR || r < kKeys) {
        *reinterpret_cast<v4u *>(buf + r * L::krow + ch * 8) = kreg[i];
        *reinterpret_cast<v4u *>(buf + kKeys * L::krow + r * L::vrow + ch * 8) = vreg[i];
      }
    });
  };

  // the first step's rows are on their way while q is prepared
  int pg[2] = {0, 0};
  auto gone_of = [&] { return PAGED ? (pg[0] < 0 ? 1u : 0u) | (pg[1] < 0 ? 2u : 0u) : 0u; };
  int kb = key_lo + group * kKeys;
  unsigned gone = 0, next_gone = 0;
  if (kb < key_hi) {
    pages_at(kb, pg);
    gone = gone_of();
    fetch(kb, pg);
  }

  // ---- q rows in two binary16 parts; the scale's sign goes with them, so that the largest product is the maximum
  v8h qh[KS], ql[L::q_low ? 1 : KS];
  v8h *qlow = reinterpret_cast<v8h *>(tile_lds + 2 * L::side) + wave * KS * 64 + lane;
  float factor;
  {
    const float *qr = a.q + (long long)(s.q0 + tok) * a.q_stride + (long long)head * D + h * 8;
    const float sign = a.scale_log2 < 0.0f ? -1.0f : (a.scale_log2 == 0.0f ? 0.0f : 1.0f);
    float mx = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, __builtin_fabsf(qr[ks * 16 + i]));
    mx = max_halves(mx);
    const int e = q_row_exponent(mx);
    // never 0: it multiplies the -inf of hidden keys (a factor this small makes every score vanish all the same)
    factor = sign == 0.0f ? 1.0f : fmaxf(__builtin_ldexpf(__builtin_fabsf(a.scale_log2), -e), 0x1p-126f);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __builtin_ldexpf(qr[ks * 16 + i], e) * sign;
      v8h low;
      split8(x, qh[ks], low);
      if constexpr (L::q_low)
        qlow[ks * 64] = low;
      else
        ql[ks] = low;
    }
  }

  // One step on a buffer; bit i of gone: its keys 16i.. are on no page.  CUT: the mask, the piece's end or the last key
  // runs through it.
  auto step = [&](auto cut, const _Float16 *buf, int kb, unsigned gone) {
    constexpr bool CUT = cut;
    const _Float16 *kl = buf + c * L::krow + h * 8;
    const _Float16 *vl =
        buf + kKeys * L::krow + (4 * h + (lane & 15) / 4) * L::vrow + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    v16f sc = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const v8h k8 = *reinterpret_cast<const v8h *>(kl + ks * 16);
      sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8, qh[ks], sc, 0, 0, 0);
      sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8, L::q_low ? qlow[ks * 64] : ql[L::q_low ? 0 : ks], sc, 0, 0, 0);
    }
    unsigned seen = 0xffffu;  // of this lane's 16 keys, those its row sees
    if constexpr (CUT) {
      seen = 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = kb + 8 * (r >> 2) + 4 * h + (r & 3), d = key - s.off;
        bool on = key < lim;
        if (tree && !on) on = d < a.mask_words * 64 && ((words[d >> 6] >> (d & 63)) & 1);
        if (on && key < key_hi) seen |= 1u << r;
      }
    }
    if constexpr (PAGED) seen &= ~((gone & 1 ? 0xffu : 0u) | (gone & 2 ? 0xff00u : 0u));
    if (CUT || (PAGED && gone)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = (seen >> r) & 1 ? sc[r] : -__builtin_inff();
    }
    float mx = sc[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, sc[r]);
    mx = max_halves(mx) * factor;
    if (__ballot(mx > m + kAttnLazy)) {
      const float nm = fmaxf(m, mx);
      const float alpha = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - nm);
      m = nm;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] *= alpha;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : kAttnWeightShift - m;
#pragma unroll
    for (int st = 0; st < 2; ++st) {  // 16 keys
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * st + j], factor, ref));
        l += p[j];
      }
      v8h ph, pl;
      split8(p, ph, pl);
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const v4h a0 = read_transposed(vl + 16 * st * L::vrow + t * 32);
        const v4h a1 = read_transposed(vl + (16 * st + 8) * L::vrow + t * 32);
        v8h v8 = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (CUT)
          if (__ballot(any_nonfinite(v8))) {
            const v8h sees = seen_part(seen >> (8 * st));
            const v16f z = {};
            const v16f up = __builtin_amdgcn_mfma_f32_32x32x16_f16(infinite_part(v8, false), sees, z, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[t][r] += up[r] > 0.0f ? __builtin_inff() : 0.0f;
            const v16f down = __builtin_amdgcn_mfma_f32_32x32x16_f16(infinite_part(v8, true), sees, z, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[t][r] -= down[r] > 0.0f ? __builtin_inff() : 0.0f;
            v8 = finite_part(v8);
          }
        acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8, ph, acc[t], 0, 0, 0);
        acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8, pl, acc[t], 0, 0, 0);
      }
    }
  };

  // ---- the keys, 32 at a time: while one buffer is read, the other is filled and the step after fetched
  if (key_lo < key_hi) {
    if (kb < key_hi) store(tile_lds);
    if (kb + kStride < key_hi) {
      pages_at(kb + kStride, pg);
      next_gone = gone_of();
      fetch(kb + kStride, pg);
    }
    pages_at(kb + 2 * kStride, pg);
    __syncthreads();
    int at = 0;
    for (int k0 = key_lo; k0 < key_hi; k0 += kStride, kb += kStride) {  // as many rounds for both groups
      unsigned after = 0;
      if (kb + kStride < key_hi) {
        store(tile_lds + (at ^ 1) * L::side);
        if (kb + 2 * kStride < key_hi) {
          after = gone_of();
          fetch(kb + 2 * kStride, pg);
          pages_at(kb + 3 * kStride, pg);
        }
      }
      const _Float16 *buf = tile_lds + at * L::side;
      // through a vector register: as a scalar branch the two forms of the step cost 50 to 500 bytes of spills
      int end = kb + kKeys;
      asm("" : "+v"(end));
      if (end <= lim_min && end <= key_hi)
        step(std::false_type{}, buf, kb, gone);
      else if (end - kKeys < lim_max && end - kKeys < key_hi)
        step(std::true_type{}, buf, kb, gone);
      __syncthreads();
      at ^= 1;
      gone = next_gone;
      next_gone = after;
    }
  }

  if constexpr (PAIR) {  // the second group's result into the first's
    static_assert(4 * 64 * (DT * 16 + 2) * 4 <= 2 * L::bytes, "the buffers hold a group's accumulators");
    float *x = reinterpret_cast<float *>(lds) + wave * 64 * (DT * 16 + 2) + lane * 4;
    float *ml = reinterpret_cast<float *>(lds) + wave * 64 * (DT * 16 + 2) + 64 * DT * 16 + lane;
    if (group == 1) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<v4f *>(x + (t * 4 + q) * 256) =
              v4f{acc[t][4 * q], acc[t][4 * q + 1], acc[t][4 * q + 2], acc[t][4 * q + 3]};
      ml[0] = m;
      ml[64] = l;
    }
    __syncthreads();
    if (group == 1) return;
    const float m2 = ml[0], l2 = ml[64];
    const float nm = fmaxf(m, m2);
    const float a1 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - nm);
    const float a2 = m2 == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m2 - nm);
    l = l * a1 + l2 * a2;
    m = nm;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const v4f o = *reinterpret_cast<const v4f *>(x + (t * 4 + q) * 256);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][4 * q + r] = acc[t][4 * q + r] * a1 + o[r] * a2;
      }
  }

  l += xor_f(l, 32);
  if (c >= n_rows) return;
  float *dst;
  float mul;
  if (u.pieces == 1) {
    dst = a.out + (long long)(s.q0 + tok) * a.out_stride + (long long)head * D;
    mul = l == 0.0f ? 0.0f : 1.0f / l;  // a row that sees nothing gives zeros
  } else {
    const long long slot = ((long long)unit * a.n_kv_heads + hk) * kAttnTileRows + wave * 32 + c;
    dst = a.part_o + slot * D;
    mul = 1.0f;
    if (h == 0) {
      a.part_ml[slot * 2] = m;
      a.part_ml[slot * 2 + 1] = l;
    }
  }
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const v4f o = {acc[t][4 * q] * mul, acc[t][4 * q + 1] * mul, acc[t][4 * q + 2] * mul, acc[t][4 * q + 3] * mul};
      *reinterpret_cast<v4f_a16 *>(dst + t * 32 + 8 * q + 4 * h) = o;
    }
}

template <int D>
void tiles_launch(const AttnArgs &a, bool paged, unsigned grid, hipStream_t stream) {
  // Pairs where every tile has a compute unit's half to itself: the longest tile is then the call (one prompt, 32/8
  // heads x 128, 1500 tokens 69 -> 57 us, 512 27 -> 26; 2048 tokens, 28/4 heads 92 -> 80).  With more tiles two of
  // them side by side hide each other's start and end (13 prompts of 6001 tokens 152 us against 188, 20 of 8192 141
  // against 189), and heads of 64 leave little to halve (700 tokens, 14/2 heads 25.7 against 27.1).
  if constexpr (D == 96 || D == 128) {
    if (grid <= 512 && !a.split_target && !paged) {
      enqueue(attention_tiles_kernel<D, false, true>, dim3(grid), dim3(512), 2 * TileLds<D>::bytes, stream, a);
      return;
    }
  }
  if (paged)
    enqueue(attention_tiles_kernel<D, true, false>, dim3(grid), dim3(256), TileLds<D>::bytes, stream, a);
  else
    enqueue(attention_tiles_kernel<D, false, false>, dim3(grid), dim3(256), TileLds<D>::bytes, stream, a);
}

}  // namespace

void launch_attention_tiles(const AttnArgs &a, int head_dim, bool paged, unsigned grid, hipStream_t stream) {
  switch (head_dim) {
    case 64: tiles_launch<64>(a, paged, grid, stream); break;
    case 96: tiles_launch<96>(a, paged, grid, stream); break;
    case 128: tiles_launch<128>(a, paged, grid, stream); break;
    case 160: tiles_launch<160>(a, paged, grid, stream); break;
    case 192: tiles_launch<192>(a, paged, grid, stream); break;
    case 224: tiles_launch<224>(a, paged, grid, stream); break;
    case 256: tiles_launch<256>(a, paged, grid, stream); break;
  }
}

}  // namespace v7g
