// k_attention_rows.hip -- attention of a few rows over a long run of keys, gfx950: the tokens of a decoding step or
// of a tree of drafts over the paged cache, and any head_dim the matrix tiles of the prompt kernel do not cover.
//
// out = sum_j softmax_j(q . k_j * scale) v_j with an online softmax: one pass over K and V, a running reference and
// sum per row.  Such a call is bound by reading K and V once from HBM: a workgroup takes 16 rows (the query heads of
// one KV head, times the tokens) and a piece of the keys; its four waves take blocks of 32 keys in turn, each with
// its own softmax, and meet once at the end.  No wave waits for another inside the loop, and no LDS stands between
// the loads and the matrix instructions:
//   S^T = K Q^T: A operand (16 keys x 32 dims), lane (g = lane/16, c = lane%16) holds key c's dims 8g..8g+7, 16 bytes
//     of a K row straight from memory.  The result leaves lane (g, c) the scores of row c at keys 4g..4g+3.
//   O^T = V^T P^T over 32 keys: the two S tiles already are the B operand if contraction index 8g+j means key 4g+j of
//     the first tile (j < 4) or 4g+j-4 of the second.  Lane (g, c) loads a slice of its 8 keys' V rows (16 bytes at
//     head_dim 128: 16 lanes read 256 bytes of a row); the row index c of tile t then stands for element 8c+t, and
//     the A operand of every tile comes from the lane's own registers with one v_perm per pair of keys.
#include "v7g_attention.h"
#include "v7g_internal.h"

namespace v7g {

namespace {

// A head's dims in slices of 128, then 64, then 32: a lane holds 8, 4 or 2 consecutive elements of a slice of each of
// its 8 keys, and the slice makes as many 16-row tiles.  Tile t of the slice at `base`: row index r is element
// base + r * WIDTH + t.
template <int D>
struct VSlices {
  static constexpr int n128 = D / 128, has64 = (D % 128) / 64, has32 = (D % 64) / 32;
  static constexpr int count = n128 + has64 + has32;
  static constexpr int width(int i) { return i < n128 ? 8 : (has64 && i == n128 ? 4 : 2); }
  static constexpr int base(int i) { return i <= n128 ? i * 128 : n128 * 128 + 64; }
  static constexpr int tile(int i) { return base(i) / 16; }
};

template <int WIDTH>
__device__ __forceinline__ void load_slice(const uint16_t *p, uint32_t (&v)[4]) {
  if constexpr (WIDTH == 8) {
    const v4u x = *reinterpret_cast<const v4u_a8 *>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else if constexpr (WIDTH == 4) {
    const v2u x = *reinterpret_cast<const v2u_a4 *>(p);
    v[0] = x.x, v[1] = x.y;
  } else {
    v[0] = *reinterpret_cast<const uint32_t *>(p);
  }
}

// A operand of tile t of a slice: the pairs of keys at element t.
__device__ __forceinline__ v4u v_tile(const uint32_t (&v)[8][4], int t) {
  const unsigned sel = (t & 1) ? 0x07060302u : 0x05040100u;
  v4u f;
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) f[jj] = __builtin_amdgcn_perm(v[2 * jj + 1][t / 2], v[2 * jj][t / 2], sel);
  return f;
}

template <int D, bool PAGED>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void attention_rows_kernel(AttnArgs a) {
  using S = VSlices<D>;
  constexpr int KS = D / 32, NT = D / 16;
  // Two blocks' K and V rows fit in registers: one is computed while the other is on its way (8 waves of a compute
  // unit keep 16 KB each in flight at head_dim 128).  Wider heads load each slice as it is used.
  constexpr bool AHEAD = D <= 256;
  constexpr auto slices = std::make_integer_sequence<int, S::count>{};
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  // heads first: workgroups that run at the same time read different pages (37 sequences: 182 -> 169 us against the
  // other order, 64 of 1000-4000 keys 158 -> 148)
  int hk, unit = blockIdx.x;
  AttnUnit u;
  if (!attn_find<PAGED, FIND_HEADS_FIRST>(a, kAttnRowShift, unit, hk, u) || unit >= a.units) return;
  const AttnSeq s = u.s;
  const int rows = s.nq * a.group, row0 = u.tile * 16;
  const int n_rows = rows - row0 < 16 ? rows - row0 : 16;
  // this lane's row; the tile's rows behind the last one compute what that one does and are not stored
  const int row = row0 + (c < n_rows ? c : n_rows - 1);
  const int tok = row / a.group, head = hk * a.group + row % a.group;
  const bool tree = PAGED && a.mask_words;
  const int64_t *words = a.mask + (long long)(s.q0 + tok) * a.mask_words;
  // keys below lim are seen by the row, keys from lim on by the mask's bits or not at all
  const int ctx = min(s.off, s.kv);
  const int lim = tree ? ctx : attn_limit(s, tok);
  const int lim_min = tree ? ctx : attn_limit(s, row0 / a.group);
  const int lim_max = tree ? s.kv : attn_limit(s, (row0 + n_rows - 1) / a.group);
  const int key_lo = u.piece ? u.piece * u.piece_keys : 0;
  const int key_hi = u.piece + 1 < u.pieces ? min((u.piece + 1) * u.piece_keys, lim_max) : lim_max;
  const int full_hi = min(key_hi, lim_min);  // up to here every row sees every key

  v4f acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = v4f{0, 0, 0, 0};
  float m = -__builtin_inff(), l = 0.0f;

  const uint16_t *kbase = a.k + (long long)hk * D, *vbase = a.v + (long long)hk * D;
  // A block's two halves of 16 keys lie within one page each (pages hold a multiple of 16 tokens).
  struct Block {
    const uint16_t *k[2], *v[2];
    bool ok[2];
    int last;  // the block's last key of this piece; rows behind it are read there and masked
  };
  auto block_at = [&](int kb) {
    Block b;
    b.last = min(key_hi - 1 - kb, 31);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key0 = h && b.last < 16 ? kb : kb + 16 * h;
      b.ok[h] = true;
      if constexpr (PAGED) {
        int page = page_entry(a.table, (long long)u.seq * a.table_width + (key0 >> a.page_shift));
        b.ok[h] = (unsigned)page < (unsigned)a.n_pages;  // a page outside the pool: its keys are absent
        if (!b.ok[h]) page = 0;
        const int in = key0 & ((1 << a.page_shift) - 1);
        b.k[h] = kbase + page * a.page_stride + in * a.k_stride;
        b.v[h] = vbase + page * a.page_stride + in * a.v_stride;
      } else {
        b.k[h] = kbase + (long long)(s.kv0 + key0) * a.k_stride;
        b.v[h] = vbase + (long long)(s.kv0 + key0) * a.v_stride;
      }
    }
    return b;
  };

  // One block's rows in registers.
  struct Rows {
    v4u k[2][KS];
    uint32_t v[AHEAD ? S::count : 1][8][4];
    bool ok[2];
  };
  // Row offsets of a whole block (all 32 keys inside); CUT: rows behind the last key are read at that key.
  const long long k_row = c * a.k_stride + g * 8, v_row = 4 * g * a.v_stride;
  auto load_k = [&](auto cut, const Block &b, v4u (&k)[2][KS]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t *r = b.k[h] + k_row;
      if constexpr (cut) {
        const int last = h && b.last >= 16 ? b.last - 16 : min(b.last, 15);
        r = b.k[h] + (long long)min(c, last) * a.k_stride + g * 8;
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) k[h][ks] = *reinterpret_cast<const v4u_a8 *>(r + ks * 32);
    }
  };
  auto load_v = [&](auto cut, const Block &b, auto i, uint32_t (&v)[8][4]) {
    constexpr int W = S::width(i);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint16_t *r = b.v[j >> 2] + v_row + (j & 3) * a.v_stride;
      if constexpr (cut) {
        const int last = j >= 4 && b.last >= 16 ? b.last - 16 : min(b.last, 15);
        r = b.v[j >> 2] + (long long)min(4 * g + (j & 3), last) * a.v_stride;
      }
      load_slice<W>(r + S::base(i) + c * W, v[j]);
    }
  };
  constexpr auto whole = std::false_type{};
  constexpr auto cut = std::true_type{};
  auto load = [&](int kb, Rows &r) {
    const Block b = block_at(kb);
    r.ok[0] = b.ok[0], r.ok[1] = b.ok[1];
    load_k(whole, b, r.k);
    if constexpr (AHEAD) each(slices, [&](auto i) { load_v(whole, b, i, r.v[i]); });
  };
  // the first block is on its way while q is prepared
  int kb = key_lo + wave * 32;
  Rows ra;
  if constexpr (AHEAD)
    if (kb + 32 <= full_hi) load(kb, ra);

  // ---- q rows, scaled by a power of two and split in two binary16 parts; in LDS, where all four waves read them
  v8h *qlds = reinterpret_cast<v8h *>(lds);  // [KS][2][64]
  float factor;
  {
    const float *qr = a.q + (long long)(s.q0 + tok) * a.q_stride + (long long)head * D + g * 8;
    float mx = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, __builtin_fabsf(qr[ks * 32 + i]));
    mx = fmaxf(mx, xor_f(mx, 16));
    mx = fmaxf(mx, xor_f(mx, 32));
    const int e = q_row_exponent(mx);
    factor = __builtin_ldexpf(a.scale_log2, -e);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      if (ks % 4 == wave) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_ldexpf(qr[ks * 32 + i], e);
        v8h hi, lo;
        split8(x, hi, lo);
        qlds[(ks * 2) * 64 + lane] = hi;
        qlds[(ks * 2 + 1) * 64 + lane] = lo;
      }
    __syncthreads();
  }

  auto scores = [&](const v4u (&k)[2][KS], v4f (&sc)[2]) {
    sc[0] = sc[1] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const v8h hi = qlds[(ks * 2) * 64 + lane], lo = qlds[(ks * 2 + 1) * 64 + lane];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const v8h k8 = __builtin_bit_cast(v8h, k[h][ks]);
        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, hi, sc[h], 0, 0, 0);
        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, lo, sc[h], 0, 0, 0);
      }
    }
  };
  v8h ph, pl;
  // The block's weights from its scores (log2 domain; -inf where a key is not seen).
  auto weigh = [&](float (&x)[8]) {
    float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    mx = fmaxf(mx, xor_f(mx, 16));
    mx = fmaxf(mx, xor_f(mx, 32));
    if (__ballot(mx > m + kAttnLazy)) {
      const float nm = fmaxf(m, mx);
      const float alpha = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - nm);
      m = nm;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] *= alpha;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : m - kAttnWeightShift;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f(x[j] - ref);
      l += p[j];
    }
    split8(p, ph, pl);
  };
  auto add_slice = [&](auto i, const uint32_t (&v)[8][4]) {
#pragma unroll
    for (int t = 0; t < S::width(i); ++t) {
      v4f &o = acc[S::tile(i) + t];
      const v8h v8 = __builtin_bit_cast(v8h, v_tile(v, t));
      o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, ph, o, 0, 0, 0);
      o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, pl, o, 0, 0, 0);
    }
  };

  auto compute = [&](int kb, Rows &r) {
    v4f sc[2];
    scores(r.k, sc);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = sc[j >> 2][j & 3] * factor;
    const bool gone = PAGED && (!r.ok[0] || !r.ok[1]);
    if (gone) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!r.ok[j >> 2]) x[j] = -__builtin_inff();
    }
    weigh(x);
    each(slices, [&](auto i) {
      auto &v = r.v[AHEAD ? i : 0];
      if constexpr (!AHEAD) load_v(whole, block_at(kb), i, v);
      if (gone) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int d = 0; d < 4; ++d)
            if (!r.ok[j >> 2]) v[j][d] = 0;
      }
      add_slice(i, v);
    });
  };
  // ---- blocks whose keys every row sees
  if constexpr (AHEAD) {
    Rows rb;
    while (kb + 32 <= full_hi) {
      const bool second = kb + 160 <= full_hi;
      if (second) load(kb + 128, rb);
      compute(kb, ra);
      kb += 128;
      if (!second) break;
      if (kb + 160 <= full_hi) load(kb + 128, ra);
      compute(kb, rb);
      kb += 128;
    }
  } else {
    for (; kb + 32 <= full_hi; kb += 128) {
      Rows r;
      load(kb, r);
      compute(kb, r);
    }
  }
  // ---- blocks that the mask, the piece's end or the last key cuts
  for (; kb < key_hi; kb += 128) {
    const Block b = block_at(kb);
    v4u k[2][KS];
    load_k(cut, b, k);
    v4f sc[2];
    scores(k, sc);
    // which of this lane's keys its row sees
    unsigned seen = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3), d = key - s.off;
      bool on = key < lim;
      if (tree && !on) on = d < a.mask_words * 64 && ((words[d >> 6] >> (d & 63)) & 1);
      if (on && key < key_hi && b.ok[j >> 2]) seen |= 1u << j;
    }
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (seen >> j) & 1 ? sc[j >> 2][j & 3] * factor : -__builtin_inff();
    weigh(x);
    // keys that no row may read stand for zeros, whatever their V rows hold
    each(slices, [&](auto i) {
      constexpr int W = S::width(i);
      uint32_t v[8][4];
      load_v(cut, b, i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int d = 0; d < W / 2; ++d)
          if (kb + 16 * (j >> 2) + 4 * g + (j & 3) >= key_hi || !b.ok[j >> 2]) v[j][d] = 0;
#pragma unroll
      for (int t = 0; t < W; ++t) {
        v4f &o = acc[S::tile(i) + t];
        v8h v8 = __builtin_bit_cast(v8h, v_tile(v, t));
        if (__ballot(any_nonfinite(v8))) {
          const v8h sees = seen_part(seen);
          const v4f z = {0, 0, 0, 0};
          const v4f up = __builtin_amdgcn_mfma_f32_16x16x32_f16(infinite_part(v8, false), sees, z, 0, 0, 0);
          const v4f down = __builtin_amdgcn_mfma_f32_16x16x32_f16(infinite_part(v8, true), sees, z, 0, 0, 0);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            o[k] += up[k] > 0.0f ? __builtin_inff() : 0.0f;
            o[k] -= down[k] > 0.0f ? __builtin_inff() : 0.0f;
          }
          v8 = finite_part(v8);
        }
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, ph, o, 0, 0, 0);
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, pl, o, 0, 0, 0);
      }
    });
  }

  // ---- the four waves' results meet: 2 and 3 into 0 and 1, then 1 into 0
  l += xor_f(l, 16);
  l += xor_f(l, 32);
  __syncthreads();  // q in LDS is read no more
  float *ml = lds + 2 * NT * 64 * 4;     // [2][2][64] behind the two waves' accumulators
  v4f *ov = reinterpret_cast<v4f *>(lds);
#pragma unroll
  for (int step = 2; step >= 1; step >>= 1) {
    if (wave >= step && wave < 2 * step) {
      const int w = wave - step;
#pragma unroll
      for (int t = 0; t < NT; ++t) ov[(w * NT + t) * 64 + lane] = acc[t];
      ml[(w * 2) * 64 + lane] = m;
      ml[(w * 2 + 1) * 64 + lane] = l;
    }
    __syncthreads();
    if (wave < step) {
      const float m2 = ml[(wave * 2) * 64 + lane], l2 = ml[(wave * 2 + 1) * 64 + lane];
      const float nm = fmaxf(m, m2);
      const float a1 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - nm);
      const float a2 = m2 == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m2 - nm);
      l = l * a1 + l2 * a2;
      m = nm;
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] = acc[t] * a1 + ov[(wave * NT + t) * 64 + lane] * a2;
    }
    __syncthreads();
  }
  if (wave != 0 || c >= n_rows) return;
  float *dst;
  float mul;
  if (u.pieces == 1) {
    dst = a.out + (long long)(s.q0 + tok) * a.out_stride + (long long)head * D;
    mul = l == 0.0f ? 0.0f : 1.0f / l;  // a row that sees nothing gives zeros
  } else {
    const long long slot = ((long long)unit * a.n_kv_heads + hk) * 16 + c;
    dst = a.part_o + slot * D;
    mul = 1.0f;
    if (g == 0) {
      a.part_ml[slot * 2] = m;
      a.part_ml[slot * 2 + 1] = l;
    }
  }
  each(slices, [&](auto i) {
    constexpr int W = S::width(i);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int t = 0; t < W; ++t) dst[S::base(i) + (g * 4 + k) * W + t] = acc[S::tile(i) + t][k] * mul;
  });
}

// Joins the pieces of the rows whose keys were cut: one workgroup per (token, query head).  head_dim/4 threads read one
// piece's accumulator, 16 bytes each; the others take further pieces, 4 at a time each, and the groups' sums meet in
// LDS.  A few rows have many pieces (32768 keys of one token: 32 heads, 30 to 128 pieces each), so four waves read
// them side by side; with many rows one wave per row (two for head_dim above 256) does.
template <bool PAGED>
__global__ __launch_bounds__(256) void attention_join_kernel(AttnArgs a, int head_dim, int shift) {
  __shared__ v4f sums[256];
  __shared__ float group_l[16], group_m[4];
  const int tid = threadIdx.x, lane = tid & 63;
  const unsigned heads = a.n_kv_heads * a.group;
  const int tok = (int)(blockIdx.x / heads), head = (int)(blockIdx.x - tok * heads);
  const int hk = head / a.group;
  int hr = head - hk * a.group, unit = tok;
  AttnUnit u;
  if (!attn_find<PAGED, FIND_ROW>(a, shift, unit, hr, u) || u.pieces == 1) return;
  if (unit < 0 || unit > a.units - u.pieces) return;  // offsets that do not rise: sequences overlap, and some have no room
  const int r = ((tok - u.s.q0) * a.group + hr) & ((1 << shift) - 1);
  // slot of piece p: the tile's row r in unit + p
  const long long slot0 = ((((long long)unit * a.n_kv_heads + hk) << shift) + r);
  const long long step = (long long)a.n_kv_heads << shift;
  float m = -__builtin_inff();
  for (int p = tid; p < u.pieces; p += blockDim.x) m = fmaxf(m, a.part_ml[(slot0 + p * step) * 2]);
  for (int x = 32; x; x >>= 1) m = fmaxf(m, xor_f(m, x));
  if (tid < 4) group_m[tid] = -__builtin_inff();
  __syncthreads();
  if (lane == 0) group_m[tid >> 6] = m;
  const int wide = head_dim / 4, groups = (int)blockDim.x / wide, grp = tid / wide, d = (tid - grp * wide) * 4;
  __syncthreads();
  m = fmaxf(fmaxf(group_m[0], group_m[1]), fmaxf(group_m[2], group_m[3]));
  const float ref = m == -__builtin_inff() ? 0.0f : m;
  v4f o = {0, 0, 0, 0};
  float l = 0.0f;
  if (grp < groups)
    for (int p = grp; p < u.pieces; p += 4 * groups) {
      v4f v[4];
      float mp[4], lp[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long s = slot0 + (p + j * groups < u.pieces ? p + j * groups : p) * step;
        mp[j] = a.part_ml[s * 2], lp[j] = a.part_ml[s * 2 + 1];
        v[j] = *reinterpret_cast<const v4f_a16 *>(a.part_o + s * head_dim + d);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // an empty piece weighs 2^-inf = 0
        const float w = p + j * groups < u.pieces ? __builtin_amdgcn_exp2f(mp[j] - ref) : 0.0f;
        l += w * lp[j];
        o += w * v[j];
      }
    }
  sums[tid] = o;
  if (d == 0 && grp < groups) group_l[grp] = l;
  __syncthreads();
  if (grp != 0) return;
  for (int g = 1; g < groups; ++g) {
    o += sums[g * wide + tid];
    l += group_l[g];
  }
  const float mul = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<v4f_a16 *>(a.out + (long long)tok * a.out_stride + (long long)head * head_dim + d) = o * mul;
}

template <int D>
void rows_launch(const AttnArgs &a, bool paged, unsigned grid, hipStream_t stream) {
  const unsigned lds = (2 * (D / 16) * 64 * 4 + 4 * 64) * 4;  // two waves' accumulators and softmax states; >= q's parts
  if (paged)
    enqueue(attention_rows_kernel<D, true>, dim3(grid), dim3(256), lds, stream, a);
  else
    enqueue(attention_rows_kernel<D, false>, dim3(grid), dim3(256), lds, stream, a);
}

}  // namespace

void launch_attention(const AttnArgs &a, int head_dim, bool paged, int shift, long long units, bool split,
                      hipStream_t stream) {
  const unsigned grid = (unsigned)(units * a.n_kv_heads);
  if (shift == kAttnTileShift)
    launch_attention_tiles(a, head_dim, paged, grid, stream);
  else
    switch (head_dim) {
      case 64: rows_launch<64>(a, paged, grid, stream); break;
      case 96: rows_launch<96>(a, paged, grid, stream); break;
      case 128: rows_launch<128>(a, paged, grid, stream); break;
      case 160: rows_launch<160>(a, paged, grid, stream); break;
      case 192: rows_launch<192>(a, paged, grid, stream); break;
      case 224: rows_launch<224>(a, paged, grid, stream); break;
      case 256: rows_launch<256>(a, paged, grid, stream); break;
      case 288: rows_launch<288>(a, paged, grid, stream); break;
      case 320: rows_launch<320>(a, paged, grid, stream); break;
      case 352: rows_launch<352>(a, paged, grid, stream); break;
      case 384: rows_launch<384>(a, paged, grid, stream); break;
      case 416: rows_launch<416>(a, paged, grid, stream); break;
      case 448: rows_launch<448>(a, paged, grid, stream); break;
      case 480: rows_launch<480>(a, paged, grid, stream); break;
      case 512: rows_launch<512>(a, paged, grid, stream); break;
    }
  if (split) {
    const unsigned blocks = (unsigned)(a.n_tokens * a.n_kv_heads * a.group);
    const dim3 threads(blocks <= 1024 ? 256 : (head_dim <= 256 ? 64 : 128));
    if (paged)
      enqueue(attention_join_kernel<true>, dim3(blocks), threads, 0, stream, a, head_dim, shift);
    else
      enqueue(attention_join_kernel<false>, dim3(blocks), threads, 0, stream, a, head_dim, shift);
  }
}

}  // namespace v7g
