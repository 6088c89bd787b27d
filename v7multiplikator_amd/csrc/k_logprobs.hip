// k_logprobs.hip -- log probabilities of given tokens, entropy and the most likely tokens of logit rows, gfx950.
//
//   logprob = x_id - m - log s,  entropy = log s - w / s,  s = sum e^(x-m), w = sum e^(x-m) (x-m),  m = max x
//
// One pass over the logits, which is what bounds it: each lane keeps its own running maximum and sums (a new maximum
// scales s and moves w: w' = a (w + s (m - m'))), and each wave the K best of what it has read.  A token is ordered by
// one 64-bit key, the value's bits made monotonic above the complement of its index, so equal values fall to the
// lower index, -0 and denormals (flushed, as everywhere in this library) equal 0, and NaN comes first.  A wave reads 1024
// logits at a time; those above a bar that K logits are known to reach (first the K-th best of the 64 lanes' best) are
// collected in LDS, and ranked by counting, which raises the bar, when half as many again have come together and at the
// end.  A row goes to as many workgroups as fill the chip; a second kernel then joins their results.
#include "v7g_device.h"
#include "v7g_internal.h"

namespace v7g {

namespace {

constexpr int kChunk = 1024;  // logits of one step of a wave, 16 a lane
constexpr int kBest = 64;     // at most so many alternatives
constexpr int kRoom = 128;    // keys that wait to be ranked
constexpr int kBuffer = kRoom + kChunk + 8 + kBest;  // a wave's keys: waiting, one step's, padding, the new list
typedef unsigned long long Key;
typedef float f4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// Never 0, which stands for no token.
__device__ __forceinline__ Key make_key(float x, unsigned index) {
  uint32_t b = __builtin_bit_cast(uint32_t, x);
  if ((b & 0x7f800000u) == 0) b = 0;
  b = (b & 0x7fffffffu) > 0x7f800000u ? 0xffffffffu : ((b & 0x80000000u) ? ~b : b | 0x80000000u);
  return ((Key)b << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float key_value(Key k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __builtin_bit_cast(float, b == 0xffffffffu ? 0x7fc00000u : ((b & 0x80000000u) ? b & 0x7fffffffu : ~b));
}
__device__ __forceinline__ int key_index(Key k) { return (int)(0xffffffffu - (uint32_t)k); }

__device__ __forceinline__ void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// The K-th largest of the lanes' keys: the largest that K lanes reach, bit by bit; the lower half only where values
// tie.
__device__ __forceinline__ Key kth_of_lanes(Key mine, int K) {
  const uint32_t hi = (uint32_t)(mine >> 32);
  uint32_t t = 0;
  for (int b = 31; b >= 0; --b) {
    const uint32_t c = t | (1u << b);
    if (__popcll(__ballot(hi >= c)) >= K) t = c;
  }
  Key key = (Key)t << 32;
  if (__popcll(__ballot(hi >= t)) == K) return key;
  for (int b = 31; b >= 0; --b) {
    const Key c = key | (1ull << b);
    if (__popcll(__ballot(mine >= c)) >= K) key = c;
  }
  return key;
}

// A wave's best keys, in LDS: the K best of all it was given are among the n that wait there.
struct Best {
  Key *buf;
  int K, n = 0;
  float bar = -__builtin_inff();  // K keys with this value or a larger one are there (NaN counts as the largest)
  bool full = false;              // the bar stands
  bool sorted = false;

  // The keys of the lanes that have one to give join the n that wait.
  __device__ __forceinline__ void push(bool mine, Key k) {
    const unsigned long long hit = __ballot(mine);
    if (!hit) return;
    if (mine)
      buf[n + __builtin_amdgcn_mbcnt_hi((unsigned)(hit >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)hit, 0))] = k;
    n += __popcll(hit);
    sorted = false;
  }

  // Keys of one step, N a lane, 0 for none, in any order.
  template <int N>
  __device__ __forceinline__ void add(const Key (&k)[N]) {
    Key top = k[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = k[i] > top ? k[i] : top;
    Key least = kth_of_lanes(top, K);
    least = least > 1 ? least : 1;
    if (full) {  // the keys that wait already hold the K best so far
      const Key worst = sorted ? buf[K - 1] : 0;
      least = worst + 1 > least ? worst + 1 : least;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) push(k[i] >= least, k[i]);
    settle();
  }

  // Values of one step in rising order of their indices, of which those above the bar count.
  template <int N, class F>
  __device__ __forceinline__ void add_above(const float (&v)[N], F key) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool mine = !(v[i] <= bar);  // NaN too
      if (__ballot(mine)) push(mine, mine ? key(i) : 0);
    }
    settle();
  }

  __device__ __forceinline__ void settle() {
    // a higher bar saves looks, each ranking costs about one (1500 rows of 128256, 20 alternatives: ranked from K/2 + 4
    // waiting on 159 us, from 128 keys on 185)
    if (n > K + K / 2 + 4 || (!full && n >= K)) rank();
  }

  // The K best of the n keys, sorted, to the front.
  __device__ __forceinline__ void rank() {
    Key *fresh = buf + kRoom + kChunk + 8;
    const int lane = __lane_id();
    if (lane < 8) buf[n + lane] = 0;  // read 8 at a time
    wave_lds_fence();
    for (int i0 = 0; i0 < n; i0 += 64) {
      const int i = i0 + lane;
      const Key mine = i < n ? buf[i] : 0;
      int r = 0;
      for (int j = 0; j < n; j += 8) {
        Key o[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) o[x] = buf[j + x];
#pragma unroll
        for (int x = 0; x < 8; ++x) r += o[x] > mine;
      }
      if (i < n && r < K) fresh[r] = mine;
    }
    wave_lds_fence();
    n = n < K ? n : K;
    if (lane < n) buf[lane] = fresh[lane];
    wave_lds_fence();
    sorted = true;
    if (n == K) {
      full = true;
      bar = key_value(buf[K - 1]);
    }
  }
};

struct Sums {
  float m = -__builtin_inff(), s = 0.0f, w = 0.0f;
  // Moves the sums to another maximum nm >= m.
  __device__ __forceinline__ void move(float nm) {
    if (nm > m) {
      if (m > -__builtin_inff()) {
        const float d = m - nm, a = __expf(d);
        w = a > 0.0f ? a * (w + s * d) : 0.0f;
        s *= a;
      }
      m = nm;
    }
  }
  __device__ __forceinline__ void join(float m2, float s2, float w2) {
    Sums o;
    o.m = m2, o.s = s2, o.w = w2;
    const float nm = fmaxf(m, m2);
    move(nm);
    o.move(nm);
    s += o.s;
    w += o.w;
  }
  __device__ __forceinline__ void join_lanes() {
    for (int x = 32; x; x >>= 1) {
      const float m2 = xor_f(m, x), s2 = xor_f(s, x), w2 = xor_f(w, x);
      join(m2, s2, w2);
    }
  }
};

struct LogprobArgs {
  float *logprob, *entropy, *top_logprob;
  int32_t *top_ids;
  const float *logits;
  long long stride;
  const int32_t *ids;
  int vocab, K, parts, steps;  // steps: 4-wave steps of a part
  float *part_sums;            // [row, part, 4]
  Key *part_keys;              // [row, part, K]
};

__device__ __forceinline__ void write_row(const LogprobArgs &a, long long row, const Sums &t, const Key *best) {
  const float lse = logf(t.s);
  const int lane = __lane_id();
  if (lane == 0) {
    const int id = a.ids[row];
    float lp = __builtin_nanf("");  // no such token
    if (id >= 0 && id < a.vocab) lp = (a.logits[row * a.stride + id] - t.m) - lse;
    a.logprob[row] = lp;
    a.entropy[row] = lse - t.w / t.s;
  }
  if (lane < a.K) {
    a.top_logprob[row * a.K + lane] = (key_value(best[lane]) - t.m) - lse;
    a.top_ids[row * a.K + lane] = key_index(best[lane]);
  }
}

template <bool TOP>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobArgs a) {
  __shared__ alignas(16) Key keys[TOP ? 4 : 1][TOP ? kBuffer : 1];
  __shared__ float sums[4][3];
  __shared__ int counts[4];
  __shared__ Key joined[TOP ? kBest : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const float *x = a.logits + row * a.stride;
  Sums t;
  Best best{keys[TOP ? wave : 0], a.K};
  long long at = ((long long)part * a.steps * 4 + wave) * kChunk + lane * 4;
  auto load = [&](long long p, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long q = p + i * 256;
      if (q + 4 <= a.vocab) {
        const f4_a4 y = __builtin_nontemporal_load(reinterpret_cast<const f4_a4 *>(x + q));
#pragma unroll
        for (int c = 0; c < 4; ++c) v[4 * i + c] = y[c];
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[4 * i + c] = q + c < a.vocab ? x[q + c] : -__builtin_inff();
      }
    }
  };
  float v[16], nv[16];
  load(at, v);
  for (int st = 0; st < a.steps; ++st, at += 4 * kChunk) {
    if (at - lane * 4 >= a.vocab) break;
    if (st + 1 < a.steps) load(at + 4 * kChunk, nv);
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, v[i]);
    t.move(fmaxf(t.m, mx));
    const float ref = t.m == -__builtin_inff() ? 0.0f : t.m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float z = v[i] - ref, e = __expf(z);  // NaN and +Inf make s NaN, and with it every result of the row
      t.s += e;
      t.w += e > 0.0f ? e * z : 0.0f;
    }
    if constexpr (TOP) {
      auto key = [&](int i) { return make_key(v[i], (unsigned)(at + (i >> 2) * 256 + (i & 3))); };
      if (!best.full) {
        Key k[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) k[i] = at + (i >> 2) * 256 + (i & 3) < a.vocab ? key(i) : 0;
        best.add(k);
      } else if (__ballot(!(mx <= best.bar) || !(t.s == t.s))) {
        best.add_above(v, key);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = nv[i];
  }
  t.join_lanes();
  if constexpr (TOP)
    if (!best.sorted) best.rank();
  if (lane == 0) {
    sums[wave][0] = t.m, sums[wave][1] = t.s, sums[wave][2] = t.w;
    counts[wave] = best.n;
  }
  __syncthreads();
  int n = 0;  // the waves' lists together
  if constexpr (TOP) {
    // a key's place is its place in its own list and those of the larger ones in the other three, by bisection
    const Key mine = lane < best.n ? best.buf[lane] : 0;
    int place = lane;
    for (int o = 1; o < 4; ++o) {
      const int w = (wave + o) & 3;
      int lo = 0, hi = counts[w];
      while (__ballot(lo < hi)) {
        const int mid = (lo + hi) >> 1;
        const bool larger = lo < hi && keys[w][mid] > mine;
        if (lo < hi) {
          if (larger)
            lo = mid + 1;
          else
            hi = mid;
        }
      }
      place += lo;
    }
    if (lane < best.n && place < a.K) joined[place] = mine;
    n = counts[0] + counts[1] + counts[2] + counts[3];
    __syncthreads();
  }
  if (wave != 0) return;
  for (int w = 1; w < 4; ++w) t.join(sums[w][0], sums[w][1], sums[w][2]);
  if (a.parts == 1) {
    write_row(a, row, t, joined);
    return;
  }
  const long long slot = row * a.parts + part;
  if (lane == 0) {
    float *p = a.part_sums + slot * 4;
    p[0] = t.m, p[1] = t.s, p[2] = t.w;
  }
  if (TOP && lane < a.K) a.part_keys[slot * a.K + lane] = lane < n ? joined[lane] : 0;
}

template <bool TOP>
__global__ __launch_bounds__(64) void logprobs_join_kernel(LogprobArgs a) {
  __shared__ alignas(16) Key keys[TOP ? kBuffer : 1];
  const int lane = threadIdx.x;
  const long long row = blockIdx.x;
  Sums t;
  for (int p = lane; p < a.parts; p += 64) {
    const float *q = a.part_sums + (row * a.parts + p) * 4;
    t.join(q[0], q[1], q[2]);
  }
  t.join_lanes();
  Best best{keys, a.K};
  if constexpr (TOP) {
    const Key *in = a.part_keys + row * a.parts * a.K;
    const int n = a.parts * a.K;
    for (int i0 = 0; i0 < n; i0 += kChunk) {
      Key k[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) k[i] = i0 + i * 64 + lane < n ? in[i0 + i * 64 + lane] : 0;
      best.add(k);
    }
    if (!best.sorted) best.rank();
  }
  write_row(a, row, t, best.buf);
}

}  // namespace

// Parts of a row: one workgroup for each from 1024 rows on (1000 rows of 151936, 5 alternatives: one part 107 us, two
// 129 to 135), as many as make 1024 workgroups below (64 rows: 16 parts 23 us, 32 26), no part smaller than one step of
// four waves.
int logprobs_parts(int rows, int vocab) {
  const long long steps = ((long long)vocab + 4 * kChunk - 1) / (4 * kChunk);
  const long long parts = rows > 0 && rows < 1024 ? 1024 / rows : 1;
  return (int)(parts < steps ? parts : steps);
}

long long logprobs_workspace(int rows, int vocab, int top_k) {
  const int parts = logprobs_parts(rows, vocab);
  return parts == 1 ? 0 : (long long)rows * parts * (16 + 8LL * top_k);
}

void launch_token_logprobs(float *logprob, float *entropy, float *top_logprob, int32_t *top_ids, const float *logits,
                           long long stride, const int32_t *ids, int rows, int vocab, int top_k, void *workspace,
                           hipStream_t stream) {
  LogprobArgs a{logprob, entropy, top_logprob, top_ids, logits, stride, ids, vocab, top_k};
  const long long steps = ((long long)vocab + 4 * kChunk - 1) / (4 * kChunk);
  a.parts = logprobs_parts(rows, vocab);
  a.steps = (int)((steps + a.parts - 1) / a.parts);
  a.parts = (int)((steps + a.steps - 1) / a.steps);
  a.part_sums = static_cast<float *>(workspace);
  a.part_keys = reinterpret_cast<Key *>(a.part_sums + (long long)rows * a.parts * 4);
  const dim3 grid((unsigned)((long long)rows * a.parts));
  if (top_k)
    enqueue(logprobs_kernel<true>, grid, dim3(256), 0, stream, a);
  else
    enqueue(logprobs_kernel<false>, grid, dim3(256), 0, stream, a);
  if (a.parts == 1) return;
  if (top_k)
    enqueue(logprobs_join_kernel<true>, dim3((unsigned)rows), dim3(64), 0, stream, a);
  else
    enqueue(logprobs_join_kernel<false>, dim3((unsigned)rows), dim3(64), 0, stream, a);
}

}  // namespace v7g
