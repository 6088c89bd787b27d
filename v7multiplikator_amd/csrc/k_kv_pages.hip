// k_kv_pages.hip -- the pages of a binary16 K/V cache, gfx950: rows written into them, sequences forked, freed and
// grown, accepted drafts moved down.  All of it moves bytes or counts pages; nothing is computed but the rounding to
// binary16.
#include "v7g_device.h"
#include "v7g_internal.h"

namespace v7g {

namespace {

typedef unsigned int v2u __attribute__((ext_vector_type(2)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));

// A sequence's position in its pages: the element offset of its row from page 0 of a layer, or -1 on no page.
__device__ __forceinline__ long long row_offset(const v7g_kv_pages &g, int page_shift, const int32_t *table_row,
                                                int width, long long pos) {
  if (pos < 0 || (pos >> page_shift) >= width) return -1;
  const int page = table_row[pos >> page_shift];
  if ((unsigned)page >= (unsigned)g.n_pages) return -1;
  return page * g.page_stride + (pos & ((1 << page_shift) - 1)) * g.token_stride;
}

// ---- K and V rows of tokens, binary32 -> binary16, each to its place

// A thread converts the same 4 elements of a token's K and V row (16-byte loads, 8-byte stores).  Rows below 256
// chunks share a workgroup.
__global__ __launch_bounds__(256) void kv_pack_pages_kernel(v7g_kv_pages g, const float *k_src, const float *v_src,
                                                            long long src_stride, const int32_t *table, int width,
                                                            int n_seqs, const int32_t *positions, const int32_t *seqs,
                                                            int tokens, int chunks, int rows_per_wg, int page_shift) {
  const int sub = rows_per_wg > 1 ? threadIdx.x / chunks : 0;
  const long long t = (long long)blockIdx.x * rows_per_wg + sub;
  if (sub >= rows_per_wg || t >= tokens) return;
  const int seq = seqs ? seqs[t] : (int)t;
  if ((unsigned)seq >= (unsigned)n_seqs) return;
  const long long off = row_offset(g, page_shift, table + (long long)seq * width, width, positions[t]);
  if (off < 0) return;
  for (int j = threadIdx.x - sub * chunks; j < chunks; j += 256) {
    const float4 k = ld_stream4(k_src + t * src_stride + 4 * j);
    const float4 v = ld_stream4(v_src + t * src_stride + 4 * j);
    st_stream_u2(reinterpret_cast<uint32_t *>(g.k + off + 4 * j), pack4_f16(k));
    st_stream_u2(reinterpret_cast<uint32_t *>(g.v + off + 4 * j), pack4_f16(v));
    if (rows_per_wg > 1) break;
  }
}

// ---- accepted drafts moved to the front of their sequence's new tokens

// Lane k's value, whichever lanes take part.
__device__ __forceinline__ long long lane_value(long long v, int k) {
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, k);
  const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), k);
  return (long long)(((unsigned long long)hi << 32) | lo);
}

// Token i of row r's path goes from position len + path[i] to len + i.  A path is strictly ascending, so path[i] >= i
// and moving it in order, 8 rows at a time (all 8 read before one is written), never overwrites a row that is still
// to be read.  A thread takes one unit of the row in one layer, K or V; where the rows lie is worked out once, a lane
// per token of the path, and broadcast.  Bound by the latency of that chain of reads in the small cases.
template <typename U>
__global__ __launch_bounds__(256) void kv_compact_kernel(v7g_kv_pages g, const int32_t *table, int width,
                                                         const int32_t *lens, const int32_t *path, int path_width,
                                                         const int32_t *n_path, int32_t *lens_out, int page_shift,
                                                         int units) {
  const int r = blockIdx.x, lane = threadIdx.x & 63;
  const int32_t *tr = table + (long long)r * width, *p = path + (long long)r * path_width;
  const long long cap = (long long)width << page_shift;
  const int given = n_path[r], ln = lens[r];
  const long long len = ln < 0 ? 0 : (ln > cap ? cap : ln);
  const int want = given < 0 ? 0 : (given > path_width ? path_width : given);
  const unsigned at = blockIdx.y * 256u + threadIdx.x;  // layer, K or V, unit
  const unsigned side = at / (unsigned)units;
  const bool moves = side < 2u * g.n_layers;
  constexpr int E = sizeof(U) / 2;
  uint16_t *base = ((side & 1) ? g.v : g.k) + (moves ? (side >> 1) * g.layer_stride + (at - side * units) * E : 0);
  int n = 0;
  while (n < want) {
    // the path ends at the first entry that does not ascend or has no page to come from or go to
    const int i = n + lane;
    long long src = -1, dst = -1;
    if (i < want) {
      const int from = p[i], before = i ? p[i - 1] : -1;
      if (from > before) {
        src = row_offset(g, page_shift, tr, width, len + from);
        dst = row_offset(g, page_shift, tr, width, len + i);
      }
    }
    const unsigned long long good = __ballot(src >= 0 && dst >= 0);
    const int run = good == ~0ull ? 64 : __builtin_ctzll(~good);
    n += run;
    if (moves)
      for (int i0 = 0; i0 < run; i0 += 8) {
        U v[8];
        long long to[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int k = i0 + j < run ? i0 + j : i0;
          const long long from = lane_value(src, k);
          to[j] = lane_value(dst, k);
          v[j] = *reinterpret_cast<const U *>(base + from);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (i0 + j < run) *reinterpret_cast<U *>(base + to[j]) = v[j];
      }
    if (run < 64) break;
  }
  if (blockIdx.y == 0 && threadIdx.x == 0) lens_out[r] = (int)(len + n);
}

// ---- sequences forked, freed and grown

struct AssignArgs {
  v7g_kv_pages g;
  int32_t *table_out, *lens_out, *refs_out, *short_out;
  const int32_t *table, *lens, *refs, *parents, *reserve;
  int rows, width, page_shift;
  int32_t *keep, *want, *tail;  // per row: pages kept, pages wanted, parent row whose last page is copied or -1
  int32_t *list;                // free pages found
};

// What row r takes over from row par, which holds `held` pages; owner: it takes over the last and spare ones too.
struct AssignRow {
  int n = 0, keep = 0, want = 0, tail = -1;
  __device__ AssignRow() {}
  __device__ AssignRow(const AssignArgs &a, int r, int par, int held, bool owner) {
    const long long cap = (long long)held << a.page_shift;
    const int ln = a.lens[par];
    n = ln < 0 ? 0 : (ln > cap ? (int)cap : ln);
    const int full = n >> a.page_shift, rest = n & ((1 << a.page_shift) - 1);
    keep = owner ? held : full;
    const long long more = a.reserve && a.reserve[r] > 0 ? a.reserve[r] : 0;
    long long w = (n + more + (1 << a.page_shift) - 1) >> a.page_shift;
    if (w > a.width) w = a.width;
    want = (int)(w > keep ? w : keep);
    if (!owner && rest) {
      tail = par;
      if (want < full + 1) want = full + 1;
    }
  }
};

__global__ __launch_bounds__(256) void assign_refs_kernel(AssignArgs a) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < a.g.n_pages) a.refs_out[i] = a.refs[i];
}

// Pages a row holds: its leading entries that name a page.
__device__ int pages_held(const AssignArgs &a, int row, int *scratch) {
  int held = a.width;
  const int32_t *t = a.table + (long long)row * a.width;
  for (int i = threadIdx.x; i < a.width; i += 256)
    if ((unsigned)t[i] >= (unsigned)a.g.n_pages) {
      held = i;
      break;
    }
  if (threadIdx.x == 0) *scratch = a.width;
  __syncthreads();
  if (held < a.width) atomicMin(scratch, held);
  __syncthreads();
  held = *scratch;
  __syncthreads();
  return held;
}

// One workgroup per row: what it takes over, and the counts of the pages it lets go and takes.  Integer atomics: the
// sums do not depend on their order.
__global__ __launch_bounds__(256) void assign_rows_kernel(AssignArgs a) {
  __shared__ int scratch;
  const int r = blockIdx.x;
  int par = a.parents[r];
  if (par < 0 || par >= a.rows) par = -1;
  const int held_r = pages_held(a, r, &scratch);
  AssignRow row;
  if (par >= 0) {
    const int held = par == r ? held_r : pages_held(a, par, &scratch);
    // the parent itself, else the lowest of its children, takes over the last and the spare pages
    bool owner = par == r;
    if (!owner) {
      if (threadIdx.x == 0) scratch = a.parents[par] == par ? 1 : 0;
      __syncthreads();
      for (int i = threadIdx.x; i < r; i += 256)
        if (a.parents[i] == par) atomicOr(&scratch, 1);
      __syncthreads();
      owner = scratch == 0;
    }
    row = AssignRow(a, r, par, held, owner);
  }
  const int32_t *mine = a.table + (long long)r * a.width;
  const int32_t *src = a.table + (long long)(par < 0 ? 0 : par) * a.width;
  int32_t *out = a.table_out + (long long)r * a.width;
  for (int i = threadIdx.x; i < a.width; i += 256) {
    const int old = i < held_r ? mine[i] : -1, now = i < row.keep ? src[i] : -1;
    out[i] = now;
    if (old != now) {
      if (old >= 0) atomicSub(a.refs_out + old, 1);
      if (now >= 0) atomicAdd(a.refs_out + now, 1);
    }
  }
  if (threadIdx.x == 0) {
    a.lens_out[r] = row.n;
    a.keep[r] = row.keep;
    a.want[r] = row.want;
    a.tail[r] = row.tail;
  }
}

// Exclusive sum over the 1024 threads; returns the total in `total`.
__device__ int block_scan(int v, int *scratch, int &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = v;
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 63) scratch[wave] = incl;
  __syncthreads();
  int before = 0, sum = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) before += scratch[w];
    sum += scratch[w];
  }
  __syncthreads();
  total = sum;
  return before + incl - v;
}

// One workgroup: the lowest free pages in order to the rows' requests in order.
__global__ __launch_bounds__(1024) void assign_pages_kernel(AssignArgs a) {
  __shared__ int scratch[16];
  int total = 0;
  for (int r0 = 0; r0 < a.rows; r0 += 1024) {
    const int r = r0 + (int)threadIdx.x;
    int sum;
    (void)block_scan(r < a.rows ? a.want[r] - a.keep[r] : 0, scratch, sum);
    total += sum;
  }
  int found = 0;
  for (long long p0 = 0; p0 < a.g.n_pages && found < total; p0 += 16 * 1024) {
    const long long p = p0 + threadIdx.x * 16;
    unsigned bits = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (p + i < a.g.n_pages && a.refs_out[p + i] <= 0) bits |= 1u << i;
    int sum;
    int at = found + block_scan(__builtin_popcount(bits), scratch, sum);
    for (; bits; bits &= bits - 1, ++at)
      if (at < total) a.list[at] = (int)p + __builtin_ctz(bits);
    found += sum;
  }
  if (found > total) found = total;
  __threadfence_block();
  __syncthreads();
  int base = 0;
  for (int r0 = 0; r0 < a.rows; r0 += 1024) {
    const int r = r0 + (int)threadIdx.x;
    const int keep = r < a.rows ? a.keep[r] : 0, need = r < a.rows ? a.want[r] - keep : 0;
    int sum;
    const int at = base + block_scan(need, scratch, sum);
    base += sum;
    for (int j = 0; j < need && at + j < found; ++j) {
      const int page = a.list[at + j];
      a.table_out[(long long)r * a.width + keep + j] = page;
      a.refs_out[page] = 1;
    }
    // no page for the copy of the last one: the row ends with its full pages
    if (r < a.rows && a.tail[r] >= 0 && at >= found) a.lens_out[r] = keep << a.page_shift;
  }
  if (threadIdx.x == 0) *a.short_out = total - found;
}

// All of the above in one workgroup, the counts in LDS: where they fit, one launch and a few trips to memory instead
// of three launches.
constexpr int kBookPages = 24576, kBookRows = 1024, kBookEntries = 1 << 16;

__global__ __launch_bounds__(1024) void assign_books_kernel(AssignArgs a) {
  __shared__ int scratch[16];
  extern __shared__ int lds[];
  int *held = lds, *owner = held + a.rows, *keeps = owner + a.rows, *refs = keeps + a.rows;
  const int tid = threadIdx.x, P = a.g.n_pages, W = a.width;
  const int lane = tid & 63, wave = tid >> 6;
  for (int p = tid; p < P; p += 1024) refs[p] = a.refs[p];
  int par = -1;
  if (tid < a.rows) {
    par = a.parents[tid];
    if (par >= a.rows || par < 0) par = -1;
    owner[tid] = a.rows;
  }
  // a wave takes 4 rows at a time, their entries side by side in its lanes
  constexpr int R = 4;
  for (int r0 = wave * R; r0 < a.rows; r0 += 16 * R) {
    int h[R];
#pragma unroll
    for (int j = 0; j < R; ++j) h[j] = W;
    for (int c = 0; c < W; c += 64) {
      int page[R];
#pragma unroll
      for (int j = 0; j < R; ++j)
        page[j] = r0 + j < a.rows && c + lane < W ? a.table[(r0 + j) * W + c + lane] : 0;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const unsigned long long none = __ballot(c + lane < W && (unsigned)page[j] >= (unsigned)P);
        if (none && h[j] == W) h[j] = c + __builtin_ctzll(none);
      }
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (r0 + j < a.rows && lane == j) held[r0 + j] = h[j];
  }
  __syncthreads();
  if (par >= 0) atomicMin(owner + par, par == tid ? -1 : tid);
  __syncthreads();
  AssignRow row;
  if (par >= 0) row = AssignRow(a, tid, par, held[par], par == tid || owner[par] == tid);
  __syncthreads();
  if (tid < a.rows) {
    keeps[tid] = row.keep;
    owner[tid] = par;  // from here on, where the row's pages come from
    a.keep[tid] = row.keep;
    a.tail[tid] = row.tail;
  }
  __syncthreads();
  for (int r0 = wave * R; r0 < a.rows; r0 += 16 * R)
    for (int c = 0; c < W; c += 64) {
      int old[R], now[R];
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int r = r0 + j, i = c + lane;
        old[j] = now[j] = -1;
        if (r < a.rows) {
          if (i < held[r]) old[j] = a.table[r * W + i];
          if (i < keeps[r]) now[j] = a.table[owner[r] * W + i];
        }
      }
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (r0 + j < a.rows && c + lane < W) a.table_out[(r0 + j) * W + c + lane] = now[j];
        if (old[j] != now[j]) {
          if (old[j] >= 0) atomicSub(refs + old[j], 1);
          if (now[j] >= 0) atomicAdd(refs + now[j], 1);
        }
      }
    }
  int total;
  const int need = row.want - row.keep;
  const int at = block_scan(need, scratch, total);  // its barriers end the counting too
  int found = 0;
  for (int p0 = 0; p0 < P && found < total; p0 += 16 * 1024) {
    const int p = p0 + tid * 16;
    unsigned bits = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = (i + tid) & 15;  // the lanes' 16 counts lie 16 banks apart: each starts at another of them
      if (p + k < P && refs[p + k] <= 0) bits |= 1u << k;
    }
    int sum;
    int to = found + block_scan(__builtin_popcount(bits), scratch, sum);
    for (; bits; bits &= bits - 1, ++to)
      if (to < total) a.list[to] = p + __builtin_ctz(bits);
    found += sum;
  }
  if (found > total) found = total;
  __threadfence_block();
  __syncthreads();
  for (int j = 0; j < need && at + j < found; ++j) {
    const int page = a.list[at + j];
    a.table_out[tid * a.width + row.keep + j] = page;
    refs[page] = 1;
  }
  // no page for the copy of the last one: the row ends with its full pages
  if (tid < a.rows) a.lens_out[tid] = row.tail >= 0 && at >= found ? row.keep << a.page_shift : row.n;
  if (tid == 0) *a.short_out = total - found;
  __syncthreads();
  for (int p = tid; p < P; p += 1024) a.refs_out[p] = refs[p];
}

// The tokens of the last, partly filled page of a parent copied to its child's own page, in every layer.  The page
// read is kept by the row that took it over, the page written is held by nobody else.
template <typename U>
__global__ __launch_bounds__(256) void assign_copy_kernel(AssignArgs a, int units, int tokens_per_wg) {
  const int r = blockIdx.x, layer = blockIdx.y >> 1;
  const int par = a.tail[r];
  if (par < 0) return;
  const int full = a.keep[r];
  const int rest = a.lens_out[r] - (full << a.page_shift);  // 0: no page was left
  const int t0 = blockIdx.z * tokens_per_wg;
  if (t0 >= rest) return;
  const int n = rest - t0 < tokens_per_wg ? rest - t0 : tokens_per_wg;
  const long long src = a.table[(long long)par * a.width + full], dst = a.table_out[(long long)r * a.width + full];
  uint16_t *base = ((blockIdx.y & 1) ? a.g.v : a.g.k) + layer * a.g.layer_stride + t0 * a.g.token_stride;
  constexpr int E = sizeof(U) / 2;
  for (int i = threadIdx.x; i < n * units; i += 256) {
    const int t = i / units, u = i - t * units;
    const long long off = t * a.g.token_stride + u * E;
    *reinterpret_cast<U *>(base + dst * a.g.page_stride + off) =
        *reinterpret_cast<const U *>(base + src * a.g.page_stride + off);
  }
}

// 16-byte units where every row of every page starts on 16 bytes, else the 8 bytes the pages promise.
bool wide_rows(const v7g_kv_pages &g) {
  return (((uintptr_t)g.k | (uintptr_t)g.v) & 15u) == 0 && g.token_stride % 8 == 0 && g.page_stride % 8 == 0 &&
         g.layer_stride % 8 == 0 && ((long long)g.n_kv_heads * g.head_dim) % 8 == 0;
}

}  // namespace

void launch_kv_pack_pages(const v7g_kv_pages &g, const float *k_src, const float *v_src, long long src_stride,
                          const int32_t *table, int width, int n_seqs, const int32_t *positions, const int32_t *seqs,
                          int tokens, hipStream_t stream) {
  const int chunks = g.n_kv_heads * g.head_dim / 4;
  const int per = chunks >= 256 ? 1 : 256 / chunks;
  enqueue(kv_pack_pages_kernel, dim3((unsigned)((tokens + per - 1) / per)), dim3(256), 0, stream, g, k_src, v_src,
          src_stride, table, width, n_seqs, positions, seqs, tokens, chunks, per, __builtin_ctz((unsigned)g.page_size));
}

void launch_kv_compact(const v7g_kv_pages &g, const int32_t *table, int width, int rows, const int32_t *lens,
                       const int32_t *path, int path_width, const int32_t *n_path, int32_t *lens_out,
                       hipStream_t stream) {
  const bool wide = wide_rows(g);
  const int units = g.n_kv_heads * g.head_dim / (wide ? 8 : 4);
  const dim3 grid((unsigned)rows, (unsigned)((2LL * g.n_layers * units + 255) / 256));
  const int shift = __builtin_ctz((unsigned)g.page_size);
  if (wide)
    enqueue(kv_compact_kernel<v4u>, grid, dim3(256), 0, stream, g, table, width, lens, path, path_width, n_path,
            lens_out, shift, units);
  else
    enqueue(kv_compact_kernel<v2u>, grid, dim3(256), 0, stream, g, table, width, lens, path, path_width, n_path,
            lens_out, shift, units);
}

long long kv_assign_workspace(int rows, int n_pages) { return 4LL * (3LL * rows + n_pages); }

void launch_kv_assign(const v7g_kv_pages &g, int32_t *table_out, int32_t *lens_out, int32_t *refs_out,
                      int32_t *short_out, const int32_t *table, const int32_t *lens, const int32_t *refs,
                      const int32_t *parents, const int32_t *reserve, int rows, int width, void *workspace,
                      hipStream_t stream) {
  AssignArgs a{g, table_out, lens_out, refs_out, short_out, table, lens, refs, parents, reserve, rows, width};
  a.page_shift = __builtin_ctz((unsigned)g.page_size);
  a.keep = static_cast<int32_t *>(workspace);
  a.want = a.keep + rows;
  a.tail = a.want + rows;
  a.list = a.tail + rows;
  if (g.n_pages <= kBookPages && rows <= kBookRows && (long long)rows * width <= kBookEntries) {
    enqueue(assign_books_kernel, dim3(1), dim3(1024), (unsigned)(4 * (3 * rows + g.n_pages)), stream, a);
  } else {
    if (g.n_pages)
      enqueue(assign_refs_kernel, dim3((unsigned)((g.n_pages + 255) / 256)), dim3(256), 0, stream, a);
    if (rows) enqueue(assign_rows_kernel, dim3((unsigned)rows), dim3(256), 0, stream, a);
    enqueue(assign_pages_kernel, dim3(1), dim3(1024), 0, stream, a);
  }
  if (!rows || !g.n_pages) return;
  const bool wide = wide_rows(g);
  const int units = g.n_kv_heads * g.head_dim / (wide ? 8 : 4);
  const int per = 16;  // tokens of a workgroup
  const dim3 grid((unsigned)rows, (unsigned)(2 * g.n_layers), (unsigned)((g.page_size + per - 1) / per));
  if (wide)
    enqueue(assign_copy_kernel<v4u>, grid, dim3(256), 0, stream, a, units, per);
  else
    enqueue(assign_copy_kernel<v2u>, grid, dim3(256), 0, stream, a, units, per);
}

}  // namespace v7g
