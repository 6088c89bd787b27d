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
    *reinterpret_cast<uint2 *>(g.k + off + 4 * j) = pack4_f16(k);
    *reinterpret_cast<uint2 *>(g.v + off + 4 * j) = pack4_f16(v);
    if (rows_per_wg > 1) break;
  }
}

// ---- accepted drafts moved to the front of their sequence's new tokens

// Token i of row r's path goes from position len + path[i] to len + i.  A path is strictly ascending, so path[i] >= i
// and moving it in order, 8 rows at a time (all 8 read before one is written), never overwrites a row that is still
// to be read.  A workgroup takes one sequence, one layer, K or V, and 256 units of the row.
template <typename U>
__global__ __launch_bounds__(256) void kv_compact_kernel(v7g_kv_pages g, const int32_t *table, int width,
                                                         const int32_t *lens, const int32_t *path, int path_width,
                                                         const int32_t *n_path, int32_t *lens_out, int page_shift,
                                                         int units) {
  const int r = blockIdx.x, layer = blockIdx.y >> 1;
  const int lane = threadIdx.x & 63;
  const int32_t *tr = table + (long long)r * width, *p = path + (long long)r * path_width;
  const long long cap = (long long)width << page_shift;
  const long long len = lens[r] < 0 ? 0 : (lens[r] > cap ? cap : lens[r]);
  int want = n_path[r] < 0 ? 0 : (n_path[r] > path_width ? path_width : n_path[r]);
  // the path ends at the first entry that does not ascend or has no page to come from or go to
  int n = 0;
  while (n < want) {
    const int i = n + lane;
    bool ok = false;
    if (i < want) {
      const int from = p[i], before = i ? p[i - 1] : -1;
      ok = from > before && row_offset(g, page_shift, tr, width, len + from) >= 0 &&
           row_offset(g, page_shift, tr, width, len + i) >= 0;
    }
    const unsigned long long good = __ballot(ok);
    const int run = good == ~0ull ? 64 : __builtin_ctzll(~good);
    n += run;
    if (run < 64) break;
  }
  if (blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) lens_out[r] = (int)(len + n);
  const int u = blockIdx.z * 256 + threadIdx.x;
  if (u >= units) return;
  uint16_t *base = ((blockIdx.y & 1) ? g.v : g.k) + layer * g.layer_stride;
  constexpr int E = sizeof(U) / 2;
  for (int i0 = 0; i0 < n; i0 += 8) {
    U v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < n && p[i0 + i] != i0 + i)
        v[i] = *reinterpret_cast<const U *>(base + row_offset(g, page_shift, tr, width, len + p[i0 + i]) + u * E);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < n && p[i0 + i] != i0 + i)
        *reinterpret_cast<U *>(base + row_offset(g, page_shift, tr, width, len + i0 + i) + u * E) = v[i];
  }
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
  int keep = 0, want = 0, tail = -1, n = 0;
  if (par >= 0) {
    const int held = par == r ? held_r : pages_held(a, par, &scratch);
    const long long cap = (long long)held << a.page_shift;
    const int ln = a.lens[par];
    n = ln < 0 ? 0 : (ln > cap ? (int)cap : ln);
    const int full = n >> a.page_shift, rest = n & ((1 << a.page_shift) - 1);
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
    keep = owner ? held : full;
    const long long more = a.reserve ? (a.reserve[r] > 0 ? a.reserve[r] : 0) : 0;
    long long w = (n + more + (1 << a.page_shift) - 1) >> a.page_shift;
    if (w > a.width) w = a.width;
    want = (int)(w > keep ? w : keep);
    if (!owner && rest) {
      tail = par;
      if (want < full + 1) want = full + 1;
    }
  }
  const int32_t *mine = a.table + (long long)r * a.width;
  const int32_t *src = a.table + (long long)(par < 0 ? 0 : par) * a.width;
  int32_t *out = a.table_out + (long long)r * a.width;
  for (int i = threadIdx.x; i < a.width; i += 256) {
    const int old = i < held_r ? mine[i] : -1, now = i < keep ? src[i] : -1;
    out[i] = now;
    if (old != now) {
      if (old >= 0) atomicSub(a.refs_out + old, 1);
      if (now >= 0) atomicAdd(a.refs_out + now, 1);
    }
  }
  if (threadIdx.x == 0) {
    a.lens_out[r] = n;
    a.keep[r] = keep;
    a.want[r] = want;
    a.tail[r] = tail;
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
  const dim3 grid((unsigned)rows, (unsigned)(2 * g.n_layers), (unsigned)((units + 255) / 256));
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
  if (g.n_pages)
    enqueue(assign_refs_kernel, dim3((unsigned)((g.n_pages + 255) / 256)), dim3(256), 0, stream, a);
  if (rows) enqueue(assign_rows_kernel, dim3((unsigned)rows), dim3(256), 0, stream, a);
  enqueue(assign_pages_kernel, dim3(1), dim3(1024), 0, stream, a);
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
