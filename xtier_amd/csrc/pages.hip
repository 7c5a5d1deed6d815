// Page bookkeeping of a paged cache: growing, forking, freeing and compacting the rows of a page table, and copying
// pages of every layer. Definitions in include/xtier_amd.h. Tables, counts and lengths are int32 on the device, so a
// captured step replays with whatever they hold.
//
// The free pages that a call takes are the lowest-numbered ones, in ascending order: one workgroup of 1024 threads
// counts them in 1024 contiguous spans (16-byte loads), scans the counts and then knows the rank of each. The state is
// a few hundred KB at most, so one CU reads it in a few microseconds and no second launch has to join partial counts.
#include "xt_common.h"
#include "xt_host.h"

namespace xt {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kScanWaves = kScanThreads / 64;

// Sums of x over the workgroup's threads before this one, and over all (both below 2^31). `s` holds kScanWaves values of
// the caller.
__device__ inline int block_exclusive(int x, int* s, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int upto = wave_inclusive_sum(x);
  __syncthreads();                       // earlier readers of s are done
  if (lane == 63) s[wave] = upto;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kScanWaves; ++w) {
    const int v = s[w];
    if (w < wave) before += v;
    all += v;
  }
  *total = all;
  return before + upto - x;
}

// The pages of this thread: [lo, hi), spans of a multiple of 4 pages.
__device__ inline void span_of(int64_t pages, int64_t* lo, int64_t* hi) {
  const int64_t per = ((pages + kScanThreads - 1) / kScanThreads + 3) / 4 * 4;
  const int64_t l = per * (int64_t)threadIdx.x;
  *lo = l < pages ? l : pages;
  *hi = l + per < pages ? l + per : pages;
}

__device__ inline int count_free(const int32_t* refs, int64_t lo, int64_t hi) {
  int n = 0;
  for (int64_t p = lo; p < hi; ++p) n += refs[p] == 0;
  return n;
}

// Each row b grows by add[b] tokens (see xt_pages_extend). One workgroup.
__global__ __launch_bounds__(kScanThreads) void extend_kernel(int32_t* refs, int64_t pages, int32_t* table,
                                                               int64_t table_stride, int width, int32_t* lens,
                                                               const int32_t* add, int rows, int page_shift,
                                                               uint8_t* granted, int32_t* free_list,
                                                               int64_t free_cap) {
  __shared__ int s[kScanWaves];
  int64_t lo, hi;
  int n_free;
  span_of(pages, &lo, &hi);
  const int mine = count_free(refs, lo, hi);
  int64_t rank = block_exclusive(mine, s, &n_free);
  // the free list, as far as any row may need it (free_cap entries): rank -> page
  for (int64_t p = lo; p < hi && rank < free_cap; ++p)
    if (refs[p] == 0) free_list[rank++] = (int32_t)p;
  __syncthreads();   // the list is written and every count of refs == 0 is read before any refs changes
  const int64_t mask = (1 << page_shift) - 1;
  __shared__ int s_upto[kScanThreads];         // pages needed by this round's rows up to and with this one
  __shared__ int32_t s_col[kScanThreads];      // the first new column of a granted row, -1 for one that gets none
  int64_t base = 0;                            // pages needed by the rows of earlier rounds
  for (int r0 = 0; r0 < rows; r0 += kScanThreads) {
    const int r = r0 + (int)threadIdx.x;
    int64_t c0 = 0, c1 = 0, len = 0, grow = 0;
    bool fits = false;
    if (r < rows) {
      len = lens[r];
      grow = add[r];
      c0 = (len + mask) >> page_shift;
      c1 = (len + grow + mask) >> page_shift;
      fits = len >= 0 && grow >= 0 && c1 <= width && len + grow <= 0x7FFFFFFF;
    }
    const int need = fits ? (int)(c1 - c0) : 0;    // (1024 rows of at most 2^21 - 1 columns, which the host sees to)
    int round;
    const int from = block_exclusive(need, s, &round);
    const bool granted_here = fits && (need == 0 || base + from + need <= n_free);
    s_upto[threadIdx.x] = from + need;
    s_col[threadIdx.x] = granted_here ? (int32_t)c0 : -1;
    if (r < rows) {
      if (granted_here) lens[r] = (int32_t)(len + grow);
      granted[r] = granted_here ? 1 : 0;
    }
    __syncthreads();
    // one thread a page, whichever row it belongs to: the first whose running need passes it
    for (int j = (int)threadIdx.x; j < round && base + j < n_free; j += kScanThreads) {
      int at = 0;
#pragma unroll
      for (int step = kScanThreads / 2; step > 0; step >>= 1)
        if (s_upto[at + step - 1] <= j) at += step;
      if (s_col[at] < 0) continue;
      const int32_t p = free_list[base + j];
      table[(int64_t)(r0 + at) * table_stride + s_col[at] + (j - (at ? s_upto[at - 1] : 0))] = p;
      refs[p] = 1;
    }
    base += round;
    __syncthreads();
  }
}

// One column of a child's row: the parent's full pages, which gain a reference, then the new page, then none.
__device__ inline void fork_cell(int32_t* refs, int64_t pages, int32_t* table, int64_t table_stride, int c,
                                 int32_t parent, int32_t child, int32_t full, int32_t dst) {
  int32_t p = -1;
  if (c < full) {
    p = table[(int64_t)parent * table_stride + c];
    if (p >= 0 && p < pages) atomicAdd(&refs[p], 1);
  } else if (c == full) {
    p = dst;
  }
  table[(int64_t)child * table_stride + c] = p;
}

// Checks each fork, finds its page for the unfinished one and writes its moves and lengths. Then the children's rows, if
// `plan` is NULL; else per fork {parent row or -1, pages shared, destination page or -1} for fork_rows_kernel. One
// workgroup: up to XT_PAGES_FORK_CELLS columns a second launch costs more than it gains (32 forks of 66 columns: 34 us with
// the copy of 12 layers and the rest of a step, 31 in one).
__global__ __launch_bounds__(kScanThreads) void fork_kernel(int32_t* refs, int64_t pages, int32_t* table,
                                                             int64_t table_stride, int width, int32_t* lens, int rows,
                                                             int page_shift, const int32_t* parents,
                                                             const int32_t* children, int n, int32_t* moves,
                                                             int64_t moves_stride, int32_t* plan) {
  __shared__ int s[kScanWaves];
  __shared__ int32_t s_child[kScanThreads], s_free[kScanThreads], s_plan[3][kScanThreads];
  int64_t lo, hi;
  int n_free, n_need;
  span_of(pages, &lo, &hi);
  const int i = (int)threadIdx.x;
  const bool mine = i < n;
  const int32_t parent = mine ? parents[i] : -1, child = mine ? children[i] : -1;
  s_child[i] = child;
  bool ok = mine && parent >= 0 && parent < rows && child >= 0 && child < rows;
  int64_t len = 0;
  if (ok) {
    len = lens[parent] > 0 ? lens[parent] : 0;
    ok = lens[child] == 0;
  }
  const int n_mine = count_free(refs, lo, hi);
  int rank = block_exclusive(n_mine, s, &n_free);
  for (int64_t p = lo; p < hi && rank < n; ++p)
    if (refs[p] == 0) s_free[rank++] = (int32_t)p;
  for (int j = 0; j < i && ok; ++j) ok = s_child[j] != child;   // a child takes its first fork
  const int64_t full = len >> page_shift;
  const bool need = ok && (len & ((1 << page_shift) - 1)) != 0;
  const int at = block_exclusive(need ? 1 : 0, s, &n_need);   // (its barriers: every lens is read before any is written)
  const int32_t dst = need && at < n_free && full < width ? s_free[at] : -1;
  if (mine) {
    moves[i] = dst >= 0 ? table[(int64_t)parent * table_stride + full] : -1;
    moves[moves_stride + i] = dst;
    if (ok) lens[child] = (int32_t)(need && dst < 0 ? full << page_shift : len);
    if (dst >= 0) refs[dst] = 1;
  }
  const int32_t shared = (int32_t)(full < width ? full : width);
  if (plan) {
    if (mine) {
      plan[3 * i] = ok ? parent : -1;
      plan[3 * i + 1] = shared;
      plan[3 * i + 2] = dst;
    }
    return;
  }
  s_plan[0][i] = ok ? parent : -1;
  s_plan[1][i] = shared;
  s_plan[2][i] = dst;
  __syncthreads();
  // (a row that is both a parent and a child held no tokens: none of its columns is read)
  for (int k = i; k < n * width; k += kScanThreads) {
    const int f = k / width;
    if (s_plan[0][f] >= 0)
      fork_cell(refs, pages, table, table_stride, k % width, s_plan[0][f], s_child[f], s_plan[1][f], s_plan[2][f]);
  }
}

// The table rows of the children. grid (n, column chunks).
__global__ __launch_bounds__(256) void fork_rows_kernel(int32_t* refs, int64_t pages, int32_t* table,
                                                         int64_t table_stride, int width, const int32_t* children,
                                                         const int32_t* plan) {
  const int i = (int)blockIdx.x;
  if (plan[3 * i] < 0) return;
  for (int c = (int)(blockIdx.y * 256 + threadIdx.x); c < width; c += (int)gridDim.y * 256)
    fork_cell(refs, pages, table, table_stride, c, plan[3 * i], children[i], plan[3 * i + 1], plan[3 * i + 2]);
}

// grid (n, column chunks): each entry of the row is taken by one thread (the exchange), whose count it gives back, so
// a row named twice is freed once.
__global__ __launch_bounds__(256) void free_kernel(int32_t* refs, int64_t pages, int32_t* table, int64_t table_stride,
                                                    int width, int32_t* lens, int rows, const int32_t* which) {
  const int32_t r = which[blockIdx.x];
  if (r < 0 || r >= rows) return;
  for (int c = (int)(blockIdx.y * 256 + threadIdx.x); c < width; c += (int)gridDim.y * 256) {
    const int32_t p = atomicExch(&table[(int64_t)r * table_stride + c], -1);
    if (p >= 0 && p < pages) atomicSub(&refs[p], 1);
  }
  if (blockIdx.y == 0 && threadIdx.x == 0) lens[r] = 0;
}

// The moves of a compaction, the reference counts after it, and for every page at or above the mark (the number of pages
// in use) where it is afterwards: map[page]. One workgroup.
__global__ __launch_bounds__(kScanThreads) void compact_plan_kernel(int32_t* refs, int64_t pages, int32_t* moves,
                                                                     int64_t half, int32_t* count, int32_t* map) {
  __shared__ int s[kScanWaves];
  int64_t lo, hi;
  int live, n_src;
  span_of(pages, &lo, &hi);
  int used = 0;
  for (int64_t p = lo; p < hi; ++p) used += refs[p] > 0;
  const int used_before = block_exclusive(used, s, &live);
  // pages of this span in use at or above the mark, and free below it; those before the span follow from `used_before`
  int src = 0;
  for (int64_t p = max(lo, (int64_t)live); p < hi; ++p) src += refs[p] > 0;
  int64_t rs = block_exclusive(src, s, &n_src), rd = lo - used_before;
  for (int64_t p = lo; p < hi; ++p) {
    const bool u = refs[p] > 0;
    if (p >= live) {
      map[p] = u ? -1 : (int32_t)p;
      if (u) moves[rs++] = (int32_t)p;
    } else if (!u) {
      moves[half + rd++] = (int32_t)p;
    }
  }
  // n_src <= pages / 2: as many pages in use lie above the mark as free ones below it
  for (int64_t i = n_src + threadIdx.x; i < half; i += kScanThreads) moves[i] = moves[half + i] = -1;
  if (threadIdx.x == 0) *count = (int32_t)n_src;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < n_src; i += kScanThreads) {
    const int32_t a = moves[i], b = moves[half + i];
    map[a] = b;
    refs[b] = refs[a];
    refs[a] = 0;
  }
}

// Table entries of moved pages: none lies below the first source, and from there on map holds every page.
__global__ __launch_bounds__(256) void compact_rows_kernel(int64_t pages, int32_t* table, int64_t table_stride,
                                                            int width, int rows, const int32_t* moves, const int32_t* count,
                                                            const int32_t* map) {
  const int n = *count;
  if (n == 0) return;
  const int32_t first = moves[0];
  const int64_t cells = (int64_t)rows * width;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (int64_t)gridDim.x * 256) {
    int32_t* cell = table + (i / width) * table_stride + i % width;
    const int32_t p = *cell;
    if (p >= first && p < pages) *cell = map[p];
  }
}

struct CopyArgs {
  uint8_t* base[XT_PAGES_COPY_MAX];
  int64_t stride[XT_PAGES_COPY_MAX];
  int64_t bytes[XT_PAGES_COPY_MAX];
  int64_t pages[XT_PAGES_COPY_MAX];
};

// grid (moves, buffers, chunks of a page): 16-byte pieces where a buffer's pages are aligned for them, else bytes.
__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a, const int32_t* moves, int64_t moves_stride, int n,
                                                    const int32_t* count) {
  const int buf = (int)blockIdx.y;
  const int limit = count ? min(n, *count) : n;
  const int64_t bytes = a.bytes[buf];
  const bool wide = (((uint64_t)a.base[buf] | (uint64_t)a.stride[buf]) & 15) == 0;
  const int64_t pieces = wide ? bytes / 16 : 0;
  const int64_t first = (int64_t)blockIdx.z * 256 + threadIdx.x, step = (int64_t)gridDim.z * 256;
  for (int i = (int)blockIdx.x; i < limit; i += (int)gridDim.x) {
    const int32_t src = moves[i], dst = moves[moves_stride + i];
    if (src < 0 || dst < 0 || src >= a.pages[buf] || dst >= a.pages[buf]) continue;
    const uint8_t* from = a.base[buf] + (int64_t)src * a.stride[buf];
    uint8_t* to = a.base[buf] + (int64_t)dst * a.stride[buf];
    for (int64_t p = first; p < pieces; p += step)
      reinterpret_cast<uint4*>(to)[p] = reinterpret_cast<const uint4*>(from)[p];
    for (int64_t p = pieces * 16 + first; p < bytes; p += step) to[p] = from[p];
  }
}

int page_shift_of(int page_size) {
  return page_size > 0 && (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1;
}

// The checks the table operators share.
int check_table(const char* what, const void* refs, int64_t pages, const void* table, int64_t table_stride, int width,
                int rows) {
  if (!refs || !table) return fail(XT_EINVAL, "%s: null pointer", what);
  if (pages < 1 || pages > 0x7FFFFFFF - 1024 || width < 1 || rows < 0 || (rows > 1 && table_stride < width))
    return fail(XT_EINVAL, "%s: bad sizes: %lld pages, table of %d rows x %d, row stride %lld", what, (long long)pages,
                rows, width, (long long)table_stride);
  return XT_OK;
}

int column_chunks(int width) { return width > 4096 ? 4 : (width + 1023) / 1024; }

}  // namespace
}  // namespace xt

using namespace xt;

extern "C" size_t xt_pages_workspace_bytes(int64_t pages) { return pages < 0 ? 0 : (size_t)pages * 4; }

extern "C" int xt_pages_extend(int32_t* refs, int64_t pages, int32_t* table, int64_t table_stride, int width,
                               int32_t* lens, const int32_t* add, int rows, int page_size, uint8_t* granted,
                               void* workspace, size_t workspace_bytes, xt_stream_t stream) {
  const char* what = "xt_pages_extend";
  if (const int st = check_table(what, refs, pages, table, table_stride, width, rows)) return st;
  if (rows == 0) return ok();
  const int shift = page_shift_of(page_size);
  if (!lens || !add || !granted || shift < 0)
    return fail(XT_EINVAL, "%s: null pointer or page size %d not a power of 2", what, page_size);
  if (width > 0x1FFFFF) return fail(XT_EUNSUPPORTED, "%s: a table of %d columns", what, width);
  if (!workspace || workspace_bytes < xt_pages_workspace_bytes(pages))
    return fail(XT_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes,
                xt_pages_workspace_bytes(pages));
  extend_kernel<<<1, kScanThreads, 0, stream>>>(refs, pages, table, table_stride, width, lens, add, rows, shift,
                                                granted, (int32_t*)workspace, pages);
  return check_launch(what);
}

extern "C" int xt_pages_fork(int32_t* refs, int64_t pages, int32_t* table, int64_t table_stride, int width,
                             int32_t* lens, int rows, int page_size, const int32_t* parents, const int32_t* children,
                             int forks, int32_t* moves, int64_t moves_stride, void* workspace, size_t workspace_bytes,
                             xt_stream_t stream) {
  const char* what = "xt_pages_fork";
  if (const int st = check_table(what, refs, pages, table, table_stride, width, rows)) return st;
  if (forks == 0) return ok();
  const int shift = page_shift_of(page_size);
  if (forks < 0 || !lens || !parents || !children || !moves || moves_stride < forks || shift < 0)
    return fail(XT_EINVAL, "%s: null pointer, negative count or page size %d not a power of 2", what, page_size);
  if (forks > kScanThreads) return fail(XT_EUNSUPPORTED, "%s: %d forks in one call, at most %d", what, forks, kScanThreads);
  const bool small = (int64_t)forks * width <= XT_PAGES_FORK_CELLS;
  const size_t need = small ? 0 : (size_t)forks * 12;
  if (need && (!workspace || workspace_bytes < need))
    return fail(XT_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  int32_t* plan = small ? nullptr : (int32_t*)workspace;
  fork_kernel<<<1, kScanThreads, 0, stream>>>(refs, pages, table, table_stride, width, lens, rows, shift, parents,
                                              children, forks, moves, moves_stride, plan);
  if (const int st = check_launch(what)) return st;
  if (small) return ok();
  fork_rows_kernel<<<dim3(forks, column_chunks(width)), 256, 0, stream>>>(refs, pages, table, table_stride, width,
                                                                          children, plan);
  return check_launch(what);
}

extern "C" int xt_pages_free(int32_t* refs, int64_t pages, int32_t* table, int64_t table_stride, int width,
                             int32_t* lens, int rows, const int32_t* which, int n, xt_stream_t stream) {
  const char* what = "xt_pages_free";
  if (const int st = check_table(what, refs, pages, table, table_stride, width, rows)) return st;
  if (n == 0) return ok();
  if (n < 0 || !lens || !which) return fail(XT_EINVAL, "%s: null pointer or negative count", what);
  if (n > 0xFFFFFF) return fail(XT_EUNSUPPORTED, "%s: %d rows in one call", what, n);
  free_kernel<<<dim3(n, column_chunks(width)), 256, 0, stream>>>(refs, pages, table, table_stride, width, lens, rows,
                                                                 which);
  return check_launch(what);
}

extern "C" int xt_pages_compact(int32_t* refs, int64_t pages, int32_t* table, int64_t table_stride, int width, int rows,
                                int32_t* moves, int32_t* count, void* workspace, size_t workspace_bytes,
                                xt_stream_t stream) {
  const char* what = "xt_pages_compact";
  if (const int st = check_table(what, refs, pages, table, table_stride, width, rows)) return st;
  if ((!moves && pages > 1) || !count) return fail(XT_EINVAL, "%s: null pointer", what);
  if (!workspace || workspace_bytes < xt_pages_workspace_bytes(pages))
    return fail(XT_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes,
                xt_pages_workspace_bytes(pages));
  int32_t* map = (int32_t*)workspace;
  const int64_t half = pages / 2;
  compact_plan_kernel<<<1, kScanThreads, 0, stream>>>(refs, pages, moves, half, count, map);
  if (const int st = check_launch(what)) return st;
  if (rows == 0) return ok();
  const int64_t cells = (int64_t)rows * width;
  const int blocks = (int)(cells + 1023 < 1024 * 1024 ? (cells + 1023) / 1024 : 1024);
  compact_rows_kernel<<<blocks, 256, 0, stream>>>(pages, table, table_stride, width, rows, moves, count, map);
  return check_launch(what);
}

extern "C" int xt_pages_copy(const xt_page_buffer* buffers, int n_buffers, const int32_t* moves, int64_t moves_stride,
                             int n, const int32_t* count, xt_stream_t stream) {
  const char* what = "xt_pages_copy";
  if (n_buffers < 0 || n < 0 || (n_buffers > 0 && !buffers))
    return fail(XT_EINVAL, "%s: null pointer or negative count", what);
  if (n_buffers > XT_PAGES_COPY_MAX)
    return fail(XT_EUNSUPPORTED, "%s: %d buffers in one call, at most %d", what, n_buffers, XT_PAGES_COPY_MAX);
  if (n_buffers == 0 || n == 0) return ok();
  if (!moves || moves_stride < n) return fail(XT_EINVAL, "%s: null moves or rows of %lld for %d", what,
                                              (long long)moves_stride, n);
  CopyArgs a;
  int64_t most = 0;
  for (int i = 0; i < n_buffers; ++i) {
    const xt_page_buffer& b = buffers[i];
    if (!b.base || b.pages < 0 || b.bytes < 1 || (b.pages > 1 && b.stride < b.bytes))
      return fail(XT_EINVAL, "%s: buffer %d: null, negative or pages closer than their %lld bytes", what, i,
                  (long long)b.bytes);
    a.base[i] = (uint8_t*)b.base;
    a.stride[i] = b.pages > 1 ? b.stride : 0;
    a.bytes[i] = b.bytes;
    a.pages[i] = b.pages;
    most = b.bytes > most ? b.bytes : most;
  }
  const int64_t chunks = (most / 16 + 1023) / 1024;   // four 16-byte pieces a thread
  const dim3 grid(n < 4096 ? n : 4096, n_buffers, (unsigned)(chunks < 1 ? 1 : chunks > 64 ? 64 : chunks));
  copy_kernel<<<grid, 256, 0, stream>>>(a, moves, moves_stride, n, count);
  return check_launch(what);
}
