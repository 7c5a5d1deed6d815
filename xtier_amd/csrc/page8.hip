// The 8-bit paged cache: quantize-on-append with one power-of-two scale for each page and head, and attention over
// such pages (decode, verification, prompt chunks; whole contexts or a sliding window with sinks). Definitions and
// layouts in include/xtier_amd.h.
//
// Layout. Per page and KV head the K block is [page, dim] E4M3 bytes, and the V block is stored transposed, [dim, page].
// With keys as rows of the first product (S^T = K Q^T) a lane of an MFMA result holds one query and several keys, which
// is the operand shape that the second product (O^T = V^T P^T) wants for P^T, so P never leaves its registers; V^T rows
// are then what its first operand wants, 16 bytes a lane, with no transpose anywhere in the attention. The append,
// which touches each value once, pays for the transpose.
//
// Scales are powers of two. E4M3 has the same relative precision everywhere above 2^-6, so a finer scale would gain
// less than one binade of range, while a power of two makes every step but the rounding to E4M3 exact: a page whose
// scale grows keeps its normal values unchanged, and a K value with its scale is a BF16 value, so the first product takes
// the BF16 query and the keys exactly.
#include <type_traits>

#include "xt_common.h"
#include "xt_host.h"

namespace xt {
namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr int kTile = 64;               // keys of a step
constexpr int kMinExp = 63, kMaxExp = 246;   // scale exponents an append writes: 2^-64 .. 2^119, so that 448 * scale is finite

__device__ inline float exp_bits(int biased) {   // 2^(biased - 127), biased clamped to 1 .. 254
  const int e = biased < 1 ? 1 : biased > 254 ? 254 : biased;
  return __uint_as_float((uint32_t)e << 23);
}

// --- append -----------------------------------------------------------------------------------------------------------

struct AppendArgs {
  const uint16_t *k, *v;
  int64_t k_row, k_head, v_row, v_head;
  int64_t rows;
  uint8_t *kp, *vp, *ke, *ve;
  int64_t page_stride, head_stride, exp_page_stride, exp_head_stride;
  int64_t pages;
  int page_shift, heads, dim;
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t *seq_lens, *cu_rows;
  int batch;
};

// The biased exponent of the smallest power of two that keeps a BF16 magnitude (its bits) within 448 = 1.75 * 2^8.
__device__ inline int scale_exponent(uint32_t mag) {
  const int e = (int)(mag >> 7) - 8 + ((mag & 0x7Fu) > 0x60u ? 1 : 0);
  return e < kMinExp ? kMinExp : e > kMaxExp ? kMaxExp : e;
}

// Two values rounded to E4M3 (nearest even); more than 448 (infinities too) becomes 448, a NaN stays one.
__device__ inline uint32_t e4m3_pair(float a, float b) {
#if defined(__HIP_DEVICE_COMPILE__)
  a = __builtin_fabsf(a) > 448.0f ? __builtin_copysignf(448.0f, a) : a;
  b = __builtin_fabsf(b) > 448.0f ? __builtin_copysignf(448.0f, b) : b;
  uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xFFFFu;
  // (the conversion makes every NaN 0xFF: keep its sign, as the rest of the library does)
  if (a != a) w = (w & 0xFF00u) | 0x7Fu | (__float_as_uint(a) >> 24 & 0x80u);
  if (b != b) w = (w & 0xFFu) | 0x7F00u | (__float_as_uint(b) >> 16 & 0x8000u);
  return w;
#else
  return 0;
#endif
}

// One workgroup per (touched page, head, K or V). A thread keeps its first kKeep 16-byte pieces of the new rows in
// registers between the largest magnitude and the conversion; of larger pages the rest is read again, from L2. The rows'
// addresses do not depend on the page, so their loads go out before the table's answer is in. V is transposed through
// LDS. Bound by the chain of loads and the launch: measured 4.0 us for one row each of 32 requests (4 heads
// x 128), 8.5 for a chunk of 4096, 8.8 for 24 requests of up to 300 (2 x 256, pages of 16).
constexpr int kKeep = 4;

template <int T>
__global__ __launch_bounds__(T) void append_kernel(AppendArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t s_vt[];   // [dim][page + 4] bytes of the new V rows
  __shared__ uint32_t s_mag;
  const int head = (int)blockIdx.y, tid = (int)threadIdx.x;
  const bool is_v = blockIdx.z == 1;
  const int64_t unit = blockIdx.x;
  const int page = 1 << a.page_shift;
  int b;
  int64_t ordinal, row0, n;
  if (!a.cu_rows) {
    b = (int)unit;
    ordinal = 0;
    row0 = b;
    n = 1;
  } else {
    // request b's units start at floor(cu[b] / page) + 2 b: n rows touch at most floor(n / page) + 2 pages. The last
    // request that starts at or before this unit, 64 candidates at a time (every wave alike).
    int lo = 0;
    for (int n_left = a.batch; n_left > 1;) {
      const int step = (n_left + 63) / 64, off = (tid & 63) * step;
      const bool here = off < n_left && (a.cu_rows[lo + off] >> a.page_shift) + 2 * (int64_t)(lo + off) <= unit;
      const int found = (int)__popcll(__ballot(here));     // (unsigned; none: a unit before the first request's)
      const int k = found > 0 ? (found - 1) * step : 0;
      lo += k;
      n_left = min(step, n_left - k);
    }
    b = lo;
    row0 = a.cu_rows[b];
    n = a.cu_rows[b + 1] - row0;
    ordinal = unit - ((row0 >> a.page_shift) + 2 * (int64_t)b);
  }
  const int64_t len = a.seq_lens[b];
  const int64_t start = len - n;                              // the position of the request's first row
  const int64_t first = start > 0 ? start : 0;
  const int64_t col = (first >> a.page_shift) + ordinal;
  const int64_t lo = max(first, col << a.page_shift), hi = min(len, (col + 1) << a.page_shift);
  if (ordinal < 0 || n <= 0 || lo >= hi || col >= a.width) return;
  const int64_t src0 = row0 + (lo - start);                   // the first row of k / v for this page
  const int t0 = (int)(lo & (page - 1)), m = (int)(hi - lo);
  if (src0 < 0 || src0 + m > a.rows) return;
  const int vec_shift = __builtin_ctz((unsigned)a.dim) - 3, vecs = m << vec_shift;   // 16-byte pieces of the rows
  const int64_t row = is_v ? a.v_row : a.k_row;
  const uint16_t* src = (is_v ? a.v + head * a.v_head : a.k + head * a.k_head) + src0 * row;
  auto piece = [&](int i) {
    return *reinterpret_cast<const uint4*>(src + (i >> vec_shift) * row + (i & ((1 << vec_shift) - 1)) * 8);
  };
  uint4 keep[kKeep];
#pragma unroll
  for (int j = 0; j < kKeep; ++j) {
    keep[j] = uint4{0, 0, 0, 0};
    if (tid + T * j < vecs) keep[j] = piece(tid + T * j);
  }
  const int32_t id = a.table[(int64_t)b * a.table_stride + col];
  if (tid == 0) s_mag = 0;
  __syncthreads();
  if (id < 0 || id >= a.pages) return;

  auto largest = [](uint4 w, uint32_t mag) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = ws[i] & 0x7FFFu, y = (ws[i] >> 16) & 0x7FFFu;   // magnitudes; infinities and NaN do not count
      mag = max(mag, x < 0x7F80u ? x : 0u);
      mag = max(mag, y < 0x7F80u ? y : 0u);
    }
    return mag;
  };
  uint8_t* exp = (is_v ? a.ve : a.ke) + id * a.exp_page_stride + head * a.exp_head_stride;
  const int e0 = t0 > 0 ? *exp : 0;                           // a page that takes its first row starts anew
  uint32_t mag = 0;
#pragma unroll
  for (int j = 0; j < kKeep; ++j) mag = largest(keep[j], mag);
  for (int i = tid + T * kKeep; i < vecs; i += T) mag = largest(piece(i), mag);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) mag = max(mag, (uint32_t)__shfl_xor((int)mag, d));
  if (T > 64) {
    if ((tid & 63) == 0) atomicMax(&s_mag, mag);
    __syncthreads();
    mag = s_mag;
  }
  const int e1 = max(e0, scale_exponent(mag));
  const float mul = exp_bits(254 - e1);                       // 2^(127 - e)
  uint8_t* out = (is_v ? a.vp : a.kp) + id * a.page_stride + head * a.head_stride;

  // the page's earlier rows, where the scale grew
  if (t0 > 0 && e1 > e0) {
    const float f = exp_bits(127 - (e1 - e0));
    for (int i = tid; i < t0 * a.dim; i += T) {
      uint8_t* p = is_v ? out + (i / t0 << a.page_shift) + i % t0 : out + i;
      const float x = e4m3_decode(*p) * f;
      *p = (uint8_t)e4m3_pair(x, x);
    }
  }
  const int pitch = page + 4;
  auto put = [&](int i, uint4 w) {
    uint2 q;
    q.x = e4m3_pair(bf16_bits_to_f32(w.x & 0xFFFFu) * mul, bf16_bits_to_f32(w.x >> 16) * mul) |
          e4m3_pair(bf16_bits_to_f32(w.y & 0xFFFFu) * mul, bf16_bits_to_f32(w.y >> 16) * mul) << 16;
    q.y = e4m3_pair(bf16_bits_to_f32(w.z & 0xFFFFu) * mul, bf16_bits_to_f32(w.z >> 16) * mul) |
          e4m3_pair(bf16_bits_to_f32(w.w & 0xFFFFu) * mul, bf16_bits_to_f32(w.w >> 16) * mul) << 16;
    const int r = i >> vec_shift, d = (i & ((1 << vec_shift) - 1)) * 8;
    if (!is_v) {
      *reinterpret_cast<uint2*>(out + (t0 + r) * a.dim + d) = q;
    } else if (m == 1) {                                      // one byte of each dimension: straight to its place
#pragma unroll
      for (int j = 0; j < 8; ++j) out[((d + j) << a.page_shift) + t0] = (uint8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) s_vt[(d + j) * pitch + t0 + r] = (uint8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
    }
  };
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    if (tid + T * j < vecs) put(tid + T * j, keep[j]);
  for (int i = tid + T * kKeep; i < vecs; i += T) put(i, piece(i));
  if (is_v && m > 1) {
    __syncthreads();
    // whole words of a dimension's row, and bytes at its ends
    const int w0 = (t0 + 3) >> 2, w1 = (t0 + m) >> 2, words = w1 > w0 ? w1 - w0 : 0;
    if (words > 0) {
      for (int i = tid; i < a.dim * words; i += T) {
        const int d = i / words, t = (w0 + i % words) * 4;
        *reinterpret_cast<uint32_t*>(out + (d << a.page_shift) + t) = *reinterpret_cast<uint32_t*>(s_vt + d * pitch + t);
      }
    }
    const int head_end = words > 0 ? w0 * 4 : t0 + m, tail = words > 0 ? w1 * 4 : t0 + m;
    const int ends = (head_end - t0) + (t0 + m - tail);
    for (int i = tid; i < a.dim * ends; i += T) {
      const int d = i / ends, k = i % ends, t = k < head_end - t0 ? t0 + k : tail + k - (head_end - t0);
      out[(d << a.page_shift) + t] = s_vt[d * pitch + t];
    }
  }
  if (tid == 0) *exp = (uint8_t)e1;
}

// --- attention: the work and its division ------------------------------------------------------------------------------

// A piece of a planned call: its request and row tile, and which of its entry's pieces it is; with more than one, the
// slot of its partial within the head.
struct Planned {
  int b, tile, at, count, slot, pad[3];
};

struct AttnArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  const uint8_t *kp, *vp, *ke, *ve;
  uint32_t page_stride, exp_page_stride;
  int64_t head_stride, exp_head_stride;
  uint32_t pages;
  int page_shift, heads, group;
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t *seq_lens, *cu_q;
  int batch, rows;
  int window, sinks;
  float scale;          // softmax scale * log2(e)
  void* out;
  int64_t out_row, out_head;
  int out_bf16;
  float* lse;           // [rows, heads * group] or NULL
  int entries;          // (request, row tile) pairs, some empty
  int min_tiles;        // key tiles that a workgroup takes at least
  int slots;            // workgroups on the CUs at once
  int32_t* counters;    // one per partial, zero between calls
  float* part;
  int partials;         // what `part` has room for
  int* plan;            // of a call with many entries, else NULL: pieces of a head, those of cut entries among them
  Planned* planned;     // and its pieces
  int* plan_tiles;      // scratch, an entry each
};

// A row tile of a request: rows r = token * group + head of the group, `m_rows` of them, and its key tiles. Tile t of
// the entry holds the keys from 64 * (t < sink_tiles ? t : t + skip).
struct Entry {
  int b, n;             // request and its query tokens
  int row0;             // the request's first row of q
  int r0, r1;           // rows of the tile within the request
  int len, start;       // context length, the position of the first query token
  int end;              // keys that any row may see
  int sink_tiles, skip, tiles;
};

// The row tiles of the requests before one whose first row is `row`, some of them empty.
__device__ inline int tile_base(const AttnArgs& a, int row, int m_rows) { return row * a.group / m_rows; }

// The request and row tile of an entry.
__device__ inline int request_of(const AttnArgs& a, int e, int m_rows, int* tile) {
  if (!a.cu_q) {
    const int per = (a.group + m_rows - 1) / m_rows, b = per == 1 ? e : e / per;
    *tile = e - b * per;
    return b;
  }
  // request b's tiles start at floor(cu[b] * group / m_rows) + b, which leaves room for a ragged last one
  int lo = 0, hi = a.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tile_base(a, a.cu_q[mid], m_rows) + mid <= e) lo = mid;
    else hi = mid - 1;
  }
  *tile = e - (tile_base(a, a.cu_q[lo], m_rows) + lo);
  return lo;
}

__device__ inline Entry entry_of(const AttnArgs& a, int b, int tile, int m_rows) {
  Entry x;
  x.b = b;
  if (!a.cu_q) {
    x.row0 = b;
    x.n = 1;
  } else {
    x.row0 = a.cu_q[b];
    x.n = a.cu_q[b + 1] - x.row0;
    if (x.row0 < 0 || x.n < 0 || x.row0 + (int64_t)x.n > a.rows) x.n = 0;
  }
  x.len = max(a.seq_lens[x.b], 0);
  x.start = x.len - x.n;
  const int all = x.n * a.group;          // (the host keeps rows * group within 2^30)
  x.r0 = x.r1 = x.end = x.sink_tiles = x.skip = x.tiles = 0;
  if (tile < 0 || tile > all / m_rows || tile * m_rows >= all) return x;
  x.r0 = tile * m_rows;
  x.r1 = min(x.r0 + m_rows, all);
  // (one token's heads share its position)
  const int p_lo = x.start + (x.n == 1 ? 0 : x.r0 / a.group);
  const int p_hi = x.start + (x.n == 1 ? 0 : (x.r1 - 1) / a.group);
  const int64_t cap = (int64_t)a.width << a.page_shift;
  x.end = p_hi + 1 <= 0 ? 0 : p_hi + 1 < cap ? p_hi + 1 : (int)cap;
  const int tiles = (int)(((int64_t)x.end + kTile - 1) / kTile);
  if (a.window > 0) {
    const int64_t from = (int64_t)p_lo - a.window + 1;
    int lo = from > 0 ? (int)(from / kTile) : 0;
    lo = lo < tiles ? lo : tiles;
    x.sink_tiles = (int)(((int64_t)min(a.sinks, x.end) + kTile - 1) / kTile);
    x.skip = lo > x.sink_tiles ? lo - x.sink_tiles : 0;
  }
  x.tiles = tiles - x.skip > 0 ? tiles - x.skip : 1;   // rows that see nothing still take a step, which writes them
  return x;
}

__device__ inline Entry entry_at(const AttnArgs& a, int e, int m_rows) {
  int tile;
  const int b = request_of(a, e, m_rows, &tile);
  return entry_of(a, b, tile, m_rows);
}

// Both kernels divide their work, the key tiles of every (KV head, entry), on the device: a long request is shared by
// many workgroups, whatever the lengths, and a captured launch follows the lengths of each replay. Work is numbered head
// by head, entry by entry. Every workgroup divides the work for itself if there is at most one entry to a lane (decode) or
// thread (prefill); of more, a launch before makes the plan (plan_kernel): in every workgroup again, the division grew
// with the square of the entries (decode of 1024 requests of 256 keys, with row offsets: 459 us, now 77; of 8192: 40 ms,
// now 565 us; of 256: 53, now 27). A (head, entry) that several workgroups share is merged from their partials by the last of
// them to finish, in their order.
//
// Sums of x and y over the workgroup's threads before this one, and over all of them. `s` holds 2 * T / 64 values.
template <int T>
__device__ inline void block_sums(int x, int y, int* s, int* x_before, int* x_all, int* y_before, int* y_all) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int xi = wave_inclusive_sum(x), yi = wave_inclusive_sum(y);
  __syncthreads();
  if (lane == 63) {
    s[wave] = xi;
    s[T / 64 + wave] = yi;
  }
  __syncthreads();
  int xb = 0, yb = 0, xs = 0, ys = 0;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    if (w < wave) {
      xb += s[w];
      yb += s[T / 64 + w];
    }
    xs += s[w];
    ys += s[T / 64 + w];
  }
  *x_before = xb + xi - x;
  *y_before = yb + yi - y;
  *x_all = xs;
  *y_all = ys;
}

// A workgroup's work in the decode kernel: piece `at` of the `count` that one (head, entry) is cut into. The pieces are
// as small as leaves all of them on the CUs at once (or, with more (head, entry) pairs than half the slots, only those
// well above the mean are cut: a piece has at most total / (slots / 2) tiles). Cutting at pairs only keeps every
// workgroup at one entry: equal runs that cross from one to the next cost a second entry's loads and merges in a row,
// 8 us (1 request, 2 KV heads x 256, 4099 keys: 25 us so, 17 now).
struct Piece {
  int head, at, count;
  int slot;              // of the piece's partial, if count > 1; the slots of an entry's pieces are neighbours
};

// The smallest piece that pays: n pieces of an entry of t tiles take about t / n steps and n partials to merge, whose cost
// grows with the rows, least at pieces of rows / 32 * sqrt(t) tiles (measured, with fixed sizes of 4 / 8 / 16 tiles: 1
// request of 512 tiles, 16 rows, 21.7 / 17.6 / 17.9 us; 4 of 256 tiles, 32 rows, 38.4 / 38.3 / 28.5 us; 2 of 64 tiles, 32
// rows, 19.9 / 21.4 / 24.2 us). 16 partials are read in one go, so a few more than 16 pieces become 16.
__device__ inline int least_piece(const AttnArgs& a, int m_rows, int all, int n_live) {
  const int t = all / max(n_live, 1);
  const int size = max(a.min_tiles, (int)(m_rows / 32.0f * __builtin_sqrtf((float)t))), n = (t + size - 1) / size;
  return n > 16 && n < 24 ? (t + 15) / 16 : size;
}

// Which piece a workgroup of the grid takes, of `count`: each XCD (workgroups go round robin over 8) takes an eighth of
// the pieces, neighbours in the same keys together; the grid has room for more pieces than there are, so the eighths
// are of what there is. -1: none.
__device__ inline int piece_of_xcd(int id, int count) {
  const int of_xcd = (count + 7) / 8, w = (id & 7) * of_xcd + (id >> 3);
  return (id >> 3) < of_xcd && w < count ? w : -1;
}

// Where the pieces of a head under the least size are more than there is room for: how many a second size is meant to give,
// besides one for each entry.
__device__ inline int sure_pieces(int room, int n_live) { return max(max(room - n_live, room / 2), 1); }

__device__ inline Piece planned_piece(const AttnArgs& a, int id, int m_rows, Entry* en) {
  Piece x;
  x.count = 0;
  const int per_head = uniform_load(a.plan);
  const int w = piece_of_xcd(id, per_head * a.heads);
  if (w < 0) return x;
  x.head = w / per_head;
  const int* p = &a.planned[w - x.head * per_head].b;
  *en = entry_of(a, uniform_load(p), uniform_load(p + 1), m_rows);
  x.at = uniform_load(p + 2);
  x.count = uniform_load(p + 3);
  x.slot = x.head * uniform_load(a.plan + 1) + uniform_load(p + 4);
  return x;
}

// An entry to a lane, every wave by itself: no barriers (1 request of 4099 keys, 18.5 us with them, 17.3 without).
__device__ inline Piece piece_of(const AttnArgs& a, int m_rows, int id, Entry* en) {
  Piece x;
  x.count = 0;
  const int room = max(a.slots / a.heads, 1);       // pieces of a head
  const int lane = (int)threadIdx.x & 63;
  const Entry mine = entry_at(a, min(lane, a.entries - 1), m_rows);
  const int tiles = lane < a.entries ? mine.tiles : 0;
  const int all = __builtin_amdgcn_readlane(wave_inclusive_sum(tiles), 63);
  const int n_live = __popcll(__ballot(tiles > 0)), sure = sure_pieces(room, n_live);
  const int least = least_piece(a, m_rows, all, n_live);
  // per head: the smallest size that could fit, and if it does not, one that is sure to
  int size = max((all + room - 1) / room, least), n, upto, cut;
  for (int tries = 0;; ++tries) {
    n = (tiles + size - 1) / size;
    upto = wave_inclusive_sum(n);
    cut = wave_inclusive_sum(n > 1 ? n : 0);
    if (__builtin_amdgcn_readlane(upto, 63) <= room || tries == 1) break;
    size = max((all + sure - 1) / sure, least);
  }
  const int per_head = __builtin_amdgcn_readlane(upto, 63), cut_per_head = __builtin_amdgcn_readlane(cut, 63);
  const int w = piece_of_xcd(id, per_head * a.heads);
  if (w < 0) return x;
  x.head = w / per_head;
  const int want = w - x.head * per_head;
  const int entry = __builtin_ctzll(__ballot(want < upto));    // the first entry whose running count passes it
  x.count = __builtin_amdgcn_readlane(n, entry);
  x.at = want - (__builtin_amdgcn_readlane(upto, entry) - x.count);
  x.slot = x.head * cut_per_head + __builtin_amdgcn_readlane(cut, entry) - x.count + x.at;
  // (from its lane: loading it again would cost another round trip)
  auto of_entry = [&](int v) { return __builtin_amdgcn_readlane(v, entry); };
  en->b = of_entry(mine.b);
  en->n = of_entry(mine.n);
  en->row0 = of_entry(mine.row0);
  en->r0 = of_entry(mine.r0);
  en->r1 = of_entry(mine.r1);
  en->len = of_entry(mine.len);
  en->start = of_entry(mine.start);
  en->end = of_entry(mine.end);
  en->sink_tiles = of_entry(mine.sink_tiles);
  en->skip = of_entry(mine.skip);
  en->tiles = of_entry(mine.tiles);
  return x;
}

// The plan of a call with many entries, by one workgroup: a run of entries to a thread. `room`: pieces of a head at once.
// Decode (`few` rows) cuts as piece_of does. Prefill, whose workgroups take pieces in rounds, cuts only entries that are
// longer than an equal share of all of them. Either way an entry that is cut is longer than a size that goes at most
// `room` times into their sum, so that the pieces with partials are fewer than 2 * room.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(AttnArgs a, int m_rows, int room, bool few) {
  constexpr int T = kPlanThreads;
  __shared__ int s_sum[2 * (T / 64)];
  const int tid = (int)threadIdx.x;
  const int chunk = (a.entries + T - 1) / T;
  const int e0 = (int)min((int64_t)chunk * tid, (int64_t)a.entries), e1 = min(e0 + chunk, a.entries);
  int first_tile = 0;
  const int first = e0 < e1 ? request_of(a, e0, m_rows, &first_tile) : 0;
  // the entries of this thread in order: f(entry, request, row tile); with offsets, the requests are walked through
  auto each = [&](auto f) {
    int b = first, tile = first_tile;
    const int per = (a.group + m_rows - 1) / m_rows;
    for (int e = e0; e < e1; ++e) {
      f(e, b, tile);
      ++tile;
      if (!a.cu_q) {
        if (tile == per) {
          ++b;
          tile = 0;
        }
      } else {
        int base;
        while (b + 1 < a.batch && (base = tile_base(a, a.cu_q[b + 1], m_rows) + b + 1) <= e + 1) {
          ++b;
          tile = e + 1 - base;
        }
      }
    }
  };
  int sum = 0, live = 0, before, all, cut_before, n_live;
  each([&](int e, int b, int tile) {
    const int t = entry_of(a, b, tile, m_rows).tiles;
    a.plan_tiles[e] = t;
    sum += t;
    live += t > 0;
  });
  block_sums<T>(sum, live, s_sum, &before, &all, &cut_before, &n_live);
  const int sure = few ? sure_pieces(room, n_live) : room;
  const int least = few ? least_piece(a, m_rows, all, n_live) : a.min_tiles;
  int size = max((all + room - 1) / room, least), mine, cut, per_head, cut_per_head;
  for (int tries = 0;; ++tries) {
    mine = cut = 0;
    for (int e = e0; e < e1; ++e) {
      const int n = (a.plan_tiles[e] + size - 1) / size;
      mine += n;
      cut += n > 1 ? n : 0;
    }
    block_sums<T>(mine, cut, s_sum, &before, &per_head, &cut_before, &cut_per_head);
    if (!few || per_head <= room || tries == 1) break;
    size = max((all + sure - 1) / sure, least);
  }
  if (tid == 0) {
    a.plan[0] = per_head;
    a.plan[1] = cut_per_head;
  }
  int at = before, slot = cut_before;
  each([&](int e, int b, int tile) {
    const int n = (a.plan_tiles[e] + size - 1) / size;
    for (int i = 0; i < n; ++i) a.planned[at + i] = Planned{b, tile, i, n, slot + i, {0, 0, 0}};
    at += n;
    slot += n > 1 ? n : 0;
  });
}

// The workgroup of the launch, renumbered so that each XCD (workgroups go round robin over 8) takes a contiguous run of
// the work: neighbours in it read the same keys, out of that XCD's L2.
__device__ inline int xcd_order(int id, int groups) { return (id & 7) * (groups >> 3) + (id >> 3); }

// A workgroup's work in the prefill kernel, which has one workgroup to a slot: segments, each the tiles t0 .. t1 - 1 of
// one (head, entry). Its `sharers` workgroups leave partials in slots base + step * i (the first one's moved by `bump`).
//
// Either the work is dealt out in pieces, whole entries or (with fewer of them than slots) even cuts of them, or, where
// that would leave slots idle in the last round, every workgroup takes an equal run of tiles, across entries. An entry
// costs about kStart tiles to begin and end, and kShare more where its partials go through memory (measured: 8 and 24 us
// of 2.1 us a tile at 256 rows x 128, 6 and 9 us of 1 us at 128 x 64), by which the cheaper way is chosen. Runs alone: 2
// prompts of 1024 tokens, 32 / 4 heads x 128, 118 us, 5 prompts through a window of 1000, 106 us; with the choice
// 55 and 86 us (with the cheaper masks that came with it).
//
// (What is the same in every lane but comes out of LDS goes through readfirstlane, in both kernels: the loads of an entry
// are then scalar loads, and the loops over tiles and their branches scalar ones.)
constexpr int kStart = 4, kShare = 10;
struct Run {
  bool pieces;
  int per_head;                        // pieces of a head, or its tiles
  int size, cut_per_head;              // pieces: of at most `size` tiles, those of cut entries
  int turn;                            // pieces this workgroup has had
  int per, entry_pos;                  // runs: tiles of one, and the first tile of the entry within its head
  int64_t pos, end;
};
struct Segment {
  int head, entry, t0, t1;
  int sharers, at;                     // at: this workgroup among them
  int base, step, bump, counter;
  __device__ int slot(int i) const { return base + step * i + (i == 0 ? bump : 0); }
};

template <int T>
__device__ inline Run plan_run(const AttnArgs& a, int m_rows, int groups, int id, int* s_sum, int* s_find, int* s_mine,
                                Segment* sg) {
  Run x;
  const int tid = (int)threadIdx.x;
  x.turn = 0;
  x.pos = x.end = 0;
  sg->head = sg->entry = sg->t0 = sg->t1 = 0;
  if (a.plan) {
    x.pieces = true;
    x.per_head = uniform_load(a.plan);
    x.cut_per_head = uniform_load(a.plan + 1);
    return x;
  }
  const int tiles = tid < a.entries ? entry_at(a, tid, m_rows).tiles : 0;
  int before, all, cut_before, n_live;
  if (tid == 0) s_find[0] = 0;
  block_sums<T>(tiles, tiles > 0, s_sum, &before, &all, &cut_before, &n_live);
  atomicMax(&s_find[0], tiles);
  int most;
  __syncthreads();
  most = __builtin_amdgcn_readfirstlane(s_find[0]);
  all = __builtin_amdgcn_readfirstlane(all);
  n_live = __builtin_amdgcn_readfirstlane(n_live);
  const int units = n_live * a.heads;
  const int64_t total = (int64_t)all * a.heads;
  // steps until the last workgroup is done: runs, whole entries in rounds (the last of them with the longest entry), or
  // entries cut so that all pieces are on the CUs at once
  const int run = (int)((total + groups - 1) / groups);
  const int per_slot = (units + groups - 1) / groups;
  const float by_runs = (float)run + (1.0f + (float)units / groups) * kStart + 1.5f * kShare;
  const float mean = (float)total / max(units, 1);
  const float whole = per_slot * (mean + kStart) + 0.5f * ((float)most - mean);
  const int spare = units < groups ? (groups - units) / a.heads : 0;
  int size = most;
  float by_pieces = whole;
  if (spare > 0) {
    const int cut = max((all + spare - 1) / spare, a.min_tiles);
    if (cut < most && cut + kStart + kShare < whole) {
      size = cut;
      by_pieces = (float)(cut + kStart + kShare);
    }
  }
  x.pieces = by_pieces <= by_runs;
  x.per = max(run, a.min_tiles);
  x.per_head = all;
  if (x.pieces) {
    // s_mine: the pieces before each thread's entry, its own, and the cut ones before it (in LDS: in registers they would
    // stay through the whole kernel)
    int mine;
    const int room = max(groups / a.heads, 1), tight = max((all + room - 1) / room, a.min_tiles);
    const bool try_tight = size < most && tight < size;      // the smallest size that could fit, else the sure one
    for (int tries = try_tight ? 0 : 1;; ++tries) {
      x.size = max(tries == 0 ? tight : size, 1);
      mine = (tiles + x.size - 1) / x.size;
      block_sums<T>(mine, mine > 1 ? mine : 0, s_sum, &before, &x.per_head, &cut_before, &x.cut_per_head);
      if (tries == 1 || __builtin_amdgcn_readfirstlane(x.per_head) <= room) break;
    }
    x.size = __builtin_amdgcn_readfirstlane(x.size);
    s_mine[tid] = before;
    s_mine[T + tid] = mine;
    s_mine[2 * T + tid] = cut_before;
    x.per_head = __builtin_amdgcn_readfirstlane(x.per_head);
    x.cut_per_head = __builtin_amdgcn_readfirstlane(x.cut_per_head);
    return x;
  }
  const int w = xcd_order(id, groups);
  x.pos = (int64_t)x.per * w;
  x.end = min(x.pos + x.per, total);
  if (x.pos >= x.end) return x;
  sg->head = (int)(x.pos / all);
  const int want = (int)(x.pos - (int64_t)sg->head * all);   // within the head
  __syncthreads();
  if (want >= before && want < before + tiles) {
    s_find[0] = tid;
    s_find[1] = before;
  }
  __syncthreads();
  sg->entry = __builtin_amdgcn_readfirstlane(s_find[0]);
  x.entry_pos = __builtin_amdgcn_readfirstlane(s_find[1]);
  return x;
}

// The workgroup's next segment and its entry; false when there is none.
template <int T>
__device__ inline bool next_segment(const AttnArgs& a, int m_rows, int groups, int id, int* s_find, const int* s_mine, Run& x,
                                    Segment* sg, Entry* en) {
  if (x.pieces) {
    const int w = piece_of_xcd(id + x.turn * groups, x.per_head * a.heads);
    ++x.turn;
    if (w < 0) return false;
    sg->head = w / x.per_head;
    int slot;                            // of the entry's first piece, among those of its head
    if (a.plan) {
      const int* p = &a.planned[w - sg->head * x.per_head].b;
      *en = entry_of(a, uniform_load(p), uniform_load(p + 1), m_rows);
      sg->at = uniform_load(p + 2);
      sg->sharers = uniform_load(p + 3);
      slot = uniform_load(p + 4) - sg->at;
    } else {
      const int tid = (int)threadIdx.x, want = w - sg->head * x.per_head - s_mine[tid];
      __syncthreads();
      if (want >= 0 && want < s_mine[T + tid]) {
        s_find[0] = tid;
        s_find[1] = want;
        s_find[2] = s_mine[T + tid];
        s_find[3] = s_mine[2 * T + tid];
      }
      __syncthreads();
      *en = entry_at(a, __builtin_amdgcn_readfirstlane(s_find[0]), m_rows);
      sg->at = __builtin_amdgcn_readfirstlane(s_find[1]);
      sg->sharers = __builtin_amdgcn_readfirstlane(s_find[2]);
      slot = __builtin_amdgcn_readfirstlane(s_find[3]);
    }
    const int share = en->tiles / sg->sharers, longer = en->tiles % sg->sharers;   // the first `longer` have one more
    sg->t0 = sg->at * share + min(sg->at, longer);
    sg->t1 = sg->t0 + share + (sg->at < longer ? 1 : 0);
    sg->base = sg->counter = sg->head * x.cut_per_head + slot;
    sg->step = 1;
    sg->bump = 0;
    return true;
  }
  if (x.pos >= x.end) return false;
  if (sg->t1 > 0) {                    // on to the next entry that has rows
    x.entry_pos += en->tiles;
    do {
      if (++sg->entry == a.entries) {
        sg->entry = 0;
        x.entry_pos = 0;
        ++sg->head;
      }
    } while (entry_at(a, sg->entry, m_rows).tiles == 0);
  }
  *en = entry_at(a, sg->entry, m_rows);
  const int64_t first = (int64_t)sg->head * x.per_head + x.entry_pos;       // the entry's first tile
  sg->t0 = (int)(x.pos - first);
  sg->t1 = (int)min((int64_t)en->tiles, x.end - first);
  x.pos = first + sg->t1;
  // a workgroup has two slots: for an entry that began before its run, and for one that ends after it
  const int w0 = (int)(first / x.per);
  sg->sharers = (int)((first + en->tiles - 1) / x.per) - w0 + 1;
  sg->at = xcd_order(id, groups) - w0;
  sg->base = 2 * w0;
  sg->step = 2;
  sg->bump = (int64_t)x.per * w0 < first ? 1 : 0;
  sg->counter = w0;
  return true;
}

__device__ inline void store_out(const AttnArgs& a, int64_t row, int head, int d, float4_t v) {
  const int64_t at = row * a.out_row + head * a.out_head + d;
  uint2 w;
  if (a.out_bf16) {
    w.x = pack2_16<true>(v[0], v[1]);
    w.y = pack2_16<true>(v[2], v[3]);
  } else {
    w.x = pack2_16<false>(v[0], v[1]);
    w.y = pack2_16<false>(v[2], v[3]);
  }
  *reinterpret_cast<uint2*>((uint16_t*)a.out + at) = w;
}

// The keys that a row at position p sees, as bounds on j - base: j < hi and (j >= lo or j < sink).
struct Sight {
  int hi, lo, sink;
  // for j - base = from .. from + n - 1, n <= 16, as bits
  __device__ uint32_t bits(int from, int n) const {
    auto below = [&](int x) { return (1u << min(max(x - from, 0), n)) - 1u; };
    return below(hi) & (~below(lo) | below(sink));
  }
};
// x where bit i of mask is set, -inf elsewhere.
__device__ inline float unless_hidden(float x, uint32_t mask, int i) {
  const uint32_t keep = (uint32_t)((int32_t)(mask << (31 - i)) >> 31);
  return __uint_as_float((__float_as_uint(x) & keep) | (0xFF800000u & ~keep));
}
__device__ inline Sight sight_of(const AttnArgs& a, int p_hi, int p_lo, int end, int base) {
  Sight x;
  x.hi = min(p_hi + 1, end) - base;
  x.lo = a.window > 0 ? p_lo - a.window + 1 - base : -base;
  x.sink = (a.window > 0 ? a.sinks : 0) - base;
  return x;
}

#if defined(__HIP_DEVICE_COMPILE__)

// Eight E4M3 bytes times a power of two, as BF16 (exact: E4M3 has fewer bits, and the exponents of both fit).
__device__ inline bf16x8_t e4m3x8_to_bf16(uint32_t lo, uint32_t hi, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ inline half8_t e4m3x8_to_f16(uint32_t lo, uint32_t hi, float scale) {
  const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false);
  const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true);
  const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false);
  const half2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Bits 0..3 of n as byte masks.
__device__ inline uint32_t byte_mask(uint32_t n) { return ((n & 15u) * 0x00204081u & 0x01010101u) * 0xFFu; }

// The top bit of each byte that holds an E4M3 NaN (0x7F or 0xFF).
__device__ inline uint32_t nan_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// Takes the NaN values of the keys `some` (bit i: byte i) out of 16 V bytes; returns which keys held one.
__device__ inline uint32_t take_nan(uint4& w, uint32_t some) {
  uint32_t* const ws[4] = {&w.x, &w.y, &w.z, &w.w};
  uint32_t found = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t nb = (nan_bytes(*ws[i]) & byte_mask(some >> (4 * i))) >> 7;   // 1 in each such byte
    *ws[i] &= ~(nb * 0xFFu);
    found |= (nb * 0x01020408u >> 24 & 15u) << (4 * i);                          // the four bits side by side
  }
  return found;
}

#endif

#if defined(__HIP_DEVICE_COMPILE__)

// The natural logarithm of a sum 2^m l, -inf for no keys.
__device__ inline float lse_of(float m, float l) {
  return l != 0.0f ? (m + __builtin_log2f(l)) * kLn2 : -__builtin_inff();
}

// A partial's maximum and sum, read as load_partial reads.
__device__ inline float2_t load_max_sum(__amdgpu_buffer_rsrc_t r, int byte_off) {
  typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
  const u32x2_t w = __builtin_amdgcn_raw_buffer_load_b64(r, byte_off, 0, 17 /* sc0 sc1 */);
  const uint32_t m = w[0], l = w[1];
  return float2_t{__uint_as_float(m), __uint_as_float(l)};
}

// The last workgroup of a (head, entry) merges its partials, slots of [rows][D O values, max, sum, padding]: normalized
// outputs, their maximum (of scaled scores in base 2) and their sum relative to it. slot_of(i): the i-th one's slot.
// Reads miss every cache, and what the merge takes is their round trips, so a thread has UB pieces of a row, of CB
// workgroups, in flight at once, with one maximum and sum of each. (A maximum and sum for each piece left room for half as
// much: 1 request, 2 KV heads x 256, 4099 keys, 16.7 us and 15.0 now; 2 requests of 80 rows at 63K 219 and 136. Sharing
// them through LDS, loaded 16 workgroups side by side, was slower than either: 520.)
template <int D, int M, int T, int UB, int CB, typename SlotOf>
__device__ inline void merge_partials(const AttnArgs& a, const Entry& en, int head, SlotOf slot_of, int sharers,
                                      __amdgpu_buffer_rsrc_t pr) {
  constexpr int kPer = D / 4 / UB, kPitch = D + 4, kSlot = M * kPitch;    // threads of a row
  const int units = (en.r1 - en.r0) * kPer;
  for (int i = (int)threadIdx.x; i < units; i += T) {
    const int row = i / kPer, d = i % kPer * 4;
    float mx = -__builtin_inff(), l = 0.0f;
    float4_t o[UB];
#pragma unroll
    for (int k = 0; k < UB; ++k) o[k] = float4_t{0.f, 0.f, 0.f, 0.f};
    for (int w0 = 0; w0 < sharers; w0 += CB) {
      float2_t ml[CB];
      float4_t x[UB][CB];
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        // (past the last workgroup: an offset past the buffer, which reads zeros)
        const bool real = w0 + c < sharers;
        const int at = real ? (slot_of(w0 + c) * kSlot + row * kPitch) * 4 : -16 - 4 * D;
        ml[c] = load_max_sum(pr, at + 4 * D);
#pragma unroll
        for (int k = 0; k < UB; ++k) x[k][c] = load_partial(pr, at + 4 * (d + 4 * kPer * k));
      }
      float m = mx;
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        if (w0 + c >= sharers) ml[c][0] = -__builtin_inff();
        m = fmaxf(m, ml[c][0]);
      }
      const float mu = m == -__builtin_inff() ? 0.0f : m;
      // shares of the sum, so that o stays a convex combination
      float wt[CB];
      const float old = l * __builtin_amdgcn_exp2f(mx - mu);
      float sum = old;
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        wt[c] = ml[c][1] * __builtin_amdgcn_exp2f(ml[c][0] - mu);
        sum += wt[c];
      }
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
      for (int k = 0; k < UB; ++k) {
        o[k] *= old * inv;
#pragma unroll
        for (int c = 0; c < CB; ++c) o[k] += wt[c] * inv * x[k][c];
      }
      l = sum;
      mx = m;
    }
    const int r = en.r0 + row, tok = r / a.group, qh = head * a.group + r % a.group;
#pragma unroll
    for (int k = 0; k < UB; ++k) store_out(a, en.row0 + tok, qh, d + 4 * kPer * k, o[k]);
    if (a.lse && d == 0) a.lse[(int64_t)(en.row0 + tok) * a.heads * a.group + qh] = lse_of(mx, l);
  }
}

#endif

// --- attention: few rows per request ------------------------------------------------------------------------------------

// 16 * NQ query rows a workgroup; its 4 waves take the run's key tiles in turn, straight from memory into registers, and
// merge at the end of each entry. Per tile of 64 keys a wave does S^T = K Q^T (A rows are keys, permuted so that lane
// group g holds scores of the keys 16 g .. 16 g + 15 in the order of a V^T row), the softmax of one query column per
// lane, and O^T += V^T P^T.
//
// P and V enter the second product as FP16: P is at most 1, and V as E4M3 times 2^(its page's exponent - the largest
// exponent seen) is exact within 15 binades below the largest. BF16 would round P eight times as coarsely.
//
// Workgroups on a CU at once, one wave of each to a SIMD: what the registers of O, the queries and a tile leave room for.
constexpr int decode_per_cu(int dim) { return dim == 256 ? 1 : 2; }

template <int D, int NQ>
struct DecodeGeo {
  static constexpr int kX = D / 64;                     // 16-byte pieces of a K row per lane
  static constexpr int kDT = D / 16;                    // 16-dim tiles of O
  static constexpr int kRows = 16 * NQ;
  static constexpr int kPitch = D + 4;                  // floats of a merged row in LDS: D, max, sum, padding
  static constexpr int kMerge = 4 * kRows * kPitch * 4;
  // With more than 16 rows the query operands lie in LDS, one 16-byte piece a lane for each MFMA: all waves have the same
  // rows, and in registers they would cost a wave of each SIMD (32 rows at 128) or spills (64).
  static constexpr int kQueries = NQ > 1 ? NQ * (D / 32) * 1024 : 0;
  static constexpr int kLds = kMerge + kQueries;
  static constexpr int kPoison = D > 128 ? 2 : 1;       // words of D / 4 bits
};

// A lane's share of a 64-key tile: the pages of its K and V blocks, then their data. What a load returns is looked at
// where it is needed and not before: a select on it would wait for every load in flight.
struct KvPages {
  int k, v;
};
template <int D>
struct KvStep {
  uint4 k[D / 64][4];       // [16-byte piece][16 keys]
  uint4 v[D / 16];
  int ke, ve;               // scale exponents
  bool kok, vok;            // whether the blocks hold anything
};

template <bool ONCE>
__device__ inline uint4 load16(const uint8_t* p) {
  if constexpr (ONCE) {
    const xt_u32x4_t w = __builtin_nontemporal_load(reinterpret_cast<const xt_u32x4_t*>(p));
    return uint4{w[0], w[1], w[2], w[3]};
  } else {
    return *reinterpret_cast<const uint4*>(p);
  }
}

template <int D, int NQ>
__global__ __launch_bounds__(256, decode_per_cu(D)) void decode_kernel(AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using G = DecodeGeo<D, NQ>;
  // Keys that one workgroup alone reads (up to 16 rows of a request) are loaded past the caches: 32 requests at 32K context
  // 178 us instead of 197 (6.0 TB/s), two of half a million keys 105 instead of 115. Not where a second row tile reads
  // them again (2 x 32 rows: 97 us instead of 75), and not in rows of 64 bytes (49 us instead of 46).
  constexpr bool kOnce = NQ == 1 && D >= 128;
  constexpr int M = G::kRows;
  extern __shared__ __attribute__((aligned(16))) float s_merge[];
  __shared__ int s_last;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  Entry en;
  const Piece pc = a.plan ? planned_piece(a, (int)blockIdx.x, M, &en) : piece_of(a, M, (int)blockIdx.x, &en);
  if (pc.count == 0) return;
  const int page_mask = (1 << a.page_shift) - 1;
  const int kk0 = 16 * (c >> 2) + (c & 3);   // A row c of 16-key tile t is key kk0 + 4 t of the 64
  const int head = pc.head;
  const int share = en.tiles / pc.count, longer = en.tiles % pc.count;    // the first `longer` pieces have a tile more
  const int t0 = pc.at * share + min(pc.at, longer), t1 = t0 + share + (pc.at < longer ? 1 : 0);
  {
    // query operands and positions of this lane's columns (those past the last row repeat it with a zero query, so that
    // they see what the others see)
    bf16x8_t qb[NQ == 1 ? 2 * G::kX : 1];
    uint4* const s_q = reinterpret_cast<uint4*>(s_merge + G::kMerge / 4);
    int pos[NQ];
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      const int r = en.r0 + 16 * nq + c, rr = min(r, en.r1 - 1), tok = rr / a.group;
      pos[nq] = en.start + tok;
      if (NQ > 1 && nq % 4 != wave % NQ) continue;     // (each block of 16 rows by one of the waves, or by several alike)
      const uint16_t* src = a.q + (int64_t)(en.row0 + tok) * a.q_row +
                            (head * a.group + (rr - tok * a.group)) * a.q_head + 16 * g;
#pragma unroll
      for (int x = 0; x < G::kX; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint4 w = {0, 0, 0, 0};
          if (r < en.r1) w = *reinterpret_cast<const uint4*>(src + 64 * x + 8 * y);
          if constexpr (NQ == 1) qb[2 * x + y] = __builtin_bit_cast(bf16x8_t, w);
          else s_q[(nq * 2 * G::kX + 2 * x + y) * 64 + lane] = w;
        }
    }
    if (NQ > 1) __syncthreads();
    const int p_lo = en.start + en.r0 / a.group, p_hi = en.start + (en.r1 - 1) / a.group;

    float4_t acc[NQ][G::kDT];
    float m_run[NQ], l_run[NQ];
    uint32_t poison[NQ][G::kPoison] = {};     // outputs that a NaN reached which not every row sees: bit 4 dt + i
    int e_ref = 0;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      m_run[nq] = -__builtin_inff();
      l_run[nq] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < G::kDT; ++dt) acc[nq][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    const int32_t* row_table = a.table + (int64_t)en.b * a.table_stride;
    const uint8_t *k_base = a.kp + head * a.head_stride, *v_base = a.vp + head * a.head_stride;
    const uint8_t *k_exps = a.ke + head * a.exp_head_stride, *v_exps = a.ve + head * a.exp_head_stride;
    auto key_of = [&](int t) { return kTile * (t < en.sink_tiles ? t : t + en.skip); };
    const int last = max(en.end - 1, 0);       // blocks past it look its page up and are masked
    auto pages_at = [&](int t) {
      const int base = key_of(t), kblk = base + 16 * (c >> 2), vblk = base + 16 * g;
      return KvPages{row_table[min(kblk, last) >> a.page_shift], row_table[min(vblk, last) >> a.page_shift]};
    };
    // a block that holds nothing reads page 0 and is masked
    auto load_k = [&](int t, KvPages p, KvStep<D>& st) {
      st.kok = ((uint32_t)p.k < a.pages) & (key_of(t) + 16 * (c >> 2) < en.end);
      const uint32_t page = st.kok ? p.k : 0;
      st.ke = k_exps[(uint64_t)page * a.exp_page_stride];
      const uint8_t* kp = k_base + (uint64_t)page * a.page_stride + (((key_of(t) + kk0) & page_mask) * D + 16 * g);
#pragma unroll
      for (int x = 0; x < G::kX; ++x)
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4)
          st.k[x][t4] = load16<kOnce>(kp + 64 * x + 4 * t4 * D);
    };
    auto load_v = [&](int t, KvPages p, KvStep<D>& st) {
      st.vok = ((uint32_t)p.v < a.pages) & (key_of(t) + 16 * g < en.end);
      const uint32_t page = st.vok ? p.v : 0;
      st.ve = v_exps[(uint64_t)page * a.exp_page_stride];
      const uint8_t* vp = v_base + (uint64_t)page * a.page_stride + ((c << a.page_shift) +
                                                                     ((key_of(t) + 16 * g) & page_mask));
#pragma unroll
      for (int dt = 0; dt < G::kDT; ++dt)
        st.v[dt] = load16<kOnce>(vp + ((16 * dt) << a.page_shift));
    };
    KvStep<D> st;
    KvPages cur = {-1, -1}, next = {-1, -1};
    const int first = t0 + wave;
    if (first < t1) {
      cur = pages_at(first);
      if (first + 4 < t1) next = pages_at(first + 4);
      load_k(first, cur, st);
      load_v(first, cur, st);
    }
    // Each of the tile's registers is refilled as soon as its product has read it: the next K is on its way during
    // softmax and PV, the next V during the next scores, and the pages of the tile after that.
    auto step = [&](int t, auto more_tiles) {
      constexpr bool more = decltype(more_tiles)::value;
      const int base = key_of(t);
      // scores
      float4_t s[NQ][4];
      const float ks = exp_bits(st.ke);
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) s[nq][t4] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < 2 * G::kX; ++x) {
        bf16x8_t q[NQ];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          if constexpr (NQ == 1) q[nq] = qb[x];
          else q[nq] = __builtin_bit_cast(bf16x8_t, s_q[(nq * 2 * G::kX + x) * 64 + lane]);
        }
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4) {
          const uint4 w = st.k[x / 2][t4];
          const bf16x8_t k = x % 2 == 0 ? e4m3x8_to_bf16(w.x, w.y, ks) : e4m3x8_to_bf16(w.z, w.w, ks);
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
            s[nq][t4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[nq], s[nq][t4], 0, 0, 0);
        }
        if (NQ > 1) __builtin_amdgcn_sched_barrier(0);
      }
      // (fences to the scheduler: phases that it mixes need more registers than there are)
      __builtin_amdgcn_sched_barrier(0);
      const bool pages_ok = st.kok && st.vok;
      if constexpr (more) load_k(t + 4, next, st);
      // a tile that every row sees whole needs no masks
      const bool whole = base + kTile - 1 <= p_lo && base + kTile <= en.end &&
                         (a.window <= 0 || base > p_hi - a.window || base + kTile <= a.sinks) &&
                         __ballot(!pages_ok) == 0;
      uint32_t vis[NQ];
      int ev = st.ve;
      // blocks of the V page that is gone hold keys that the K side masks too: lane group g's own block
      const int j0 = base + 16 * g;
      if (!whole) {
        uint32_t any = 0, all = 0xFFFFu;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          const Sight sight = sight_of(a, pos[nq], pos[nq], en.end, j0);
          const uint32_t mask = st.vok ? sight.bits(0, 16) : 0u;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[nq][i >> 2][i & 3] = unless_hidden(s[nq][i >> 2][i & 3], mask, i);
          vis[nq] = mask;
          any |= mask;
          all &= mask;
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
          any |= (uint32_t)__shfl_xor((int)any, d);
          all &= (uint32_t)__shfl_xor((int)all, d);
        }
        // values of keys that no row sees may be anything, NaN included: zero them
        if (any == 0) ev = -1;
        uint32_t nan = 0;
#pragma unroll
        for (int dt = 0; dt < G::kDT; ++dt) {
          uint4& w = st.v[dt];
          w.x &= byte_mask(any);
          w.y &= byte_mask(any >> 4);
          w.z &= byte_mask(any >> 8);
          w.w &= byte_mask(any >> 12);
          nan |= nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w);
        }
        const uint32_t some = any & ~all;
        if (__ballot((nan != 0) & (some != 0))) {
          // a NaN that some rows see and others do not: it leaves the product, and the outputs that it reaches become
          // NaN at the end. Which keys of a dimension hold one, and which keys a row sees, meet in LDS.
          uint16_t* map = reinterpret_cast<uint16_t*>(s_merge + wave * M * G::kPitch);   // [dim][4 blocks of 16 keys]
          uint16_t* seen = map + D * 4;                                                  // [row][4 blocks]
#pragma unroll
          for (int dt = 0; dt < G::kDT; ++dt) map[(16 * dt + c) * 4 + g] = (uint16_t)take_nan(st.v[dt], some);
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) seen[(16 * nq + c) * 4 + g] = (uint16_t)vis[nq];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) {
            const uint2 row = *reinterpret_cast<const uint2*>(seen + (16 * nq + c) * 4);
#pragma unroll 1
            for (int k = 0; k < D / 4; ++k) {          // acc[nq][k / 4][k % 4]: dimension 16 (k / 4) + 4 g + k % 4
              const uint2 dim = *reinterpret_cast<const uint2*>(map + (16 * (k >> 2) + 4 * g + (k & 3)) * 4);
              if ((dim.x & row.x) | (dim.y & row.y)) {
                if (k < 32) poison[nq][0] |= 1u << k;
                else poison[nq][G::kPoison - 1] |= 1u << (k - 32);
              }
            }
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        }
      }
      // the exponent that O is held at: the largest of any block used so far
      const int e_new = max(e_ref, (int)max4_lanes16((float)max(ev, 0)));
      const float e_drop = exp_bits(127 + max(e_ref - e_new, -126));
      e_ref = e_new;
      const float vs = exp_bits(127 + max(ev - e_ref, -126));
      half8_t pb[NQ][2];
      float f[NQ];
      bool rescale = false;
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        float mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[nq][i >> 2][i & 3]);
        const float m_new = fmaxf(m_run[nq], max4_lanes16(mx * a.scale));
        const float mu = m_new == -__builtin_inff() ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_run[nq] - mu);
        m_run[nq] = m_new;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nq][i >> 2][i & 3], a.scale, -mu));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nq][i >> 2][(i & 3) + 1], a.scale, -mu));
          sum += p0 + p1;
          const half2_t pair = __builtin_convertvector(float2_t{p0, p1}, half2_t);
          pb[nq][i >> 3][i & 7] = pair[0];
          pb[nq][i >> 3][(i & 7) + 1] = pair[1];
        }
        l_run[nq] = l_run[nq] * alpha + sum;
        f[nq] = alpha * e_drop;
        rescale |= f[nq] != 1.0f;
        if (NQ > 1) __builtin_amdgcn_sched_barrier(0);
      }
      if (__ballot(rescale)) {
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int dt = 0; dt < G::kDT; ++dt) acc[nq][dt] *= f[nq];
      }
#pragma unroll
      for (int dt = 0; dt < G::kDT; ++dt) {
        const uint4 w = st.v[dt];
        const half8_t v0 = e4m3x8_to_f16(w.x, w.y, vs), v1 = e4m3x8_to_f16(w.z, w.w, vs);
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          acc[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pb[nq][0], acc[nq][dt], 0, 0, 0);
          acc[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pb[nq][1], acc[nq][dt], 0, 0, 0);
        }
        if (NQ > 1 && dt % 2 == 1) __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (more) {
        load_v(t + 4, next, st);
        next = pages_at(min(t + 8, t1 - 1));
      }
    };
    // (the last tile's step apart: a refill on a condition would keep two copies of the registers)
    int t_now = first;
    for (; t_now + 4 < t1; t_now += 4) step(t_now, std::true_type());
    if (t_now < t1) step(t_now, std::false_type());

    // the waves' states, normalized and at their true scale, through LDS: rows of [O, max, sum]
    __syncthreads();
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      const float l = sum4_lanes16(l_run[nq]);
      float* mine = s_merge + (wave * M + 16 * nq + c) * G::kPitch;
      const float f = l != 0.0f ? exp_bits(e_ref) / l : 0.0f;   // (a NaN sum gives NaN)
#pragma unroll
      for (int dt = 0; dt < G::kDT; ++dt) {
        float4_t o = acc[nq][dt] * f;
        const uint32_t bad = poison[nq][dt / 8] >> (4 * (dt & 7));
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = bad >> i & 1u ? __builtin_nanf("") : o[i];
        *reinterpret_cast<float4_t*>(mine + 16 * dt + 4 * g) = o;
      }
      if (g == 0) {
        mine[D] = m_run[nq];
        mine[D + 1] = l;
      }
    }
    __syncthreads();
    const bool alone = pc.count == 1;
    const int rows_here = en.r1 - en.r0;
    constexpr int kPieces = D / 4;
    constexpr int kSlot = M * G::kPitch;                 // floats of a partial
    const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
        a.part, (short)0, (int)min((int64_t)a.partials * kSlot * 4, (int64_t)0x7FFFFFFF), 0x00020000);
    // O = sum_i (w_i / sum w) O_i with w_i = 2^(m_i - max m) l_i, over the waves
    for (int i = (int)threadIdx.x; i < rows_here * kPieces; i += 256) {
      const int r = i / kPieces, d = i % kPieces * 4;
      float mx = -__builtin_inff(), l = 0.0f, wt[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) mx = fmaxf(mx, s_merge[(w * M + r) * G::kPitch + D]);
      const float mu = mx == -__builtin_inff() ? 0.0f : mx;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float* src = s_merge + (w * M + r) * G::kPitch;
        wt[w] = __builtin_amdgcn_exp2f(src[D] - mu) * src[D + 1];
        l += wt[w];
      }
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      float4_t o = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) o += wt[w] * inv * *reinterpret_cast<float4_t*>(s_merge + (w * M + r) * G::kPitch + d);
      if (alone) {
        const int tok = (en.r0 + r) / a.group, qh = head * a.group + (en.r0 + r) % a.group;
        store_out(a, en.row0 + tok, qh, d, o);
        if (a.lse && d == 0)
          a.lse[(int64_t)(en.row0 + tok) * a.heads * a.group + qh] = lse_of(mx, l);
      } else {
        const int at = (pc.slot * kSlot + r * G::kPitch) * 4;
        store_partial(pr, at + 4 * d, o);
        if (d == 0) store_partial(pr, at + 4 * D, float4_t{mx, l, 0.0f, 0.0f});
      }
    }
    if (!alone) {
      const int first = pc.slot - pc.at;
      int32_t* counter = a.counters + first;
      if (arrive_last(counter, pc.count, &s_last)) {
        merge_partials<D, M, 256, D / 64, 16>(a, en, head, [&](int i) { return first + i; }, pc.count, pr);
        reset_counter(counter);
      }
    }
  }
#endif
}

// --- attention: many rows per request -----------------------------------------------------------------------------------

// 32 W query rows a workgroup, 32 for each of its W waves, on 32x32 MFMAs. The workgroup dequantizes each 64-key tile
// once, K to BF16 and V to FP16, into one of two LDS stages while it computes on the other: a wave's 32 rows alone would
// pay the conversion W times over. K rows lie in LDS in the order of the A rows of S^T (key_row).
template <int D, int W>
struct PrefillGeo {
  static constexpr int kM = 32 * W, kThreads = 64 * W;
  // Rows of a stage are padded by 16 bytes: LDS reads 16 lanes' 16-byte units at a time from 64 banks, and 16 rows in a
  // row, an odd number of units apart, put the same unit at 16 different places. (An XOR of the unit with the row
  // saves the padding, but costs an address register or instruction for every unit of a row.)
  static constexpr int kRowK = D * 2 + 16, kRowV = kTile * 2 + 16;
  static constexpr int kStageK = kTile * kRowK, kStageV = D * kRowV;
  static constexpr int kLds = 2 * (kStageK + kStageV);
  static constexpr int kLoads = kTile * D / 16 / kThreads;    // 16-byte pieces of K, and of V, that a thread stages
  static constexpr int kDT = D / 32;
};

// The LDS row of a key: A row 8 a + 4 h + i of a 32-key block is key 16 (a / 2) + 8 h + 4 (a % 2) + i, which leaves
// lane half h of S^T with eight neighbouring keys of every 16: a step's operand of P^T, in the order of a V^T row.
__device__ inline int key_row(int key) {
  return (key & 32) | (key & 16) | ((key >> 2 & 1) << 3) | ((key >> 3 & 1) << 2) | (key & 3);
}

typedef float float16_t __attribute__((ext_vector_type(16)));

// Computed at this place: the compiler otherwise moves what is first used in a later block there, away from the MFMAs that
// it is meant to run beside. (x must be the result of an ordinary vector instruction, as in max2_raw.)
template <typename T>
__device__ inline void keep_here(T& x) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(x));
#endif
}

// The step of tile t: S(t + 1) = K(t + 1) Q^T beside the softmax of S(t), then O += V(t) P(t) beside the conversion of
// V(t + 1) and K(t + 2), which lie in registers, and the loads of the pair after them. MFMAs and vector instructions of
// one wave alternate, because two waves on a SIMD (what 256 registers allow) do not fill it otherwise: a wave issues an
// instruction every 8 clocks at most, of any kind, while a vector instruction takes 4 and an MFMA 32. Fences to the
// scheduler keep that order; for the same reason the step is kept short of scalar work, and written out twice so that
// stages have fixed addresses and scores need no copies.
//
// ONE: pages of 64 tokens and more, so that a tile lies in one page, whose address is then a scalar.
template <int D, int W, bool ONE>
__global__ __launch_bounds__(64 * W, D == 256 && W == 4 ? 1 : 2) void prefill_kernel(AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using G = PrefillGeo<D, W>;
  constexpr int M = G::kM, T = G::kThreads, kPitch = D + 4, kSlot = M * kPitch, NX = D / 16, L = G::kLoads;
  extern __shared__ __attribute__((aligned(16))) uint8_t s_stage[];   // (ds_read_b128 off 16 bytes takes thrice as long)
  __shared__ int s_last;
  // whether a tile's V holds a NaN that some rows see and others do not (of four tiles), and where: [stage][dim][4 blocks
  // of 16 keys]
  __shared__ int s_nan[4];
  __shared__ __attribute__((aligned(16))) uint16_t s_where[2][D][4];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hf = lane >> 5;
  __shared__ int s_sum[2 * (T / 64)];
  __shared__ int s_find[4];
  __shared__ int s_mine[3 * T];
  const int groups = (int)gridDim.x;
  Segment sg;
  Entry en;
  Run run = plan_run<T>(a, M, groups, (int)blockIdx.x, s_sum, s_find, s_mine, &sg);
  const int page_mask = (1 << a.page_shift) - 1;
  uint8_t* const s_k = s_stage;                       // [2][64 keys] rows of D BF16
  uint8_t* const s_v = s_stage + 2 * G::kStageK;      // [2][D] rows of 64 keys, FP16

  while (next_segment<T>(a, M, groups, (int)blockIdx.x, s_find, s_mine, run, &sg, &en)) {
    const int t0 = sg.t0, t1 = sg.t1, head = sg.head;

    const int r = en.r0 + 32 * wave + c;
    const bool live = r < en.r1;
    const int rr = live ? r : en.r1 - 1;
    const int tok = rr / a.group;
    const int64_t q_row = en.row0 + tok;
    const int q_head = head * a.group + (rr - tok * a.group);
    const int pos = en.start + tok;
    bf16x8_t qb[NX];
    {
      const uint16_t* src = a.q + q_row * a.q_row + q_head * a.q_head + 8 * hf;
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        uint4 w = {0, 0, 0, 0};
        if (live) w = *reinterpret_cast<const uint4*>(src + 16 * x);
        qb[x] = __builtin_bit_cast(bf16x8_t, w);
      }
    }
    const int p_lo = en.start + en.r0 / a.group, p_hi = en.start + (en.r1 - 1) / a.group;
    auto key_of = [&](int t) { return kTile * (t < en.sink_tiles ? t : t + en.skip); };
    // the tiles that every row sees whole: t < whole_hi and (t >= whole_lo or t < whole_sink)
    const int whole_hi = (p_lo < 0 ? 0 : min(p_lo + 1, en.end) / kTile) - (en.skip > 0 ? en.skip : 0);
    int whole_lo = 0, whole_sink = 0;
    if (a.window > 0) {
      const int from = p_hi - a.window + 1;               // keys from here on are in every row's window
      whole_lo = from > 0 ? (from + kTile - 1) / kTile - en.skip : 0;
      whole_sink = min(a.sinks / kTile, en.sink_tiles);
    }
    auto whole_tile = [&](int t) {
      // (with skipped tiles the sink tiles lie whole below every row)
      return (t < whole_hi || (en.skip > 0 && t < whole_sink)) && (t >= whole_lo || t < whole_sink);
    };

    // staging: thread tid holds pieces tid + T i of the K block (key = piece / (D / 16)) and of the V block (dimension =
    // piece / 4, 16 keys piece % 4). The K of a tile is loaded a step before its V, from the page that `next` found
    // a step earlier still.
    const int32_t* row_table = a.table + (int64_t)en.b * a.table_stride;
    const uint8_t *k_base = a.kp + head * a.head_stride, *v_base = a.vp + head * a.head_stride;
    const uint8_t *k_exps = a.ke + head * a.exp_head_stride, *v_exps = a.ve + head * a.exp_head_stride;
    const int last = max(en.end - 1, 0);            // keys past it look its page up, and are masked
    struct Tile {
      int base;                                     // first key
      int k[ONE ? 1 : L], v;                        // pages of this thread's pieces
      uint64_t at;                                  // ONE, once its K is loaded: the bytes to its page,
      int ke, ve;                                   // the words that hold its exponents,
      bool ok;                                      // and whether it has a page
    };
    Tile next;
    auto find = [&](int t) {                        // (tiles past the run repeat its last one)
      Tile x;
      x.base = key_of(min(t, t1 - 1));
      if constexpr (ONE) {
        x.k[0] = x.v = uniform_load(row_table + (min(x.base, last) >> a.page_shift));
      } else {
#pragma unroll
        for (int i = 0; i < L; ++i) x.k[i] = row_table[min(x.base + (tid + T * i) / (D / 16), last) >> a.page_shift];
        x.v = row_table[min(x.base + 16 * (tid & 3), last) >> a.page_shift];
      }
      return x;
    };
    uint4 kw[L], vw[L];
    int kexp[L], vexp = 0;                          // exponents of the tiles to stage (ONE: K's in the tile)
    bool vok = false;                               // whether the V block holds anything
    // one byte by a scalar load of the word that holds it
    auto scalar_byte = [](const uint8_t* p) {
      const uint64_t at = (uint64_t)p;
      return uniform_load(reinterpret_cast<const int32_t*>(at & ~(uint64_t)3)) >> (8 * (int)(at & 3));
    };
    auto load_k = [&](Tile& x, int i) {
      const int32_t id = x.k[ONE ? 0 : i];
      if constexpr (ONE) {
        if (i == 0) {
          x.ok = ((uint32_t)id < a.pages) & (x.base < en.end);
          const uint32_t page = x.ok ? id : 0;
          x.at = (uint64_t)page * a.page_stride;
          const uint64_t exp = (uint64_t)page * a.exp_page_stride;
          x.ke = scalar_byte(k_exps + exp);
          x.ve = scalar_byte(v_exps + exp);
        }
        const uint8_t* block = k_base + x.at + (uint32_t)((x.base & page_mask) * D);
        kw[i] = *reinterpret_cast<const uint4*>(block + (uint32_t)(tid * 16) + 16 * T * i);
      } else {
        const uint32_t page = (uint32_t)id < a.pages ? id : 0;
        const int piece = tid + T * i;
        kw[i] = *reinterpret_cast<const uint4*>(k_base + (uint64_t)page * a.page_stride +
                                                (((x.base + piece / (D / 16)) & page_mask) * D + piece % (D / 16) * 16));
        kexp[i] = k_exps[(uint64_t)page * a.exp_page_stride];
      }
    };
    const uint32_t v_off = (uint32_t)((tid >> 2) << a.page_shift) + (ONE ? 16 * (tid & 3) : 0);
    auto load_v = [&](const Tile& x, int i) {
      if constexpr (ONE) {
        if (i == 0) {
          vok = x.ok;
          vexp = x.ve & 0xFF;
        }
        vw[i] = *reinterpret_cast<const uint4*>(v_base + x.at + (uint32_t)(x.base & page_mask) +
                                                ((uint32_t)(16 * W * i) << a.page_shift) + v_off);
      } else {
        const int key = x.base + 16 * (tid & 3);
        const bool ok = ((uint32_t)x.v < a.pages) & (key < en.end);
        const uint32_t page = ok ? x.v : 0;
        if (i == 0) {
          vok = ok;
          vexp = v_exps[(uint64_t)page * a.exp_page_stride];
        }
        vw[i] = *reinterpret_cast<const uint4*>(v_base + (uint64_t)page * a.page_stride + (uint32_t)(key & page_mask) +
                                                ((uint32_t)(16 * W * i) << a.page_shift) + v_off);
      }
    };
    int e_ref = 0;                                  // the exponent that O is held at once the staged tile is added
    float e_drop = 1.0f;                            // and what O is multiplied by before that
    float v_scale = 1.0f;
    uint32_t block_ok = 0;                          // bit b: the staged V tile's 16-key block b has a page
    bool plain = false;                             // every row sees the staged tile whole
    // before V of tile t is converted into stage buf: hidden values out of the way, and its scale
    auto prepare_v = [&](int t, int buf) {
      block_ok = ONE ? (vok ? 15u : 0u) : (uint32_t)__ballot(vok) & 15u;
      plain = whole_tile(t) && t < t1 && block_ok == 15u;
      int ev = vexp;
      if (!plain) {
        // values of keys that no row sees may be anything, NaN included: zero them
        const int j0 = key_of(min(t, t1 - 1)) + 16 * (tid & 3);
        const Sight widest = sight_of(a, p_hi, p_lo, en.end, j0), least = sight_of(a, p_lo, p_hi, en.end, j0);
        const uint32_t any = vok ? widest.bits(0, 16) : 0u, all = least.bits(0, 16);
        if (any == 0) ev = -1;
        const uint32_t some = any & ~all;
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < L; ++i) {
          vw[i].x &= byte_mask(any);
          vw[i].y &= byte_mask(any >> 4);
          vw[i].z &= byte_mask(any >> 8);
          vw[i].w &= byte_mask(any >> 12);
          // a NaN that some rows see and others do not leaves the product; the outputs that it reaches become NaN at the
          // end
          const uint32_t found = take_nan(vw[i], some);
          s_where[buf][(tid >> 2) + 16 * W * i][tid & 3] = (uint16_t)found;
          nan |= found;
        }
        if (nan) s_nan[t & 3] = 1;
      }
      int e_max = max(ev, 0);
      if (!ONE || !plain) {
        e_max = max(e_max, __shfl_xor(e_max, 1));
        e_max = max(e_max, __shfl_xor(e_max, 2));
        e_max = __builtin_amdgcn_readfirstlane(e_max);
      }
      const int e_new = max(e_ref, e_max);
      e_drop = exp_bits(127 + max(e_ref - e_new, -126));
      e_ref = e_new;
      v_scale = exp_bits(127 + max(ev - e_ref, -126));
    };
    // (the LDS places of a thread's first pieces; the others are a fixed number of rows further)
    const int k_put = key_row(tid / (D / 16)) * G::kRowK + tid % (D / 16) * 32;
    const int v_put = (tid >> 2) * G::kRowV + (tid & 3) * 32;
    auto convert_k = [&](const Tile& x, int i, int buf) {
      constexpr int kRows = T / (D / 16);           // keys between a thread's pieces: their LDS rows differ as they do
      const float ks = exp_bits(ONE ? x.ke & 0xFF : kexp[i]);
      const int put = kRows % 16 == 0 ? k_put + kRows * i * G::kRowK
                                      : key_row((tid + T * i) / (D / 16)) * G::kRowK + tid % (D / 16) * 32;
      uint8_t* dst = s_k + buf * G::kStageK + put;
      *reinterpret_cast<bf16x8_t*>(dst) = e4m3x8_to_bf16(kw[i].x, kw[i].y, ks);
      *reinterpret_cast<bf16x8_t*>(dst + 16) = e4m3x8_to_bf16(kw[i].z, kw[i].w, ks);
    };
    auto convert_v = [&](int i, int buf) {
      uint8_t* dst = s_v + buf * G::kStageV + v_put + 16 * W * i * G::kRowV;
      *reinterpret_cast<half8_t*>(dst) = e4m3x8_to_f16(vw[i].x, vw[i].y, v_scale);
      *reinterpret_cast<half8_t*>(dst + 16) = e4m3x8_to_f16(vw[i].z, vw[i].w, v_scale);
    };
    const uint8_t *k_get = s_k + c * G::kRowK + hf * 16, *v_get = s_v + c * G::kRowV + hf * 16;
    auto read_k = [&](int buf, int x, int kb) {
      return *reinterpret_cast<const bf16x8_t*>(k_get + buf * G::kStageK + 32 * kb * G::kRowK + x * 32);
    };
    auto read_v = [&](int buf, int u, int dt) {
      return *reinterpret_cast<const half8_t*>(v_get + buf * G::kStageV + 32 * dt * G::kRowV + u * 32);
    };

    float16_t acc[G::kDT];
    float m_run = -__builtin_inff(), l_run = 0.0f;
    uint32_t poison[D / 64] = {};         // outputs that a NaN reached which not every row sees: bit 16 dt + 4 a + i
#pragma unroll
    for (int dt = 0; dt < G::kDT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[dt][i] = 0.0f;

    __syncthreads();        // the stages' and flags' earlier readers are done
    if (tid < 4) s_nan[tid] = 0;
    __syncthreads();
    // K and V of the first tile and K of the second into LDS, their successors into registers; the loads of all three on
    // their way together
    Tile now = find(t0);
    next = find(t0 + 1);
    Tile third = find(t0 + 2);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      load_k(now, i);
      load_v(now, i);
    }
    uint4 k_first[L];
    int e_first[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      k_first[i] = kw[i];
      e_first[i] = kexp[i];
    }
#pragma unroll
    for (int i = 0; i < L; ++i) load_k(next, i);
    prepare_v(t0, 0);
#pragma unroll
    for (int i = 0; i < L; ++i) convert_v(i, 0);
#pragma unroll
    for (int i = 0; i < L; ++i) load_v(next, i);
    float drop = e_drop;                // of the tile whose PV comes next
    uint32_t tile_ok = block_ok;
    bool tile_plain = plain;
#pragma unroll
    for (int i = 0; i < L; ++i) convert_k(next, i, 1);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      kw[i] = k_first[i];
      kexp[i] = e_first[i];
    }
#pragma unroll
    for (int i = 0; i < L; ++i) convert_k(now, i, 0);
    now = third;
#pragma unroll
    for (int i = 0; i < L; ++i) load_k(now, i);
    next = find(t0 + 3);                // in the step of t: `now` is tile t + 2, its K loaded; `next` t + 3
    __syncthreads();
    float16_t s0[2], s1[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s0[kb][i] = 0.0f;
#pragma unroll
      for (int x = 0; x < NX; ++x)
        s0[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_k(0, x, kb), qb[x], s0[kb], 0, 0, 0);
    }
    __syncthreads();                    // K of the first tile is read before the step converts the third into its place

    // s: this tile's scores, n: the next one's; B: this tile's stage
    auto step = [&](int t, float16_t (&s)[2], float16_t (&n)[2], auto stage) {
      constexpr int B = decltype(stage)::value;
      // s[kb][4 a + i] is key base + 32 kb + 16 (a / 2) + 8 hf + 4 (a % 2) + i
      uint32_t vis = 0xFFFFFFFFu;
      const bool hidden = !tile_plain;
      if (hidden) {
        vis = 0;                              // bit 16 kb + i
        const Sight sight = sight_of(a, pos, pos, en.end, key_of(t) + 8 * hf);
#pragma unroll
        for (int u = 0; u < 4; ++u) vis |= (tile_ok >> u & 1u ? sight.bits(16 * u, 8) : 0u) << (8 * u);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[kb][i] = unless_hidden(s[kb][i], vis, 16 * kb + i);
      }
      // scores of the next tile beside this one's softmax: a quarter of the chunks for the maximum, the others for the
      // exponentials
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) n[kb][i] = 0.0f;
      xt_u32x4_t pw[4];
      float mx = -__builtin_inff(), mu = 0.0f, alpha = 1.0f, sum = 0.0f;
      constexpr int kMaxChunks = NX / 4;
      bf16x8_t kf[2][2];
      kf[0][0] = read_k(B ^ 1, 0, 0);
      kf[0][1] = read_k(B ^ 1, 0, 1);
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        if (x + 1 < NX) {
          kf[(x + 1) & 1][0] = read_k(B ^ 1, x + 1, 0);
          kf[(x + 1) & 1][1] = read_k(B ^ 1, x + 1, 1);
        }
        n[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[x & 1][0], qb[x], n[0], 0, 0, 0);
        n[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[x & 1][1], qb[x], n[1], 0, 0, 0);
        if (x < kMaxChunks) {
          constexpr int kEach = 32 / kMaxChunks;
#pragma unroll
          for (int e = 0; e < kEach; ++e) mx = fmaxf(mx, s[(x * kEach + e) >> 4][(x * kEach + e) & 15]);
          if (x == kMaxChunks - 1) {
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * a.scale;
            const float m_new = fmaxf(m_run, mx);
            mu = m_new == -__builtin_inff() ? 0.0f : m_new;
            alpha = __builtin_amdgcn_exp2f(m_run - mu);
            m_run = m_new;
          }
        } else {
          constexpr int kLeft = NX - kMaxChunks;
          const int y = x - kMaxChunks, from = 16 * y / kLeft * 2, to = 16 * (y + 1) / kLeft * 2;   // pairs
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            if (e >= from && e < to) {
              const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 4][e & 15], a.scale, -mu));
              const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 4][(e & 15) + 1], a.scale, -mu));
              sum += p0 + p1;
              uint32_t pair = pack2_16<false>(p0, p1);
              keep_here(pair);
              pw[e >> 3][(e & 7) / 2] = pair;
            }
          keep_here(sum);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      l_run = l_run * alpha + sum;
      if (hidden && s_nan[t & 3]) {
        // vis holds keys 16 u + 8 hf + i as bit 8 u + i: the row's 16-bit blocks are its bytes and the other half's
        const auto sw = __builtin_amdgcn_permlane32_swap(vis, vis, false, false);
        const uint32_t low = sw[0], high = sw[1];
#pragma unroll 1
        for (int k = 0; k < D / 2; ++k) {          // acc[k / 16][4 a + i]: dimension 32 (k / 16) + 8 a + 4 hf + i
          const uint16_t* w = s_where[B][32 * (k >> 4) + 8 * (k >> 2 & 3) + 4 * hf + (k & 3)];
          uint32_t hit = 0;
#pragma unroll
          for (int u = 0; u < 4; ++u) hit |= w[u] & ((low >> (8 * u) & 0xFFu) | (high >> (8 * u) & 0xFFu) << 8);
#pragma unroll
          for (int x = 0; x < D / 64; ++x) poison[x] |= hit && k >> 5 == x ? 1u << (k & 31) : 0u;
        }
      }
      const float f = alpha * drop;
      if (__ballot(f != 1.0f)) {
#pragma unroll
        for (int dt = 0; dt < G::kDT; ++dt) acc[dt] *= f;
      }
      prepare_v(t + 1, B ^ 1);
      drop = e_drop;
      tile_ok = block_ok;
      tile_plain = plain;
      // this tile's values beside the conversion of the next V and the K after it, each register refilled once it is
      // converted
      half8_t vf[2][G::kDT];
#pragma unroll
      for (int dt = 0; dt < G::kDT; ++dt) vf[0][dt] = read_v(B, 0, dt);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (u + 1 < 4) {
#pragma unroll
          for (int dt = 0; dt < G::kDT; ++dt) vf[(u + 1) & 1][dt] = read_v(B, u + 1, dt);
        }
#pragma unroll
        for (int dt = 0; dt < G::kDT; ++dt)
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[u & 1][dt], __builtin_bit_cast(half8_t, pw[u]), acc[dt],
                                                           0, 0, 0);
#pragma unroll
        for (int i = 0; i < L; ++i) {
          if (2 * i * 4 / (2 * L) == u) {
            convert_v(i, B ^ 1);
            load_v(now, i);
          }
          if ((2 * i + 1) * 4 / (2 * L) == u) {
            convert_k(now, i, B);
            load_k(next, i);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      now = next;
      next = find(t + 4);
      if (tid == 0) s_nan[(t + 2) & 3] = 0;      // read last two steps ago
      __syncthreads();
    };
    for (int t = t0;;) {
      step(t, s0, s1, std::integral_constant<int, 0>());
      if (++t == t1) break;
      step(t, s1, s0, std::integral_constant<int, 1>());
      if (++t == t1) break;
    }

    // every wave has its rows whole: outputs or partials straight from registers (acc[dt][4 a + i] is dimension
    // 32 dt + 8 a + 4 hf + i)
    const bool alone = sg.sharers == 1;
    const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
        a.part, (short)0, (int)min((int64_t)a.partials * kSlot * 4, (int64_t)0x7FFFFFFF), 0x00020000);
    float l = l_run;
    {
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
      l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    }
    const float f = l != 0.0f ? exp_bits(e_ref) / l : 0.0f;
    const int my_slot = sg.slot(sg.at);
    if (live) {
#pragma unroll
      for (int dt = 0; dt < G::kDT; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float4_t o = float4_t{acc[dt][4 * q], acc[dt][4 * q + 1], acc[dt][4 * q + 2], acc[dt][4 * q + 3]} * f;
          const uint32_t bad = poison[dt / 2] >> (16 * (dt & 1) + 4 * q);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = bad >> i & 1u ? __builtin_nanf("") : o[i];
          const int d = 32 * dt + 8 * q + 4 * hf;
          if (alone) store_out(a, q_row, q_head, d, o);
          else store_partial(pr, (my_slot * kSlot + (r - en.r0) * kPitch + d) * 4, o);
        }
      if (hf == 0) {
        if (!alone) store_partial(pr, (my_slot * kSlot + (r - en.r0) * kPitch + D) * 4, float4_t{m_run, l, 0.f, 0.f});
        else if (a.lse) a.lse[q_row * a.heads * a.group + q_head] = lse_of(m_run, l);
      }
    }
    if (!alone) {
      int32_t* counter = a.counters + sg.counter;
      if (arrive_last(counter, sg.sharers, &s_last)) {
        merge_partials<D, M, T, 4, 8>(a, en, head, [&](int i) { return sg.slot(i); }, sg.sharers, pr);
        reset_counter(counter);
      }
    }
  }
#endif
}

int page_shift_of(int page_size) {
  return page_size >= 16 && page_size <= 128 && (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size)
                                                                                    : -1;
}

// Query rows of a workgroup, by the rows (tokens x heads of a group) that a request has on average: 16 or 32 in the
// decode kernel, which reads its keys from memory wave by wave, up to 64 rows of a request (2 x 32 at head size 128: 16
// requests of 64 rows at 16K context take 79 us so, 106 as 1 x 64, whose registers leave a SIMD one wave, and 114 in the
// prefill kernel, half empty; at head size 64, 1 x 64 takes 56 us and 2 x 32 73); above that the prefill kernel's 32 for
// each wave: 4 waves, or 8 at head size 128 (at 64 a tile has too few pieces for 8 waves, at 256 a wave needs a SIMD's
// registers to itself), which take 2.06 ms for 4096 tokens at 32K context where 4 take 2.25.
int tile_rows(int64_t rows, int batch, int group, int dim) {
  const int64_t all = rows * group;
  if (all <= 16 * (int64_t)batch) return 16;
  if (all <= 32 * (int64_t)batch) return 32;
  if (all <= 64 * (int64_t)batch) return dim == 64 ? 64 : 32;
  return dim == 128 ? 256 : 128;
}

constexpr int64_t kMaxRows = 1 << 30;   // rows x heads of a group: 32-bit row numbers in the kernels
constexpr int64_t kMaxUnits = 1 << 23;  // (KV head, row tile) pairs: the threads of a launch stay below 2^32
constexpr int kMinTiles = 4;   // key tiles of a workgroup at least: one for each wave of the decode kernel

struct Launch {
  int m, entries, slots, groups;
  int partials;                // of m rows each
  int planned;                 // pieces of a head that a plan has room for, 0 without one
};

// The prefill kernel has one workgroup to a slot, each with at
// most two partials. The decode kernel has as many pieces as slots, or one for each (head, entry) and `sure` more a head
// (piece_of); those with partials, of entries longer than a size that goes at most `room` times into their sum, are
// fewer than twice that.
Launch plan_launch(int rows, int batch, int heads, int group, int dim, bool ragged) {
  Launch x;
  x.m = tile_rows(rows, batch, group, dim);
  const bool prefill = x.m >= 128;
  x.entries = ragged ? (int)((int64_t)rows * group / x.m) + batch : batch * ((group + x.m - 1) / x.m);
  const int per_cu = prefill ? (x.m == 256 || dim == 256 ? 1 : 2) : decode_per_cu(dim);
  x.slots = per_cu * device_cus() / 8 * 8;
  const int64_t units = (int64_t)x.entries * heads, room = x.slots > heads ? x.slots : heads;
  x.groups = prefill ? x.slots : (int)((units < kMaxUnits ? units + room + 7 : 0) / 8 * 8);
  x.partials = (int)(prefill ? 2 * x.slots : 2 * room);
  const int alone = !prefill ? 64 : x.m == 256 ? 512 : 256;      // entries that a workgroup divides by itself
  x.planned = x.entries > alone ? x.entries + (int)(room / heads) : 0;
  return x;
}

// The workspace: the fixed region of arrival counters (one per partial; at the same place for every shape, so that calls of
// any shape may share it), then the partials, then the plan: two numbers, its pieces and its entries' tiles.
size_t plan_at(const Launch& x, int dim) { return kCounterBytes + (size_t)x.partials * x.m * (dim + 4) * 4; }
size_t attention_bytes(const Launch& x, int dim) {
  return plan_at(x, dim) + (x.planned ? 32 + x.planned * sizeof(Planned) + (size_t)x.entries * 4 : 0);
}

}  // namespace
}  // namespace xt

using namespace xt;

static int check_pool(const char* what, const void* k, const void* vt, const void* k_exp, const void* v_exp,
                      int64_t pages, int heads, int dim, int page_size, int64_t* page_stride, int64_t* head_stride,
                      int64_t* exp_page_stride, int64_t* exp_head_stride) {
  if (!k || !vt || !k_exp || !v_exp) return fail(XT_EINVAL, "%s: null pool pointer", what);
  if (dim != 64 && dim != 128 && dim != 256)
    return fail(XT_EUNSUPPORTED, "%s: head size %d (64, 128 or 256)", what, dim);
  if (page_shift_of(page_size) < 0)
    return fail(XT_EUNSUPPORTED, "%s: page size %d (16, 32, 64 or 128)", what, page_size);
  if (pages < 1 || pages > 0x7FFFFFFF || heads < 1 || heads > 65535)
    return fail(XT_EINVAL, "%s: %lld pages, %d KV heads", what, (long long)pages, heads);
  const int64_t block = (int64_t)page_size * dim;
  if (*head_stride == 0) *head_stride = block;
  if (*page_stride == 0) *page_stride = *head_stride * heads;
  if (*exp_head_stride == 0) *exp_head_stride = 1;
  if (*exp_page_stride == 0) *exp_page_stride = *exp_head_stride * heads;
  if (!aligned(k, 16) || !aligned(vt, 16) || *page_stride % 16 || *head_stride % 16 || *head_stride < block ||
      *page_stride < block || *exp_head_stride < 1 || *exp_page_stride < 1)
    return fail(XT_EINVAL, "%s: blocks must be 16-byte aligned and %lld bytes or more apart (page stride %lld, head "
                "stride %lld)", what, (long long)block, (long long)*page_stride, (long long)*head_stride);
  if (*page_stride > 0xFFFFFFFFll || *exp_page_stride > 0xFFFFFFFFll)
    return fail(XT_EUNSUPPORTED, "%s: pages %lld bytes apart", what, (long long)*page_stride);
  return XT_OK;
}

static int check_rows(const char* what, const int32_t* table, int64_t table_stride, int width, const int32_t* seq_lens,
                      const int32_t* cu, int batch, int64_t rows) {
  if (!table || !seq_lens) return fail(XT_EINVAL, "%s: null table or lengths", what);
  if (width < 1 || (batch > 1 && table_stride < width))
    return fail(XT_EINVAL, "%s: table of %d columns, row stride %lld", what, width, (long long)table_stride);
  if (!cu && rows != batch)
    return fail(XT_EINVAL, "%s: %lld rows for %d requests without row offsets", what, (long long)rows, batch);
  return XT_OK;
}

extern "C" int xt_page8_append(const void* k, int64_t k_row_stride, int64_t k_head_stride, const void* v,
                               int64_t v_row_stride, int64_t v_head_stride, int64_t rows, uint8_t* k_pages,
                               uint8_t* vt_pages, uint8_t* k_exp, uint8_t* v_exp, int64_t pages, int kv_heads, int dim,
                               int page_size, int64_t page_stride, int64_t head_stride, int64_t exp_page_stride,
                               int64_t exp_head_stride, const int32_t* table, int64_t table_stride, int width,
                               const int32_t* seq_lens, const int32_t* cu_rows, int batch, xt_stream_t stream) {
  const char* what = "xt_page8_append";
  if (rows < 0 || rows > 0x7FFFFFFF || batch < 0)
    return fail(XT_EINVAL, "%s: %lld rows, %d requests", what, (long long)rows, batch);
  if (const int st = check_pool(what, k_pages, vt_pages, k_exp, v_exp, pages, kv_heads, dim, page_size, &page_stride,
                                &head_stride, &exp_page_stride, &exp_head_stride))
    return st;
  if (rows == 0 || batch == 0) return ok();
  if (const int st = check_rows(what, table, table_stride, width, seq_lens, cu_rows, batch, rows)) return st;
  if (!k || !v || !aligned(k, 16) || !aligned(v, 16) || k_row_stride % 8 || v_row_stride % 8 || k_head_stride % 8 ||
      v_head_stride % 8)
    return fail(XT_EINVAL, "%s: k and v rows must be 16-byte aligned", what);
  AppendArgs a{(const uint16_t*)k, (const uint16_t*)v, k_row_stride, k_head_stride, v_row_stride, v_head_stride, rows,
               k_pages, vt_pages, k_exp, v_exp, page_stride, head_stride, exp_page_stride, exp_head_stride, pages,
               page_shift_of(page_size), kv_heads, dim, table, table_stride, width, seq_lens, cu_rows, batch};
  const int64_t units = cu_rows ? rows / page_size + 2 * (int64_t)batch : batch;
  if (units * 1024 > 0xFFFFFFFFll)
    return fail(XT_EUNSUPPORTED, "%s: %lld rows of %d requests in one call", what, (long long)rows, batch);
  const dim3 grid((unsigned)units, kv_heads, 2);
  const size_t lds = (size_t)dim * (page_size + 4);
  // as many threads as keep a page's new rows, those that a request brings on average, in registers: 610 requests of up to 5
  // rows, 4 heads x 64, 27 us with 256 threads and 10 with 64; 574 rows, 4 x 256, pages of 128, 17 with 256 and 10 with
  // 1024; 8 x 1024 rows, 4 x 128, pages of 128, 14.4 with 256, 12.7 with 512, 15.8 with 1024
  const int64_t pieces = (rows < (int64_t)batch * page_size ? (rows + batch - 1) / batch : page_size) * (dim / 8);
  if (pieces <= 64 * kKeep) append_kernel<64><<<grid, 64, lds, stream>>>(a);
  else if (pieces <= 256 * kKeep) append_kernel<256><<<grid, 256, lds, stream>>>(a);
  else if (pieces <= 512 * kKeep) append_kernel<512><<<grid, 512, lds, stream>>>(a);
  else append_kernel<1024><<<grid, 1024, lds, stream>>>(a);
  return check_launch(what);
}

extern "C" size_t xt_page8_attention_workspace_bytes(int rows, int batch, int q_heads, int kv_heads, int dim) {
  if (rows < 0 || batch < 1 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || dim < 1 ||
      (int64_t)rows * (q_heads / kv_heads) > kMaxRows || (int64_t)batch * q_heads > kMaxRows)
    return 0;
  const size_t a = attention_bytes(plan_launch(rows, batch, kv_heads, q_heads / kv_heads, dim, true), dim);
  const size_t b = attention_bytes(plan_launch(rows, batch, kv_heads, q_heads / kv_heads, dim, false), dim);
  return a > b ? a : b;
}

template <int D, int NQ>
static int launch_decode(const char* what, const AttnArgs& a, int groups, xt_stream_t stream) {
  const size_t lds = DecodeGeo<D, NQ>::kLds;
  if (const int st = allow_lds((const void*)decode_kernel<D, NQ>, lds, what)) return st;
  decode_kernel<D, NQ><<<groups, 256, lds, stream>>>(a);
  return check_launch(what);
}

template <int D, int W, bool ONE>
static int launch_prefill_as(const char* what, const AttnArgs& a, int groups, xt_stream_t stream) {
  const size_t lds = PrefillGeo<D, W>::kLds;
  if (const int st = allow_lds((const void*)prefill_kernel<D, W, ONE>, lds, what)) return st;
  prefill_kernel<D, W, ONE><<<groups, 64 * W, lds, stream>>>(a);
  return check_launch(what);
}

template <int D, int W>
static int launch_prefill(const char* what, const AttnArgs& a, int groups, xt_stream_t stream) {
  return 1 << a.page_shift >= kTile ? launch_prefill_as<D, W, true>(what, a, groups, stream)
                                    : launch_prefill_as<D, W, false>(what, a, groups, stream);
}

extern "C" int xt_page8_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, const uint8_t* k_pages,
                                  const uint8_t* vt_pages, const uint8_t* k_exp, const uint8_t* v_exp, int64_t pages,
                                  int kv_heads, int q_heads, int dim, int page_size, int64_t page_stride,
                                  int64_t head_stride, int64_t exp_page_stride, int64_t exp_head_stride,
                                  const int32_t* table, int64_t table_stride, int width, const int32_t* seq_lens,
                                  const int32_t* cu_q, int batch, int rows, int window, int sinks, float scale,
                                  void* out, int64_t out_row_stride, int64_t out_head_stride, int out_dtype,
                                  float* lse, void* workspace, size_t workspace_bytes, xt_stream_t stream) {
  const char* what = "xt_page8_attention";
  if (rows < 0 || batch < 0 || window < 0 || sinks < 0)
    return fail(XT_EINVAL, "%s: negative size (%d rows, %d requests, window %d, %d sinks)", what, rows, batch, window,
                sinks);
  if (const int st = check_pool(what, k_pages, vt_pages, k_exp, v_exp, pages, kv_heads, dim, page_size, &page_stride,
                                &head_stride, &exp_page_stride, &exp_head_stride))
    return st;
  if (q_heads < kv_heads || q_heads % kv_heads)
    return fail(XT_EINVAL, "%s: %d query heads for %d KV heads", what, q_heads, kv_heads);
  const int group = q_heads / kv_heads;
  if (group > 128) return fail(XT_EUNSUPPORTED, "%s: %d query heads to a KV head, at most 128", what, group);
  if (!(scale > 0.0f && scale < __builtin_inff()))
    return fail(XT_EINVAL, "%s: a positive finite softmax scale expected, got %g", what, (double)scale);
  if (out_dtype != XT_DTYPE_BF16 && out_dtype != XT_DTYPE_F16)
    return fail(XT_EINVAL, "%s: output type %d", what, out_dtype);
  if (rows == 0 || batch == 0) return ok();
  if ((int64_t)rows * group > kMaxRows || (int64_t)batch * q_heads > kMaxRows)
    return fail(XT_EUNSUPPORTED, "%s: %d rows, %d requests, %d query heads", what, rows, batch, q_heads);
  if (const int st = check_rows(what, table, table_stride, width, seq_lens, cu_q, batch, rows)) return st;
  if (!q || !out || !aligned(q, 16) || q_row_stride % 8 || q_head_stride % 8 || !aligned(out, 8) ||
      out_row_stride % 4 || out_head_stride % 4)
    return fail(XT_EINVAL, "%s: query rows must be 16-byte aligned, output rows 8-byte aligned", what);
  const Launch x = plan_launch(rows, batch, kv_heads, group, dim, cu_q != nullptr);
  // (positions on the table and windows within 2^30 keep sums of two of them within 32 bits; a window that wide sees
  // every key that there is)
  if ((int64_t)width * page_size > kMaxRows)
    return fail(XT_EUNSUPPORTED, "%s: a table of %d pages of %d tokens", what, width, page_size);
  window = window > kMaxRows ? (int)kMaxRows : window;
  sinks = sinks > kMaxRows ? (int)kMaxRows : sinks;
  const int64_t tiles = ((int64_t)width * page_size + kTile - 1) / kTile;    // of an entry at most
  if (tiles > 0x7FFFFFFF / x.entries || tiles * x.entries > ((int64_t)1 << 38) / kv_heads)
    return fail(XT_EUNSUPPORTED, "%s: %d row tiles over a table of %d pages", what, x.entries, width);
  if ((int64_t)x.entries * kv_heads >= kMaxUnits)
    return fail(XT_EUNSUPPORTED, "%s: %d row tiles of %d KV heads in one call", what, x.entries, kv_heads);
  if (x.partials > kCounterSlots)
    return fail(XT_EUNSUPPORTED, "%s: %d KV heads, at most %d", what, kv_heads, kCounterSlots / 2);
  const size_t need = attention_bytes(x, dim);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
    return fail(XT_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed (256-byte aligned)", what, workspace_bytes, need);
  // no more workgroups than the table's width could keep busy
  const int64_t most = (int64_t)x.entries * kv_heads * ((tiles + kMinTiles - 1) / kMinTiles);
  const int groups = most < x.groups ? (int)((most + 7) / 8 * 8) : x.groups;
  AttnArgs a{(const uint16_t*)q, q_row_stride, q_head_stride, k_pages, vt_pages, k_exp, v_exp, (uint32_t)page_stride,
             (uint32_t)exp_page_stride, head_stride, exp_head_stride, (uint32_t)pages, page_shift_of(page_size), kv_heads,
             group, table,
             table_stride, width, seq_lens, cu_q, batch, rows, window, sinks, scale * kLog2e, out, out_row_stride,
             out_head_stride, out_dtype == XT_DTYPE_BF16 ? 1 : 0, lse, x.entries, kMinTiles, x.slots,
             (int32_t*)workspace, (float*)((uint8_t*)workspace + kCounterBytes), x.partials, nullptr, nullptr, nullptr};
  const int m = x.m;
  if (x.planned) {
    a.plan = (int*)((uint8_t*)workspace + plan_at(x, dim));
    a.planned = (Planned*)(a.plan + 8);
    a.plan_tiles = (int*)(a.planned + x.planned);
    const int room = (m >= 128 ? groups : x.slots) / kv_heads;
    plan_kernel<<<1, kPlanThreads, 0, stream>>>(a, m, room > 1 ? room : 1, m < 128);
    if (const int st = check_launch(what)) return st;
  }
  if (m == 16) {
    if (dim == 64) return launch_decode<64, 1>(what, a, groups, stream);
    if (dim == 128) return launch_decode<128, 1>(what, a, groups, stream);
    return launch_decode<256, 1>(what, a, groups, stream);
  }
  if (m == 32) {
    if (dim == 64) return launch_decode<64, 2>(what, a, groups, stream);
    if (dim == 128) return launch_decode<128, 2>(what, a, groups, stream);
    return launch_decode<256, 2>(what, a, groups, stream);
  }
  if (m == 64) return launch_decode<64, 4>(what, a, groups, stream);
  if (m == 256) return launch_prefill<128, 8>(what, a, groups, stream);
  if (dim == 64) return launch_prefill<64, 4>(what, a, groups, stream);
  return launch_prefill<256, 4>(what, a, groups, stream);
}
