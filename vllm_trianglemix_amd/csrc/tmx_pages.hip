// Pages of a paged K/V cache as units: which ones no sequence uses, sequences that start from others (shared full pages, a
// copy of the partial one), a pool closed up so that its pages in use are the lowest ones, and plain copies.  A page is a
// run of bytes, so one set of kernels serves every cache type; all layers' K and V go in one launch.  (The copies are
// what the reference's copy_blocks does per layer; which page goes where it decides on the host.)
//
// Which pages are in use follows from the block table and the sequence lengths alone -- row r holds its first
// ceil(lens[r] / page_size) entries -- so there is no count to keep in step: a sequence is freed by setting its length to
// 0.  "In use" is one bit per page; with a running count per 32-bit word every page knows its rank among the used
// (or free) ones, which is its place in every list here: no list depends on the order in which workgroups run.
#include <type_traits>

#include "tmx_common.h"

namespace tmx {

constexpr int kPagesPerLaunch = 128;  // cache pointers per launch: they travel as kernel arguments (1 KB)
struct PageCaches {
  char* at[kPagesPerLaunch];
};

struct PageTable {
  const int32_t* table;
  int64_t stride;
  const int32_t* lens;
  int rows, cols, page_shift, num_pages;
};

// entries of row r that hold pages
__device__ __forceinline__ int pg_live(const PageTable& t, int r) {
  const int64_t n = t.lens[r];
  if (n <= 0) return 0;
  const int64_t c = (n + (1ll << t.page_shift) - 1) >> t.page_shift;
  return c < t.cols ? (int)c : t.cols;
}

// pages in use before page p, from the bits and the words' running counts
__device__ __forceinline__ int pg_before(const unsigned* bits, const int* count, int p) {
  return count[p >> 5] + __popc(bits[p >> 5] & ((1u << (p & 31)) - 1u));
}
__device__ __forceinline__ bool pg_used(const unsigned* bits, int p) { return (bits[p >> 5] >> (p & 31)) & 1u; }

// Running counts over `words` words by one workgroup of 1024 threads (sm: 17 ints); the total comes back.  count[words]
// is the total too, so that pg_before answers for p = num_pages (with bits[words] = 0).
__device__ __forceinline__ int pg_scan(const unsigned* bits, int* count, int words, int* sm) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int base = 0;
  for (int w0 = 0; w0 < words; w0 += 1024) {
    const int w = w0 + tid;
    const int mine = w < words ? __popc(bits[w]) : 0;
    int inc = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(inc, d, 64);
      if (lane >= d) inc += up;
    }
    if (lane == 63) sm[wave] = inc;
    __syncthreads();
    int before = base, all = 0;
    for (int x = 0; x < 16; ++x) {
      if (x < wave) before += sm[x];
      all += sm[x];
    }
    if (w < words) count[w] = before + inc - mine;
    base += all;
    __syncthreads();
  }
  if (tid == 0) count[words] = base;
  __syncthreads();
  return base;
}

// The lists, for pages p = first, first + step, ...: free pages ascending with -1 behind them, or the moves that close the
// pool up -- of the `used` pages in use the k-th one at or past `used` goes to the k-th free page before it.
__device__ __forceinline__ void pg_emit_free(const unsigned* bits, const int* count, int num_pages, int used, int32_t* out, int first, int step) {
  for (int p = first; p < num_pages; p += step) {
    if (!pg_used(bits, p)) out[p - pg_before(bits, count, p)] = p;
    if (p >= num_pages - used) out[p] = -1;
  }
}
__device__ __forceinline__ void pg_emit_moves(const unsigned* bits, const int* count, int num_pages, int used, int2* moves, int first, int step) {
  const int low = pg_before(bits, count, used);
  for (int p = first; p < num_pages; p += step) {
    const bool u = pg_used(bits, p);
    const int before = pg_before(bits, count, p);
    if (p < used && !u) moves[p - before].y = p;
    if (p >= used && u) moves[before - low].x = p;
  }
}
// a row of the table after the moves: entries past the live ones become -1, entries that name no page stay as they are
__device__ __forceinline__ int pg_moved(const unsigned* bits, const int* count, int num_pages, int used, int low, const int2* moves, int e) {
  if (e < used || e >= num_pages) return e;
  return moves[pg_before(bits, count, e) - low].y;
}

enum { PG_FREE = 0, PG_COMPACT = 1 };

// ---- one workgroup does it all, bits and counts in LDS: tables of up to kPageSmall entries (both sides measured where it
// is launched) ----
template <int WHAT>
__global__ __launch_bounds__(1024) void pg_small_kernel(const PageTable t, int32_t* __restrict__ list, int32_t* __restrict__ total,
                                                         int32_t* __restrict__ new_table) {
  extern __shared__ unsigned pg_lds[];
  __shared__ int sm[17];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int words = (t.num_pages + 31) >> 5;
  unsigned* bits = pg_lds;                                       // [words + 1]
  int* count = reinterpret_cast<int*>(pg_lds + words + 1);       // [words + 1]
  for (int w = tid; w <= words; w += 1024) bits[w] = 0;
  __syncthreads();
  for (int r = wave; r < t.rows; r += 16) {
    const int live = pg_live(t, r);
    const int32_t* row = t.table + r * t.stride;
    for (int c = lane; c < live; c += 64) {
      const unsigned e = (unsigned)row[c];
      if (e < (unsigned)t.num_pages) atomicOr(&bits[e >> 5], 1u << (e & 31));
    }
  }
  __syncthreads();
  const int used = pg_scan(bits, count, words, sm);
  if constexpr (WHAT == PG_FREE) {
    if (tid == 0) total[0] = t.num_pages - used;
    pg_emit_free(bits, count, t.num_pages, used, list, tid, 1024);
  } else {
    int2* moves = reinterpret_cast<int2*>(list);
    const int low = pg_before(bits, count, used);
    if (tid == 0) total[0] = used, total[1] = used - low;
    pg_emit_moves(bits, count, t.num_pages, used, moves, tid, 1024);
    __threadfence_block();
    __syncthreads();
    for (int r = wave; r < t.rows; r += 16) {
      const int live = pg_live(t, r);
      const int32_t* row = t.table + r * t.stride;
      int32_t* dst = new_table + (int64_t)r * t.cols;
      for (int c = lane; c < t.cols; c += 64) dst[c] = c < live ? pg_moved(bits, count, t.num_pages, used, low, moves, row[c]) : -1;
    }
  }
}

// ---- larger ones: the same steps as launches over the whole chip, bits and counts in the work area ----
__global__ __launch_bounds__(256) void pg_clear_kernel(unsigned* bits, int words) {
  const int w = blockIdx.x * 256 + threadIdx.x;
  if (w <= words) bits[w] = 0;
}
__global__ __launch_bounds__(256) void pg_mark_kernel(const PageTable t, unsigned* bits) {
  for (int r = blockIdx.y; r < t.rows; r += gridDim.y) {
    const int live = pg_live(t, r);
    const int32_t* row = t.table + r * t.stride;
    for (int c = blockIdx.x * 256 + threadIdx.x; c < live; c += gridDim.x * 256) {
      const unsigned e = (unsigned)row[c];
      if (e < (unsigned)t.num_pages) atomicOr(&bits[e >> 5], 1u << (e & 31));
    }
  }
}
__global__ __launch_bounds__(1024) void pg_scan_kernel(const unsigned* bits, int* count, int num_pages, int what, int32_t* total) {
  __shared__ int sm[17];
  const int words = (num_pages + 31) >> 5;
  const int used = pg_scan(bits, count, words, sm);
  __threadfence_block();
  __syncthreads();
  if (threadIdx.x == 0) {
    if (what == PG_FREE) total[0] = num_pages - used;
    else total[0] = used, total[1] = used - pg_before(bits, count, used);
  }
}
template <int WHAT>
__global__ __launch_bounds__(256) void pg_emit_kernel(const unsigned* bits, const int* count, int num_pages, int32_t* list) {
  const int used = count[(num_pages + 31) >> 5];
  const int first = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
  if constexpr (WHAT == PG_FREE) pg_emit_free(bits, count, num_pages, used, list, first, step);
  else pg_emit_moves(bits, count, num_pages, used, reinterpret_cast<int2*>(list), first, step);
}
__global__ __launch_bounds__(256) void pg_table_kernel(const PageTable t, const unsigned* bits, const int* count, const int2* moves,
                                                       int32_t* new_table) {
  const int used = count[(t.num_pages + 31) >> 5];
  const int low = pg_before(bits, count, used);
  for (int r = blockIdx.y; r < t.rows; r += gridDim.y) {
    const int live = pg_live(t, r);
    const int32_t* row = t.table + r * t.stride;
    int32_t* dst = new_table + (int64_t)r * t.cols;
    for (int c = blockIdx.x * 256 + threadIdx.x; c < t.cols; c += gridDim.x * 256)
      dst[c] = c < live ? pg_moved(bits, count, t.num_pages, used, low, moves, row[c]) : -1;
  }
}

// ---- copies: bound by memory, 2 x page bytes per copy and cache.  2046 moves of 8.7 KB in 72 caches (2.56 GB read +
// written) take 519 us with the plan, 4.9 TB/s; a plain copy of 1 GiB reaches 5.15.  What it took: all moves of one cache
// before the next cache's, so that the pages in flight lie close together (595 us pair by pair); loads and stores past the
// caches (555 us with neither, 568 with cached stores); a grid of 2048 workgroups that take further chunks in turn (8 per
// CU: 524 to 530 us from 1536 to 4096). ----
// A chunk of a page, `units` 16-byte units, is copied by LANES threads: a whole workgroup, or one wave where a page is so
// small that most of a workgroup would idle (pages up to 4 KB: 8928 copies of 1088 bytes 5.6 us by waves, 9.7 by workgroups;
// 72000 of 8704 bytes 269 and 264).  A thread's four loads are under way before its first store (two at a time: 549 us for
// the case above).
template <int LANES>
__device__ __forceinline__ void pg_copy_chunk(const char* src, char* dst, int units) {
  typedef __attribute__((ext_vector_type(4))) unsigned u4;
  const int lane = (int)threadIdx.x & (LANES - 1);
  u4 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = i * LANES + lane;
    if (u < units) x[i] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(src) + u);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = i * LANES + lane;
    if (u < units) __builtin_nontemporal_store(x[i], reinterpret_cast<u4*>(dst) + u);
  }
}
// this copier's number among the launch's, and how many there are
template <int LANES>
__device__ __forceinline__ unsigned pg_copier() {
  return __builtin_amdgcn_readfirstlane(blockIdx.x * (256u / LANES) + threadIdx.x / LANES);
}

struct PageShape {
  int64_t stride;    // bytes from page to page
  int units;         // 16-byte units of a page
  int lanes;         // threads that copy a chunk: 64 or 256
  int chunk, chunks; // units per chunk (at most 4 x lanes), chunks per page
  int num_pages, num_caches;
};

template <typename T, int LANES>
__global__ __launch_bounds__(256) void pg_copy_kernel(const PageCaches caches, const PageShape s, const T* __restrict__ pairs, int cap,
                                                      const int32_t* __restrict__ count) {
  const int n = count ? imax(0, imin(cap, *count)) : cap;
  const unsigned items = (unsigned)n * s.num_caches * s.chunks;  // (below 2^31: checked before the launch)
  for (unsigned i = pg_copier<LANES>(); i < items; i += gridDim.x * (256u / LANES)) {
    const unsigned pc = i / (unsigned)s.chunks, cache = pc / (unsigned)n;
    const int ch = (int)(i - pc * s.chunks), pair = (int)(pc - cache * n);
    const int64_t a = pairs[2ll * pair], b = pairs[2ll * pair + 1];
    if (a < 0 || b < 0 || a >= s.num_pages || b >= s.num_pages || a == b) continue;
    const int u0 = ch * s.chunk;
    pg_copy_chunk<LANES>(caches.at[cache] + a * s.stride + 16ll * u0, caches.at[cache] + b * s.stride + 16ll * u0, imin(s.chunk, s.units - u0));
  }
}

template <int LANES>
__global__ __launch_bounds__(256) void pg_fork_kernel(const PageCaches caches, const PageShape s, const PageTable t,
                                                      const int32_t* __restrict__ parents, const int32_t* __restrict__ fresh, int children,
                                                      int32_t* __restrict__ child_table) {
  const int ps = 1 << t.page_shift;
  if (child_table != nullptr) {
    for (int i = blockIdx.x; i < children; i += gridDim.x) {
      const int r = parents[i];
      const bool ok = r >= 0 && r < t.rows;
      const int len = ok ? imax(t.lens[r], 0) : 0;
      const int full = len >> t.page_shift;
      const int32_t* row = t.table + (ok ? r : 0) * t.stride;
      const int f = fresh[i];
      for (int c = threadIdx.x; c < t.cols; c += 256) {
        int e = -1;
        if (c < full) e = row[c];
        else if (c == full && (len & (ps - 1)) != 0) e = f;
        child_table[(int64_t)i * t.cols + c] = e;
      }
    }
  }
  const unsigned items = (unsigned)children * s.num_caches * s.chunks;
  for (unsigned i = pg_copier<LANES>(); i < items; i += gridDim.x * (256u / LANES)) {
    const unsigned pc = i / (unsigned)s.chunks, cache = pc / (unsigned)children;
    const int ch = (int)(i - pc * s.chunks), child = (int)(pc - cache * children);
    const int r = parents[child];
    if (r < 0 || r >= t.rows) continue;
    const int len = t.lens[r], full = len >> t.page_shift;
    if (len <= 0 || (len & (ps - 1)) == 0 || full >= t.cols) continue;  // whole pages only: shared, nothing to copy
    const int a = t.table[r * t.stride + full], b = fresh[child];
    if (a < 0 || b < 0 || a >= s.num_pages || b >= s.num_pages || a == b) continue;
    const int u0 = ch * s.chunk;
    pg_copy_chunk<LANES>(caches.at[cache] + a * s.stride + 16ll * u0, caches.at[cache] + b * s.stride + 16ll * u0, imin(s.chunk, s.units - u0));
  }
}

constexpr int64_t kPageSmall = 16384;      // table entries up to which one workgroup makes the plan
constexpr int kPageSmallPages = 1 << 17;   // pages whose bits and counts it holds in LDS (32 KB)

static int pg_check_table(const char* fn, const int32_t* table, int64_t stride, int rows, int cols, const int32_t* lens, int page_size,
                          int64_t num_pages) {
  TMX_CHECK_ARG(rows >= 0 && cols >= 0 && stride >= 0 && num_pages >= 0, "%s: bad sizes", fn);
  TMX_CHECK_SUPPORTED(page_size > 0 && (page_size & (page_size - 1)) == 0, "%s: page_size %d must be a power of two", fn, page_size);
  TMX_CHECK_SUPPORTED(num_pages <= (1 << 30), "%s: more than 2^30 pages", fn);
  TMX_CHECK_SUPPORTED((int64_t)rows * cols <= 0x7fffffff, "%s: the block table has more than 2^31 - 1 entries", fn);
  TMX_CHECK_ARG(rows == 0 || cols == 0 || (table && lens), "%s: NULL pointer", fn);
  return TMX_OK;
}

static int pg_shape(const char* fn, void* const* caches, int num_caches, int64_t page_bytes, int64_t stride_page, int64_t num_pages,
                    int64_t copies, PageShape* s) {
  TMX_CHECK_ARG(num_caches >= 0 && page_bytes > 0 && num_pages >= 0, "%s: bad sizes", fn);
  TMX_CHECK_SUPPORTED(num_pages <= (1 << 30) && page_bytes <= (1 << 30), "%s: more than 2^30 pages, or a page of more than 2^30 bytes", fn);
  TMX_CHECK_SUPPORTED(page_bytes % 16 == 0 && stride_page % 16 == 0, "%s: pages must be multiples of 16 bytes (%lld, stride %lld)", fn,
                      (long long)page_bytes, (long long)stride_page);
  TMX_CHECK_ARG(stride_page >= page_bytes, "%s: pages overlap (stride %lld, %lld bytes)", fn, (long long)stride_page, (long long)page_bytes);
  TMX_CHECK_ARG(num_caches == 0 || caches != nullptr, "%s: NULL pointer", fn);
  s->units = (int)(page_bytes / 16);
  s->lanes = page_bytes <= 4096 ? 64 : 256;
  const int64_t chunks = (s->units + 4 * s->lanes - 1) / (4 * s->lanes);
  TMX_CHECK_SUPPORTED(copies * imin(num_caches, kPagesPerLaunch) * chunks <= 0x7fffffff, "%s: too many copies for one call", fn);
  for (int i = 0; i < num_caches; ++i)
    TMX_CHECK_ARG(caches[i] != nullptr && (uintptr_t)caches[i] % 16 == 0, "%s: cache %d is NULL or not 16-byte aligned", fn, i);
  s->stride = stride_page;
  s->chunks = (int)chunks;
  s->chunk = (s->units + s->chunks - 1) / s->chunks;
  s->num_pages = (int)num_pages;
  s->num_caches = num_caches;
  return TMX_OK;
}

// workgroups of a copy: enough to fill the chip eight deep, each takes further chunks in turn
static unsigned pg_grid(int64_t items, int lanes) {
  const int64_t n = (items * lanes + 255) / 256;
  return (unsigned)(n < 1 ? 1 : (n < 2048 ? n : 2048));
}

// words of bits (and of counts), one past the last among them
static int64_t pg_words(int64_t num_pages) { return (num_pages + 31) / 32 + 1; }
static bool pg_small(int64_t entries, int64_t num_pages) { return entries <= kPageSmall && num_pages <= kPageSmallPages; }

template <int WHAT>
static int pg_plan(const char* fn, const PageTable& t, int32_t* list, int32_t* total, int32_t* new_table, int32_t* work, int64_t work_ints,
                   hipStream_t s) {
  // One launch against four or five: the search for free pages takes 3.0 against 8.1 us for 8 x 64 entries, 5.6 against 11.4
  // for 64 x 128, 13.0 against 14.5 for 64 x 512 and 23.8 against 16.8 for 128 x 512; with the new table 13, 18 / 32, 26.
  if (pg_small((int64_t)t.rows * t.cols, t.num_pages)) {
    const size_t lds = 8 * (size_t)pg_words(t.num_pages);
    pg_small_kernel<WHAT><<<1, 1024, lds, s>>>(t, list, total, new_table);
  } else {
    const int64_t words = pg_words(t.num_pages);
    TMX_CHECK_ARG(work != nullptr && work_ints >= 2 * words, "%s: the work area holds %lld ints, %lld are needed (tmx_pages_work_ints)", fn,
                  (long long)work_ints, (long long)(2 * words));
    unsigned* bits = reinterpret_cast<unsigned*>(work);
    int* count = work + words;
    const int nw = (int)words - 1;
    const dim3 table_grid((unsigned)imin(64, (t.cols + 255) / 256 > 0 ? (t.cols + 255) / 256 : 1), (unsigned)imin(1024, t.rows > 0 ? t.rows : 1));
    const unsigned page_grid = (unsigned)imin(1024, t.num_pages / 256 + 1);
    pg_clear_kernel<<<(unsigned)(nw / 256 + 1), 256, 0, s>>>(bits, nw);
    pg_mark_kernel<<<table_grid, 256, 0, s>>>(t, bits);
    pg_scan_kernel<<<1, 1024, 0, s>>>(bits, count, t.num_pages, WHAT, total);
    pg_emit_kernel<WHAT><<<page_grid, 256, 0, s>>>(bits, count, t.num_pages, list);
    if (WHAT == PG_COMPACT) pg_table_kernel<<<table_grid, 256, 0, s>>>(t, bits, count, reinterpret_cast<const int2*>(list), new_table);
  }
  TMX_CHECK_HIP(hipGetLastError());
  return TMX_OK;
}

}  // namespace tmx

extern "C" int64_t tmx_pages_work_ints(int32_t rows, int32_t cols, int64_t num_pages) {
  using namespace tmx;
  return num_pages < 0 || pg_small((int64_t)rows * cols, num_pages) ? 0 : 2 * pg_words(num_pages);
}

extern "C" int tmx_free_pages(const int32_t* block_table, int64_t block_table_stride, int32_t rows, int32_t cols, const int32_t* seq_lens,
                              int32_t page_size, int64_t num_pages, int32_t* free_out, int32_t* count_out, int32_t* work, int64_t work_ints,
                              void* stream) {
  using namespace tmx;
  const int rc = pg_check_table("tmx_free_pages", block_table, block_table_stride, rows, cols, seq_lens, page_size, num_pages);
  if (rc != TMX_OK) return rc;
  TMX_CHECK_ARG(count_out != nullptr && (num_pages == 0 || free_out != nullptr), "tmx_free_pages: NULL pointer");
  const PageTable t{block_table, block_table_stride, seq_lens, cols ? rows : 0, cols, __builtin_ctz(page_size), (int)num_pages};
  return pg_plan<PG_FREE>("tmx_free_pages", t, free_out, count_out, nullptr, work, work_ints, (hipStream_t)stream);
}

extern "C" int tmx_plan_compaction(const int32_t* block_table, int64_t block_table_stride, int32_t rows, int32_t cols, const int32_t* seq_lens,
                                   int32_t page_size, int64_t num_pages, int32_t* new_table, int32_t* moves_out, int32_t* totals_out,
                                   int32_t* work, int64_t work_ints, void* stream) {
  using namespace tmx;
  const int rc = pg_check_table("tmx_plan_compaction", block_table, block_table_stride, rows, cols, seq_lens, page_size, num_pages);
  if (rc != TMX_OK) return rc;
  TMX_CHECK_ARG(totals_out != nullptr && moves_out != nullptr && (rows == 0 || cols == 0 || new_table != nullptr),
                "tmx_plan_compaction: NULL pointer");
  TMX_CHECK_ARG((uintptr_t)moves_out % 8 == 0, "tmx_plan_compaction: moves must be 8-byte aligned");
  const PageTable t{block_table, block_table_stride, seq_lens, cols ? rows : 0, cols, __builtin_ctz(page_size), (int)num_pages};
  return pg_plan<PG_COMPACT>("tmx_plan_compaction", t, moves_out, totals_out, new_table, work, work_ints, (hipStream_t)stream);
}

extern "C" int tmx_copy_pages(void* const* caches, int32_t num_caches, int64_t page_bytes, int64_t stride_page, int64_t num_pages,
                              const void* pairs, int32_t pair_bits, int32_t num_pairs, const int32_t* count, void* stream) {
  using namespace tmx;
  TMX_CHECK_ARG(num_pairs >= 0, "tmx_copy_pages: bad sizes");
  PageShape s{};
  const int rc = pg_shape("tmx_copy_pages", caches, num_caches, page_bytes, stride_page, num_pages, num_pairs, &s);
  if (rc != TMX_OK) return rc;
  TMX_CHECK_SUPPORTED(pair_bits == 32 || pair_bits == 64, "tmx_copy_pages: pairs are int32 or int64");
  if (num_pairs == 0 || num_caches == 0 || num_pages == 0) return TMX_OK;
  TMX_CHECK_ARG(pairs != nullptr, "tmx_copy_pages: NULL pointer");
  for (int c0 = 0; c0 < num_caches; c0 += kPagesPerLaunch) {
    PageCaches p;
    s.num_caches = imin(kPagesPerLaunch, num_caches - c0);
    for (int i = 0; i < s.num_caches; ++i) p.at[i] = (char*)caches[c0 + i];
    for (int i = s.num_caches; i < kPagesPerLaunch; ++i) p.at[i] = nullptr;
    const unsigned grid = pg_grid((int64_t)num_pairs * s.num_caches * s.chunks, s.lanes);
    auto launch = [&](auto lanes) {
      constexpr int L = decltype(lanes)::value;
      if (pair_bits == 64) pg_copy_kernel<int64_t, L><<<grid, 256, 0, (hipStream_t)stream>>>(p, s, (const int64_t*)pairs, num_pairs, count);
      else pg_copy_kernel<int32_t, L><<<grid, 256, 0, (hipStream_t)stream>>>(p, s, (const int32_t*)pairs, num_pairs, count);
    };
    if (s.lanes == 64) launch(std::integral_constant<int, 64>{});
    else launch(std::integral_constant<int, 256>{});
    TMX_CHECK_HIP(hipGetLastError());
  }
  return TMX_OK;
}

extern "C" int tmx_fork_pages(void* const* caches, int32_t num_caches, int64_t page_bytes, int64_t stride_page, int64_t num_pages,
                              const int32_t* block_table, int64_t block_table_stride, int32_t rows, int32_t cols, const int32_t* seq_lens,
                              int32_t page_size, const int32_t* parents, const int32_t* fresh, int32_t children, int32_t* child_table,
                              void* stream) {
  using namespace tmx;
  TMX_CHECK_ARG(children >= 0, "tmx_fork_pages: bad sizes");
  PageShape s{};
  int rc = pg_shape("tmx_fork_pages", caches, num_caches, page_bytes, stride_page, num_pages, children, &s);
  if (rc != TMX_OK) return rc;
  rc = pg_check_table("tmx_fork_pages", block_table, block_table_stride, rows, cols, seq_lens, page_size, num_pages);
  if (rc != TMX_OK) return rc;
  if (children == 0 || cols == 0) return TMX_OK;
  TMX_CHECK_SUPPORTED((int64_t)children * cols <= 0x7fffffff, "tmx_fork_pages: the children's table has more than 2^31 - 1 entries");
  TMX_CHECK_ARG(parents && fresh && child_table, "tmx_fork_pages: NULL pointer");
  const PageTable t{block_table, block_table_stride, seq_lens, rows, cols, __builtin_ctz(page_size), (int)num_pages};
  for (int c0 = 0; c0 == 0 || c0 < num_caches; c0 += kPagesPerLaunch) {
    PageCaches p;
    s.num_caches = imin(kPagesPerLaunch, num_caches - c0);
    for (int i = 0; i < s.num_caches; ++i) p.at[i] = (char*)caches[c0 + i];
    for (int i = s.num_caches; i < kPagesPerLaunch; ++i) p.at[i] = nullptr;
    const int64_t items = (int64_t)children * (s.num_caches > 0 ? s.num_caches : 1) * s.chunks;
    auto* kernel = s.lanes == 64 ? pg_fork_kernel<64> : pg_fork_kernel<256>;
    kernel<<<pg_grid(items, s.lanes), 256, 0, (hipStream_t)stream>>>(p, s, t, parents, fresh, children, c0 == 0 ? child_table : nullptr);
    TMX_CHECK_HIP(hipGetLastError());
  }
  return TMX_OK;
}
