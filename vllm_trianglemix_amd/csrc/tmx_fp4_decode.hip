// Attention of a step's query rows against a 4-bit (MXFP4) paged K/V cache, for gfx950 (MI355X): one row per request
// (decode) or the last few positions of each (drafted tokens checked in one step).  Such a step reads all of its K/V
// once and multiplies little, so it is bound by the bytes of the cache; what the kernel has to do is ask for them in whole
// lines, early, and keep the vector units out of their way.
//
//   workgroup = 4 waves = a span of 32-key tiles x one K/V head; the waves take the span's tiles in turn and meet only at
//   a request's end.  Rows = rows_per_request x (query heads per K/V head), up to 32 of them columns of the same products, so
//   a head's K/V are read and converted once for them whatever the group size.  33 to 64 rows are two groups, each with
//   workgroups of its own that read and convert K/V again (16 x 2878 .. 4111 tokens, 64 / 8 heads, bf16, 1 / 2 / 4 / 8 rows per
//   request, i.e. 8 to 64 per K/V head: 19.8 / 21.5 / 30.9 / 43.0 us).
//   Scores S^T = K Q^T (v_mfma_f32_16x16x32_bf16, D / 32 of them per 16 keys): lane (m = lane % 16, g = lane / 16) holds
//   columns [g D/4, (g + 1) D/4) of key row m, one load and one scale; the codes become bf16, which is exact (one fraction
//   bit, power-of-two scales).  The head dimension may be summed in any order as long as Q^T is laid out alike.  fp16
//   queries are split into two bf16 terms (exact: 11 bits in 8 + 8).  (The scaled product that takes 4-bit operands as
//   they are would save these conversions, but it sums 8 neighbouring products with some 14 bits below the largest of
//   them: a query column 2^7 below its neighbours would not count.)
//   Output O^T = V^T P^T (the same product): lane (m, g) needs columns [m D/16, (m + 1) D/16) of the 8 keys whose scores
//   it holds, 4 g .. 4 g + 3 and 16 + 4 g .. + 3.  The cache keeps V in that order (tmx_fp4.h), so V comes straight from
//   memory, becomes bf16 by 32 conversions and is paired by 32 byte permutes; the probabilities never leave their lane.
//   No LDS in the loop.
//   Probabilities are held as two bf16 terms (16 significant bits; one term alone would cost as much accuracy as the
//   rounding of the output).  Up to 8 rows, columns 8..15 repeat the rows and carry the second term: no extra product.
//   Their sum is one more product, with ones.
//   Every load instruction of the loop reads one contiguous run of a page-half (16 keys: 1 KB of codes, 512 bytes at head
//   size 64) from a scalar base.
//   The running maximum is raised only when a score exceeds it by more than 2^kSlack (factors stay below 2^8 in fp32).
#include <atomic>
#include <type_traits>

#include "tmx_common.h"
#include "tmx_fp4.h"

namespace tmx {

typedef __attribute__((ext_vector_type(4))) float f4_f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 f4_bf16x8;
typedef __attribute__((ext_vector_type(2))) float f4_f32x2;

constexpr float kFp4MinusBig = -3.0e38f;  // below every finite score, and finite
constexpr float kFp4Slack = 8.0f;

struct Fp4DecodeParams {
  const void* q;
  void* out;
  const uint8_t* k;
  const uint8_t* v;
  int64_t stride_page;
  int num_pages;
  const int32_t* block_table;
  int64_t block_table_stride;
  int max_blocks, page_shift;
  const int32_t* seq_lens;
  int batch, m, H, Hkv, G;
  int len_cap;  // keys the block table has room for, + m: longer sequences read as this long (and as NaN)
  int64_t q_stride_t, q_stride_h, out_stride_t, out_stride_h;  // elements
  int out_f32;
  float scale_log2;
  float* partial_o;   // [slot][row of the request][head][D]
  float* partial_ml;  // [slot][row of the request][head][2]
  int* pieces;        // [request][2]: the span its first tile lies in, the number of spans that hold its tiles
  int spans;       // workgroups per unit
  int row_groups;  // groups of 32 rows of a K/V head, each with workgroups of its own
  int units;       // K/V heads x row groups
};

// Asks for the arguments at once.  They lie in four cache lines, and loads placed where each value is first used miss one after
// the other (1 x 517: 9.0 -> 8.5 us, 8 x 65536 of one K/V head 21.6 -> 21.0).
__device__ __forceinline__ void fp4_ask_for_arguments(const Fp4DecodeParams& p) {
  asm volatile("" ::"s"(p.q), "s"(p.out), "s"(p.k), "s"(p.v), "s"(p.stride_page), "s"(p.num_pages), "s"(p.block_table),
               "s"(p.block_table_stride), "s"(p.max_blocks), "s"(p.page_shift), "s"(p.seq_lens), "s"(p.batch), "s"(p.m), "s"(p.G),
               "s"(p.len_cap), "s"(p.q_stride_t), "s"(p.q_stride_h), "s"(p.scale_log2), "s"(p.partial_o), "s"(p.spans), "s"(p.units));
}

template <typename T>
__device__ __forceinline__ T fp4_sload(const T* ptr) {  // uniform address: through the scalar cache
  return *reinterpret_cast<const __attribute__((address_space(4))) T*>((const __attribute__((address_space(4))) void*)ptr);
}
__device__ __forceinline__ unsigned fp4_pack_bf16(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f4_f32x2{a, b}, fp4_bf16x2));
}
// the value of lane ^ 8 (within 16 lanes a rotation by 8)
__device__ __forceinline__ float fp4_other8(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, true));
}
__device__ __forceinline__ float fp4_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ void fp4_store_out(void* out, int64_t at, float x, bool f32, bool bf16) {
  if (f32) reinterpret_cast<float*>(out)[at] = x;
  else if (bf16) reinterpret_cast<__bf16*>(out)[at] = (__bf16)x;
  else reinterpret_cast<_Float16*>(out)[at] = (_Float16)x;
}

// ---- the plan: the 32-key tiles of all requests, one after the other, are cut into equal spans, one per workgroup and
// K/V head, whatever the requests' lengths are.  A request's beginning counts as kFp4Begin tiles more: what it costs to
// change over (queries split anew, the waves' sums joined and written).  A span may begin and end inside requests: piece
// (span w, request b) of a request that lies in several spans leaves its result in slot w + b -- both only grow along the
// tiles, so no two pieces share a slot -- and the pieces are joined afterwards.  Every wave works the plan out for itself,
// without a barrier: lane l counts the tiles of a run of requests, six lane moves sum them up.  The join does not: the workgroup
// of a request's first tile has noted which spans hold it (1024 requests of 64 tokens 122 -> 62 us, 1 x 517 10.7 -> 9.1). ----
constexpr int kFp4MinSpan = 4;  // a tile per wave
constexpr int kFp4Begin = 12;
__device__ __forceinline__ int fp4_len(const Fp4DecodeParams& p, int n) { return imin(n, p.len_cap); }
__device__ __forceinline__ int fp4_tiles(int n) { return n > 0 ? (n + kBlockN - 1) / kBlockN : 0; }
__device__ __forceinline__ int fp4_cost(int n) { return n > 0 ? fp4_tiles(n) + kFp4Begin : 0; }
__device__ __forceinline__ int fp4_span(int tiles, int spans) {
  const int c = ((tiles + spans - 1) / spans + 3) & ~3;
  return imax(c, kFp4MinSpan);
}
struct Fp4Plan {
  int per;                  // requests per lane
  int len;                  // the last one's length (per == 1: lane b holds request b's)
  int mine, before, total;  // cost of this lane's requests, of those before them, of all
};
__device__ __forceinline__ Fp4Plan fp4_plan(const Fp4DecodeParams& p, int lane) {
  Fp4Plan r;
  r.per = (p.batch + 63) >> 6;
  const int j0 = imin(p.batch, lane * r.per), j1 = imin(p.batch, j0 + r.per);
  r.mine = r.len = 0;
#pragma unroll 8
  for (int j = j0; j < j1; ++j) {
    r.len = fp4_len(p, p.seq_lens[j]);
    r.mine += fp4_cost(r.len);
  }
  // inclusive sum over the lanes: within rows of 16, then the rows' totals down the wave
  int inc = r.mine;
  inc += __builtin_amdgcn_update_dpp(0, inc, 0x111, 0xf, 0xf, false);  // row_shr:1
  inc += __builtin_amdgcn_update_dpp(0, inc, 0x112, 0xf, 0xf, false);  // row_shr:2
  inc += __builtin_amdgcn_update_dpp(0, inc, 0x114, 0xf, 0xf, false);  // row_shr:4
  inc += __builtin_amdgcn_update_dpp(0, inc, 0x118, 0xf, 0xf, false);  // row_shr:8
  inc += __builtin_amdgcn_update_dpp(0, inc, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  inc += __builtin_amdgcn_update_dpp(0, inc, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  r.before = inc - r.mine;
  r.total = __builtin_amdgcn_readlane(inc, 63);
  return r;
}

// request b's length (uniform): from the lane that counted it, or from memory
__device__ __forceinline__ int fp4_len_of(const Fp4DecodeParams& p, const Fp4Plan& plan, int b) {
  return plan.per == 1 ? __builtin_amdgcn_readlane(plan.len, b) : fp4_len(p, fp4_sload(p.seq_lens + b));
}

// Workgroups resident per CU.  Two per CU with a tile read ahead per wave have 70 KB in flight at head size 128, all that the
// memory system takes (whole calls on inputs that no cache holds: 64 x 8192 tokens 92.2 us with two, 99.1 with three, 95.4
// with two that read two tiles ahead; 4 x 16384 21.0 and 22.9 with three; 32 ragged requests 33.2 and 35.2).  Head size 64 has
// half the bytes per tile and would leave room for four, but gains nothing by it (bf16, 4 rows per K/V head, two / three /
// four: 64 x 8192 65 / 65 / 67 us, 32 ragged requests 25.4 / 24.9 / 25.9, 8 x 65536 of one K/V head 17.7 / 17.7 / 19.4; fp16,
// 16 rows: 67 / 72 / 69, 27.0 / 27.5 / 28.5, 19.3 / 19.4 / 21.7, with registers spilled at four).
constexpr int kFp4WgsPerCu = 2;

// NT column tiles of 16 rows; HALF: one tile, at most 8 rows, columns 8..15 carry the probabilities' second terms
template <int D, bool BF16, int NT, bool HALF>
__global__ __launch_bounds__(256, kFp4WgsPerCu) void fp4_decode_kernel(const Fp4DecodeParams p) {
  static_assert(!HALF || NT == 1, "the half form has one tile");
  constexpr int DT = D / 16;        // row tiles of the second product
  constexpr int VW = D / 32;        // words of V codes per lane and page-half
  constexpr int KS = D / 32;        // k-steps of the first product
  constexpr int TERMS = BF16 ? 1 : 2;  // of the query
  constexpr int ROWS = HALF ? 8 : 16 * NT;
  __shared__ __attribute__((aligned(16))) float sm_o[4][ROWS][D + 4];  // (+ 4: the rows a wave writes at once start in different banks)
  __shared__ f4_f32x2 sm_ml[4][ROWS];

  fp4_ask_for_arguments(p);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  // Workgroups go round the 8 XCDs: this order gives an XCD a run of spans with all their heads, so that the heads of a
  // page -- and the cache lines in which two heads' scale bytes meet -- are read through one L2 at about the same time
  // (64 x 8192 tokens, 32 / 8 heads: 92.6 us against 95.2 with the heads spread over the XCDs; head size 64 64.0 against 65.9).
  const int lin = ((int)blockIdx.x & 7) * ((int)gridDim.x >> 3) + ((int)blockIdx.x >> 3);
  const int w = lin / p.units, unit = lin - w * p.units;
  const int h = unit / p.row_groups, row0 = 32 * (unit - h * p.row_groups);
  if (w >= p.spans) return;
  // A SIMD issues for its oldest wave first: of two workgroups on a CU the one launched first finished its equal span at 75 us,
  // the other at 89 us, alone with its loads at the end.  The younger half of the grid takes precedence on every other tile, and
  // both finish together (64 x 8192 tokens: the whole call 96.7 -> 92.2 us, 32 ragged requests 34.0 -> 33.2).
  const bool younger = blockIdx.x >= gridDim.x / 2;

  // the request at which this workgroup's span begins, and where in it
  int b, off, left, line, span;  // line: where the request begins on the line of all tiles
  const Fp4Plan plan = fp4_plan(p, lane);
  {
    span = fp4_span(plan.total, p.spans);
    const long long begin_ = (long long)w * span;
    if (begin_ >= plan.total) return;  // fewer spans in this step than the grid provides for
    const int begin = (int)begin_;
    const unsigned long long own = __ballot(begin >= plan.before && begin < plan.before + plan.mine);
    const int src = __builtin_ctzll(own);  // (one lane holds it: begin < total)
    b = src * plan.per;
    int at = __builtin_amdgcn_readlane(plan.before, src);
    for (; b < p.batch - 1; ++b) {
      const int cj = fp4_cost(fp4_len_of(p, plan, b));
      if (begin < at + cj) break;
      at += cj;
    }
    line = at;
    off = begin - at - kFp4Begin;  // (negative: the request begins in this span)
    left = imin(plan.total - begin, span);
  }
  const int R = imin(p.m * p.G - row0, ROWS);  // this workgroup's rows: row0 .. row0 + R - 1 of the head
  const int ps = 1 << p.page_shift;
  const int64_t head_codes = (int64_t)h * ps * (D / 2);
  const int scales_from_codes = (int)(fp4_code_bytes(p.Hkv, ps, D) + (int64_t)h * ps * (D / 32) - head_codes);
  // byte offsets of a lane inside a page-half of a head
  const int k_lane = c16 * (D / 2) + g * (D / 8);
  const int v_lane = D == 128 ? g * 256 + c16 * 16 : (g >> 1) * 256 + c16 * 16 + (g & 1) * 8;
  const int ks_lane = (D == 128 ? g : g >> 1) * ps + (c16 & ~3), ks_shift = 8 * (c16 & 3);
  const int vs_lane = (D == 128 ? c16 >> 2 : c16 >> 3) * ps + 4 * g;

  struct Raw {
    unsigned k[2][KS];               // D / 4 codes of key 16 x + c16
    unsigned v[2 * VW];              // codes of keys 4 g .. + 3 and 16 + 4 g .. + 3, D / 16 columns each
    unsigned ks[2];                  // scale bytes of four keys, key 16 x + c16 among them (a word: a byte would be widened at once,
                                     // which waits for it)
    unsigned vs[2];                  // four keys' scale bytes each
    unsigned bad;                    // bit x: half x has no page
  };
  struct Pages {
    int e0, e1;
  };
  // The piece of a request that is being computed: keys, tiles tile0 .. tile_end - 1, of which every row attends to all keys
  // of those before full_end
  int n, tile_end, full_end, t0;
  bool whole;
  const int32_t* bt;
  uint4 qraw[NT][D / 32];  // (asked for one piece ahead as long as the registers allow)
  constexpr bool QAHEAD = NT == 1;
  Raw ring[2];  // the tile that is computed and the next one
  Pages pg{0, 0};

  // The pages of a tile, looked up a tile ahead of its loads.  (Past the row's end its last entry is read and not used.)
  auto pages_of = [&](int tile, Pages& pg) {
    const int key0 = tile * kBlockN;
    const int key1 = key0 + 16 < n ? key0 + 16 : key0;  // a half past the end reads the first one again
    const int blk0 = key0 >> p.page_shift, blk1 = key1 >> p.page_shift, last = p.max_blocks - 1;
    const int e0 = fp4_sload(bt + imax(imin(blk0, last), 0)), e1 = fp4_sload(bt + imax(imin(blk1, last), 0));
    pg.e0 = blk0 <= last ? e0 : -1;
    pg.e1 = blk1 <= last ? e1 : -1;
  };
  // `there` is false past the piece's end: the loads are made all the same, from buffers of no length, which touches no
  // memory.  With a branch around them the compiler cannot count the loads in flight, and every second tile waited for the
  // next one's (whole calls: 64 x 8192 tokens 100.4 -> 92.3 us, 32 ragged requests 34.2 -> 33.1).
  auto load = [&](int tile, const Pages& pg, Raw& r, bool there) {
    const int size = there ? 0x7fffffff : 0;
    const int key0 = tile * kBlockN;
    const int key1 = key0 + 16 < n ? key0 + 16 : key0;
    r.bad = ((unsigned)pg.e0 >= (unsigned)p.num_pages ? 1u : 0u) | ((unsigned)pg.e1 >= (unsigned)p.num_pages ? 2u : 0u);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int e = (r.bad >> x) & 1 ? 0 : (x ? pg.e1 : pg.e0);
      const int at = (x ? key1 : key0) & (ps - 1);
      const int64_t base = e * p.stride_page + head_codes + at * (D / 2);
      const int scales = scales_from_codes + at - at * (D / 2);
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.k) + base, 0, size, 0x00020000);
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.v) + base, 0, size, 0x00020000);
      constexpr int kStream = 2;  // codes are read once: non-temporal (64 x 8192: 92.2 against 106.0 us; 32 ragged requests 33.2 and 38.3)
      if constexpr (D == 128) {
        const fp4_u32x4 z = __builtin_bit_cast(fp4_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_lane, 0, kStream));
#pragma unroll
        for (int i = 0; i < 4; ++i) r.k[x][i] = z[i];
        const fp4_u32x4 y = __builtin_bit_cast(fp4_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, v_lane, 0, kStream));
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[4 * x + i] = y[i];
      } else {
        const fp4_u32x2 z = __builtin_bit_cast(fp4_u32x2, __builtin_amdgcn_raw_buffer_load_b64(rk, k_lane, 0, kStream));
        r.k[x][0] = z[0];
        r.k[x][1] = z[1];
        const fp4_u32x2 y = __builtin_bit_cast(fp4_u32x2, __builtin_amdgcn_raw_buffer_load_b64(rv, v_lane, 0, kStream));
        r.v[2 * x] = y[0];
        r.v[2 * x + 1] = y[1];
      }
      r.ks[x] = (unsigned)__builtin_amdgcn_raw_buffer_load_b32(rk, ks_lane, scales, 0);
      r.vs[x] = (unsigned)__builtin_amdgcn_raw_buffer_load_b32(rv, vs_lane, scales, 0);
    }
  };
  // Query rows: lane column c16 = row, k-step i covers columns g D/4 + 8 i .. + 7.  Row r is position n - m + r / G, head
  // h G + r % G.
  auto load_q = [&]() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int x = HALF ? (c16 & 7) : 16 * t + c16;
      const int r = row0 + (x < R ? x : 0);  // (columns without a row repeat the first)
      const int j = r / p.G, hd = h * p.G + (r - j * p.G);
      const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + ((int64_t)b * p.m + j) * p.q_stride_t + hd * p.q_stride_h;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) qraw[t][i] = *reinterpret_cast<const uint4*>(src + g * (D / 4) + 8 * i);
    }
  };
  // The next piece of the span: its query rows and first tiles are asked for here, before the one that ends is written out.
  auto start = [&]() {
    n = fp4_len_of(p, plan, b);
    const int tiles = fp4_tiles(n), take = imin(left, tiles - off);
    left -= take;
    tile_end = off + take;
    if (off <= 0 && unit == 0 && tid == 0) {  // the request's first tile: where its pieces are, for their join
      p.pieces[2 * b] = w;
      p.pieces[2 * b + 1] = (line + kFp4Begin + tiles - 1) / span - w + 1;
    }
    line += kFp4Begin + tiles;
    off = imax(off, 0);
    whole = off == 0 && tile_end == tiles;
    full_end = imin(tile_end, imax(0, n - p.m + 1) / kBlockN);
    t0 = off + wave;
    bt = p.block_table + b * p.block_table_stride;
    if constexpr (QAHEAD) load_q();
    pages_of(t0, pg);
    load(t0, pg, ring[0], t0 < tile_end);
    pages_of(t0 + 4, pg);
  };

  if (left + imin(off, 0) <= 0) return;  // (the span holds no more than a request's beginning)
  start();
  for (;;) {
    if constexpr (!QAHEAD) load_q();
    uint4 qt[NT][TERMS][KS];
    int pos[NT];  // the position of this lane's row
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = HALF ? (c16 & 7) : 16 * t + c16;
      pos[t] = n - p.m + (row0 + (row < R ? row : 0)) / p.G;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        if constexpr (BF16) {
          qt[t][0][i] = qraw[t][i];
        } else {
          const unsigned xs[4] = {qraw[t][i].x, qraw[t][i].y, qraw[t][i].z, qraw[t][i].w};
          unsigned hi[4], lo[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const fp4_f16x2 f = __builtin_bit_cast(fp4_f16x2, xs[y]);
            const float f0 = (float)f[0], f1 = (float)f[1];
            hi[y] = fp4_pack_bf16(f0, f1);
            const float h0 = __uint_as_float(hi[y] << 16), h1 = __uint_as_float(hi[y] & 0xffff0000u);
            // (an infinity less itself is NaN: so is its row without it)
            lo[y] = fp4_pack_bf16(f0 - h0, f1 - h1);
          }
          qt[t][0][i] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          qt[t][TERMS - 1][i] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
    }

    f4_f32x4 o[NT][DT], l[NT];
    float mx[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      mx[t] = kFp4MinusBig;
      l[t] = f4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DT; ++i) o[t][i] = f4_f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // The conversion takes the exponent field of its scale alone: the byte moved there, whatever lies around it.
    auto scale_of = [](unsigned word, int byte) -> float { return __uint_as_float(byte < 3 ? word << (23 - 8 * byte) : word >> 1); };

    // ---- O^T += V^T P^T with the probabilities in pb (and their second terms in pl unless HALF), one byte of every
    // key's codes -- a pair of columns, two row tiles -- at a time; and the probabilities' sums ----
    auto weighted_sum = [&](const Raw& r, const uint4 (&pb)[NT], const uint4 (&pl)[NT]) {
      const f4_bf16x8 ones = __builtin_bit_cast(f4_bf16x8, make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        l[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(f4_bf16x8, pb[t]), l[t], 0, 0, 0);
        if constexpr (!HALF) l[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(f4_bf16x8, pl[t]), l[t], 0, 0, 0);
      }
      float sc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) sc[j] = scale_of(r.vs[j >> 2], j & 3);
      auto pair = [&](auto at) {
        constexpr int B = decltype(at)::value;
        unsigned c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (D == 128) c[j] = fp4_bf16<B>(r.v[j], sc[j]);
          else c[j] = (j & 1) ? fp4_bf16<2 + (B & 1)>(r.v[j >> 1], sc[j]) : fp4_bf16<B & 1>(r.v[j >> 1], sc[j]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const unsigned sel = e ? 0x07060302u : 0x05040100u;
          const f4_bf16x8 av = __builtin_bit_cast(f4_bf16x8, make_uint4(
              __builtin_amdgcn_perm(c[1], c[0], sel), __builtin_amdgcn_perm(c[3], c[2], sel),
              __builtin_amdgcn_perm(c[5], c[4], sel), __builtin_amdgcn_perm(c[7], c[6], sel)));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            f4_f32x4& d = o[t][2 * B + e];
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, __builtin_bit_cast(f4_bf16x8, pb[t]), d, 0, 0, 0);
            if constexpr (!HALF) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, __builtin_bit_cast(f4_bf16x8, pl[t]), d, 0, 0, 0);
          }
        }
      };
      pair(std::integral_constant<int, 0>{});
      pair(std::integral_constant<int, 1>{});
      if constexpr (D == 128) {
        pair(std::integral_constant<int, 2>{});
        pair(std::integral_constant<int, 3>{});
      }
    };
    // takes key j (of the lane's 8) out of V
    auto drop_key = [&](Raw& r, int j) {
      if constexpr (D == 128) r.v[j] = 0;
      else r.v[j >> 1] &= (j & 1) ? 0x0000ffffu : 0xffff0000u;
      r.vs[j >> 2] &= ~(0xffu << (8 * (j & 3)));
    };

    // TAIL: the tile may hold keys past a row's position, or past the sequence (their V must not enter even as 0 x NaN)
    auto process = [&](auto tail_, Raw& r, int tile) {
      constexpr bool TAIL = decltype(tail_)::value;
      const int key0 = tile * kBlockN + 4 * g;  // the lane's keys: key0 + 16 (j / 4) + j % 4
      if (r.bad) {  // keys without a page count as NaN
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if ((r.bad >> x) & 1) r.ks[x] = r.vs[x] = ~0u;
      }
      // scores
      f4_f32x4 s[NT][2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float sc = __uint_as_float((r.ks[x] >> ks_shift) << 23);
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][x] = f4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const unsigned word = r.k[x][i];
          const f4_bf16x8 a = __builtin_bit_cast(f4_bf16x8, make_uint4(fp4_bf16<0>(word, sc), fp4_bf16<1>(word, sc), fp4_bf16<2>(word, sc), fp4_bf16<3>(word, sc)));
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int z = TERMS - 1; z >= 0; --z)
              s[t][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(f4_bf16x8, qt[t][z][i]), s[t][x], 0, 0, 0);
        }
      }
      if (TAIL && tile * kBlockN + kBlockN > n) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (key0 + 16 * (j >> 2) + (j & 3) >= n) drop_key(r, j);
      }
      if (TAIL && p.m > 1) {
        // A NaN in V at a position that only some rows may see must not reach the others as 0 x NaN: such blocks are
        // taken out, and the rows that see them set to NaN.  (Lane (c16, g) holds V of column block c16 / (512 / D) and
        // outputs of block g D / 128.)
        unsigned nan = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) nan |= ((r.vs[j >> 2] >> (8 * (j & 3))) & 0xffu) == 0xffu ? 1u << j : 0u;
        if (__any(nan != 0)) {
          const unsigned long long mine = D == 128 ? 0x000f000f000f000full << (4 * g) : 0x00ff00ff00ff00ffull << (8 * (g >> 1));
          for (int at = 0; at < p.m; ++at) {
            const int last = n - p.m + at;
            unsigned upto = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) upto |= key0 + 16 * (j >> 2) + (j & 3) <= last ? 1u << j : 0u;
            const bool hit = (__ballot((nan & upto) != 0) & mine) != 0;
#pragma unroll
            for (int t = 0; t < NT; ++t)
              if (hit && pos[t] == last)
#pragma unroll
                for (int i = 0; i < DT; ++i) o[t][i] = f4_f32x4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((nan >> j) & 1) drop_key(r, j);
        }
      }
      uint4 pb[NT], pl[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = s[t][j >> 2][j & 3];
        if constexpr (TAIL) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (key0 + 16 * (j >> 2) + (j & 3) > pos[t]) x[j] = -__builtin_inff();
        }
        const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * p.scale_log2;
        if (__any(top > mx[t] + kFp4Slack)) {
          float m2 = fmaxf(top, __shfl_xor(top, 16, 64));
          m2 = fmaxf(m2, __shfl_xor(m2, 32, 64));
          m2 = fmaxf(m2, mx[t]);
          const float f = fp4_exp2(mx[t] - m2);
          mx[t] = m2;
          l[t] *= f;
#pragma unroll
          for (int i = 0; i < DT; ++i) o[t][i] *= f;
        }
        float pr[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) pr[j] = fp4_exp2(__builtin_fmaf(x[j], p.scale_log2, -mx[t]));
        unsigned hi[4], lo[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          hi[y] = fp4_pack_bf16(pr[2 * y], pr[2 * y + 1]);
          const float d0 = pr[2 * y] - __uint_as_float(hi[y] << 16), d1 = pr[2 * y + 1] - __uint_as_float(hi[y] & 0xffff0000u);
          lo[y] = fp4_pack_bf16(d0, d1);
          if constexpr (HALF) hi[y] = c16 < 8 ? hi[y] : lo[y];
        }
        pb[t] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        pl[t] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      weighted_sum(r, pb, pl);
    };

    if (t0 < full_end) {
      for (;;) {
        bool done = false;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          load(t0 + 4, pg, ring[1 - x], t0 + 4 < tile_end);
          pages_of(t0 + 8, pg);
          if (younger) {
            if (x == 0) __builtin_amdgcn_s_setprio(1);
            else __builtin_amdgcn_s_setprio(0);
          }
          process(std::false_type{}, ring[x], t0);
          t0 += 4;
          if (t0 >= full_end) {
            if (x == 0) ring[0] = ring[1];
            done = true;
            break;
          }
        }
        if (done) break;
      }
    }
    while (t0 < tile_end) {  // (the first of them is loaded already; more than one only where rows end in several tiles)
      process(std::true_type{}, ring[0], t0);
      t0 += 4;
      if (t0 < tile_end) {
        pages_of(t0, pg);
        load(t0, pg, ring[0], true);
      }
    }

    // ---- the piece is done; the next one's loads go out before it is written ----
    const int b_done = b, n_done = n;
    const bool whole_done = whole;
    bool more = left > kFp4Begin;
    if (more) {
      do ++b;
      while (b < p.batch && fp4_len_of(p, plan, b) <= 0);
      more = b < p.batch;
    }
    if (more) {
      off = -kFp4Begin;
      start();
    }

    // ---- join the waves ----
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float sum = l[t][0];
      if constexpr (HALF) {
        sum += fp4_other8(sum);
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int y = 0; y < 4; ++y) o[t][i][y] += fp4_other8(o[t][i][y]);
      }
      const int r = HALF ? c16 : 16 * t + c16;
      if (r < ROWS) {
        if (g == 0) sm_ml[wave][r] = f4_f32x2{mx[t], sum};
        // O^T tile i: row 4 g + y of it is column (4 g + y) D/16 + i
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int i = 0; i < DT; i += 4)
            *reinterpret_cast<f4_f32x4*>(&sm_o[wave][r][(4 * g + y) * DT + i]) = f4_f32x4{o[t][i][y], o[t][i + 1][y], o[t][i + 2][y], o[t][i + 3][y]};
      }
    }
    __syncthreads();
    for (int u = tid; u < R * (D / 4); u += 256) {
      const int r = u / (D / 4), d = 4 * (u % (D / 4));
      const int j = (row0 + r) / p.G, hd = h * p.G + (row0 + r - j * p.G);
      // The row's common maximum and every wave's factor.  A wave without tiles holds (lowest, 0): factor 0 or, if no wave
      // saw a key, 1 on zeros.
      f4_f32x2 ml[4];
      float top = kFp4MinusBig, ls = 0.f;
#pragma unroll
      for (int wv = 0; wv < 4; ++wv) {
        ml[wv] = sm_ml[wv][r];
        top = fmaxf(top, ml[wv][0]);
      }
      f4_f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int wv = 0; wv < 4; ++wv) {
        const float f = fp4_exp2(ml[wv][0] - top);
        ls += ml[wv][1] * f;
        x += *reinterpret_cast<const f4_f32x4*>(&sm_o[wv][r][d]) * f;
      }
      if (n_done - p.m + j < 0) continue;  // the sequence is shorter than the step's rows: no such position
      if (whole_done) {
        const float inv = 1.f / ls;
        const int64_t at = ((int64_t)b_done * p.m + j) * p.out_stride_t + hd * p.out_stride_h + d;
#pragma unroll
        for (int y = 0; y < 4; ++y) fp4_store_out(p.out, at + y, x[y] * inv, p.out_f32 != 0, BF16);
      } else {
        const int64_t slot = ((int64_t)(w + b_done) * p.m + j) * p.H + hd;
        *reinterpret_cast<f4_f32x4*>(p.partial_o + slot * D + d) = x;
        if (d == 0) *reinterpret_cast<f4_f32x2*>(p.partial_ml + 2 * slot) = f4_f32x2{top, ls};
      }
    }
    if (!more) return;
    __syncthreads();  // (the next piece's sums go to the same LDS)
  }
}

// Joins the pieces of output rows, D / 4 lanes along a row, PIECES of its pieces at a time.
template <int D, bool BF16, int PIECES>
__global__ __launch_bounds__(D / 4 * PIECES < 256 ? 256 : D / 4 * PIECES) void fp4_join_kernel(const Fp4DecodeParams p) {
  constexpr int LANES = D / 4, THREADS = LANES * PIECES < 256 ? 256 : LANES * PIECES, ROWS = THREADS / (LANES * PIECES);
  __shared__ float sm_ml[ROWS][PIECES][2];
  __shared__ float sm_o[ROWS][PIECES][D];
  fp4_ask_for_arguments(p);
  const int tid = threadIdx.x;
  const int b = blockIdx.y;
  const int n = fp4_sload(p.seq_lens + b), first = fp4_sload(p.pieces + 2 * b), pieces = fp4_sload(p.pieces + 2 * b + 1);
  if (n <= 0 || pieces <= 1) return;  // (padding: nobody has written its pieces)
  const int row = tid / (LANES * PIECES), part = tid / LANES % PIECES, c = tid % LANES;
  const int rh = (int)blockIdx.x * ROWS + row;  // row of the request x head
  const int j = rh / p.H, hd = rh - j * p.H;
  const bool there = j < p.m && n - p.m + j >= 0;
  float top = kFp4MinusBig, sum = 0.f;
  f4_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (there) {
#pragma unroll 4
    for (int y = part; y < pieces; y += PIECES) {
      const int64_t slot = ((int64_t)(first + y + b) * p.m + j) * p.H + hd;
      const f4_f32x2 ml = *reinterpret_cast<const f4_f32x2*>(p.partial_ml + 2 * slot);
      const f4_f32x4 o1 = *reinterpret_cast<const f4_f32x4*>(p.partial_o + slot * D + 4 * c);
      const float m2 = fmaxf(top, ml[0]);
      const float fa = fp4_exp2(top - m2), fb = fp4_exp2(ml[0] - m2);
      acc = acc * fa + o1 * fb;
      sum = sum * fa + ml[1] * fb;
      top = m2;
    }
  }
  if constexpr (PIECES > 1) {
    if (c == 0) sm_ml[row][part][0] = top, sm_ml[row][part][1] = sum;
    *reinterpret_cast<f4_f32x4*>(&sm_o[row][part][4 * c]) = acc;
    __syncthreads();
    if (part != 0) return;
    float tm = kFp4MinusBig, tl = 0.f;
    f4_f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int y = 0; y < PIECES; ++y) tm = fmaxf(tm, sm_ml[row][y][0]);
#pragma unroll
    for (int y = 0; y < PIECES; ++y) {
      const float f = fp4_exp2(sm_ml[row][y][0] - tm);
      tl += sm_ml[row][y][1] * f;
      x += *reinterpret_cast<const f4_f32x4*>(&sm_o[row][y][4 * c]) * f;
    }
    acc = x;
    sum = tl;
  }
  if (there) {
    const int64_t at = ((int64_t)b * p.m + j) * p.out_stride_t + hd * p.out_stride_h + 4 * c;
#pragma unroll
    for (int y = 0; y < 4; ++y) fp4_store_out(p.out, at + y, acc[y] / sum, p.out_f32 != 0, BF16);
  }
}

// Spans per unit: as many as there are workgroups resident together on the chip.
static int fp4_row_groups(int64_t rows) { return (int)((rows + 31) / 32); }
static int fp4_spans(int64_t rows, int kv_heads, int cus) {
  return imax(1, cus * kFp4WgsPerCu / (kv_heads * fp4_row_groups(rows)));
}

static int fp4_cus(int* out) {
  static std::atomic<int> cache[64];
  int dev = 0;
  TMX_CHECK_HIP(hipGetDevice(&dev));
  int cus = (dev >= 0 && dev < 64) ? cache[dev].load(std::memory_order_relaxed) : 0;
  if (cus == 0) {
    TMX_CHECK_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    if (dev >= 0 && dev < 64) cache[dev].store(cus, std::memory_order_relaxed);
  }
  *out = cus;
  return TMX_OK;
}

template <int D, bool BF16>
static void fp4_launch(const Fp4DecodeParams& p, hipStream_t s) {
  const unsigned grid = ((unsigned)p.spans * (unsigned)p.units + 7) / 8 * 8;
  const int R = p.m * p.G;
  if (R <= 8) fp4_decode_kernel<D, BF16, 1, true><<<grid, 256, 0, s>>>(p);
  else if (R <= 16) fp4_decode_kernel<D, BF16, 1, false><<<grid, 256, 0, s>>>(p);
  else fp4_decode_kernel<D, BF16, 2, false><<<grid, 256, 0, s>>>(p);
  // Pieces of a row that are joined side by side, by how many an average request can have (four more of each are in
  // flight), with 2 / 8 / 32 of them: 16 x 4 drafted rows of up to 5 pieces 4.7 / 5.2 / 16.7 us, 8 requests of 64 pieces 6.1 /
  // 4.6 / 4.6, one of 512 pieces 22.9 / 8.2 / 6.0.  (One request with nearly all pieces beside many short ones is joined as
  // the average would be: the whole call for 131072 tokens of one K/V head takes 16.3 us, beside 64 requests of 64 32.2.)
  const unsigned rows = (unsigned)(p.m * p.H);
  const int pieces = p.spans / p.batch;
  auto join = [&](auto pieces_) {
    constexpr int P = decltype(pieces_)::value;
    constexpr unsigned threads = D / 4 * P < 256 ? 256 : D / 4 * P, per = threads / (D / 4 * P);
    fp4_join_kernel<D, BF16, P><<<dim3((rows + per - 1) / per, (unsigned)p.batch), threads, 0, s>>>(p);
  };
  if (pieces < 8) join(std::integral_constant<int, 2>{});
  else if (pieces <= 64) join(std::integral_constant<int, 8>{});
  else join(std::integral_constant<int, 32>{});
}

}  // namespace tmx

extern "C" int64_t tmx_decode_fp4_workspace_rows(int batch, int rows_per_request, int num_heads, int num_kv_heads, int head_dim, int num_cus) {
  using namespace tmx;
  if (batch <= 0 || rows_per_request <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0) return 0;
  if (num_cus <= 0 && fp4_cus(&num_cus) != TMX_OK) return -1;
  const int64_t R = (int64_t)rows_per_request * (num_heads / num_kv_heads);
  return (fp4_spans(R > 64 ? 64 : R, num_kv_heads, num_cus) + (int64_t)batch) * rows_per_request * num_heads + batch;
}

extern "C" int tmx_decode_attention_fp4(const tmx_decode_fp4_args_t* a, void* stream) {
  using namespace tmx;
  TMX_CHECK_ARG(a != nullptr, "tmx_decode_attention_fp4: args is NULL");
  TMX_CHECK_ARG(a->struct_size == sizeof(tmx_decode_fp4_args_t), "tmx_decode_attention_fp4: struct_size %u != %zu (ABI mismatch)",
                a->struct_size, sizeof(tmx_decode_fp4_args_t));
  TMX_CHECK_SUPPORTED(a->io_dtype == TMX_BF16 || a->io_dtype == TMX_F16,
                      "tmx_decode_attention_fp4: q dtype %d not supported (bf16 and fp16 are)", a->io_dtype);
  TMX_CHECK_SUPPORTED(a->out_dtype == a->io_dtype || a->out_dtype == TMX_F32,
                      "tmx_decode_attention_fp4: out dtype %d must equal the input dtype or be fp32", a->out_dtype);
  TMX_CHECK_ARG(a->num_heads > 0 && a->num_kv_heads > 0 && a->num_heads % a->num_kv_heads == 0,
                "tmx_decode_attention_fp4: num_heads %d must be a positive multiple of num_kv_heads %d", a->num_heads,
                a->num_kv_heads);
  TMX_CHECK_SUPPORTED(a->head_dim == 64 || a->head_dim == 128, "tmx_decode_attention_fp4: head_dim %d not covered (64 and 128 are)",
                      a->head_dim);
  TMX_CHECK_ARG(a->batch >= 0 && a->rows_per_request > 0, "tmx_decode_attention_fp4: bad sizes");
  const int64_t R = (int64_t)a->rows_per_request * (a->num_heads / a->num_kv_heads);
  TMX_CHECK_SUPPORTED(R <= 64, "tmx_decode_attention_fp4: %lld rows per K/V head (rows_per_request x query heads per K/V head): at "
                      "most 64 (longer steps: tmx_gather_dequant_kv_fp4 and tmx_attention)", (long long)R);
  TMX_CHECK_SUPPORTED(a->batch <= 65535, "tmx_decode_attention_fp4: more than 65535 requests");
  TMX_CHECK_ARG(a->scale > 0.f && a->scale < 3.0e38f, "tmx_decode_attention_fp4: scale %g must be positive and finite",
                (double)a->scale);
  TMX_CHECK_SUPPORTED(a->page_size >= 16 && a->page_size <= (1 << 20) && (a->page_size & (a->page_size - 1)) == 0,
                      "tmx_decode_attention_fp4: page_size %d not supported (powers of two from 16 to 2^20 are)", a->page_size);
  TMX_CHECK_SUPPORTED(a->num_kv_heads <= 1024 && fp4_page_bytes(a->num_kv_heads, a->page_size, a->head_dim) <= 0x7fffffff,
                      "tmx_decode_attention_fp4: more than 1024 K/V heads, or a page of 2^31 bytes or more");
  if (a->batch == 0) return TMX_OK;
  TMX_CHECK_ARG(a->q && a->out && a->k && a->v && a->seq_lens && a->block_table, "tmx_decode_attention_fp4: NULL tensor");
  TMX_CHECK_ARG(a->num_pages > 0 && a->num_pages <= 0x7fffffff && a->max_blocks >= 0 && a->block_table_stride >= 0,
                "tmx_decode_attention_fp4: bad sizes of the cache or the block table");
  TMX_CHECK_ARG(a->kv_stride_page >= fp4_page_bytes(a->num_kv_heads, a->page_size, a->head_dim) && a->kv_stride_page % 16 == 0,
                "tmx_decode_attention_fp4: the page stride %lld must be a multiple of 16 bytes and hold a page of %lld",
                (long long)a->kv_stride_page, (long long)fp4_page_bytes(a->num_kv_heads, a->page_size, a->head_dim));
  TMX_CHECK_ARG(((uintptr_t)a->q % 16 == 0) && ((uintptr_t)a->k % 16 == 0) && ((uintptr_t)a->v % 16 == 0) &&
                    ((uintptr_t)a->out % 4 == 0),
                "tmx_decode_attention_fp4: q / k / v must be 16-byte aligned, out 4-byte");
  TMX_CHECK_ARG(a->q_stride_t >= 0 && a->q_stride_h >= 0 && a->q_stride_t % 8 == 0 && a->q_stride_h % 8 == 0 &&
                    a->out_stride_t >= 0 && a->out_stride_h >= 0,
                "tmx_decode_attention_fp4: strides must not be negative, those of q multiples of 8 elements");
  // tiles of a step are counted in 32 bits
  const int64_t len_cap = (int64_t)a->max_blocks * a->page_size + a->rows_per_request;
  TMX_CHECK_SUPPORTED(len_cap <= 0x7ffff000 && (len_cap / kBlockN + 2 + kFp4Begin) * a->batch <= 0x7fff0000,
                      "tmx_decode_attention_fp4: the block table has room for more than 2^31 tiles of 32 keys");
  int cus = 0;
  {
    const int rc = fp4_cus(&cus);
    if (rc != TMX_OK) return rc;
  }
  Fp4DecodeParams p{};
  p.spans = fp4_spans(R, a->num_kv_heads, cus);
  p.row_groups = fp4_row_groups(R);
  p.units = a->num_kv_heads * p.row_groups;
  const int64_t rows = (p.spans + (int64_t)a->batch) * a->rows_per_request * a->num_heads;
  TMX_CHECK_ARG(a->partial_o != nullptr && a->partial_ml != nullptr && ((uintptr_t)a->partial_o % 16 == 0),
                "tmx_decode_attention_fp4: the work area is missing (tmx_decode_fp4_workspace_rows)");
  TMX_CHECK_ARG(a->workspace_rows >= rows + a->batch,
                "tmx_decode_attention_fp4: the work area holds %lld rows, this batch size needs %lld (tmx_decode_fp4_workspace_rows)",
                (long long)a->workspace_rows, (long long)rows + a->batch);
  p.q = a->q;
  p.out = a->out;
  p.k = (const uint8_t*)a->k;
  p.v = (const uint8_t*)a->v;
  p.stride_page = a->kv_stride_page;
  p.num_pages = (int)a->num_pages;
  // (a table without columns: an entry of the lengths is read in its place and not used)
  p.block_table = a->max_blocks > 0 ? a->block_table : a->seq_lens;
  p.block_table_stride = a->max_blocks > 0 ? a->block_table_stride : 0;
  p.max_blocks = a->max_blocks;
  p.page_shift = __builtin_ctz(a->page_size);
  p.seq_lens = a->seq_lens;
  p.len_cap = (int)len_cap;
  p.batch = a->batch;
  p.m = a->rows_per_request;
  p.H = a->num_heads;
  p.Hkv = a->num_kv_heads;
  p.G = a->num_heads / a->num_kv_heads;
  p.q_stride_t = a->q_stride_t;
  p.q_stride_h = a->q_stride_h;
  p.out_stride_t = a->out_stride_t;
  p.out_stride_h = a->out_stride_h;
  p.out_f32 = a->out_dtype == TMX_F32;
  p.scale_log2 = a->scale * kLog2e;
  p.partial_o = a->partial_o;
  p.partial_ml = a->partial_ml;
  p.pieces = reinterpret_cast<int*>(a->partial_ml + 2 * rows);
  hipStream_t s = (hipStream_t)stream;
  const bool bf16 = a->io_dtype == TMX_BF16;
  if (a->head_dim == 128) {
    if (bf16) fp4_launch<128, true>(p, s);
    else fp4_launch<128, false>(p, s);
  } else {
    if (bf16) fp4_launch<64, true>(p, s);
    else fp4_launch<64, false>(p, s);
  }
  TMX_CHECK_HIP(hipGetLastError());
  return TMX_OK;
}
