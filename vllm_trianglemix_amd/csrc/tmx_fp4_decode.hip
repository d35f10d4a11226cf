// Attention of a step's query rows against a 4-bit (MXFP4) paged K/V cache, for gfx950 (MI355X): one row per request
// (decode) or the last few positions of each (drafted tokens checked in one step).  Such a step reads all of its K/V
// once and multiplies little, so it is bound by the bytes of the cache; the 4-bit codes become bf16 in registers, which is
// exact (a code has one fraction bit, the scale is a power of two), and both products run on the matrix cores.
//
//   workgroup = 4 waves = one piece of a request's keys x one K/V head; the waves take the piece's 32-key tiles in turn
//   and meet only at the end.  Rows = rows_per_request x (query heads per K/V head), all of them columns of the same
//   products, so a head's K/V are read once whatever the group size.
//   Scores S^T = K Q^T (v_mfma_f32_16x16x32_bf16, 2 x D / 32 of them): lane (m = lane % 16, g = lane / 16) holds key row m
//   and columns [g D/4, (g + 1) D/4) of it, one 16-byte load and one scale for D = 128; the head dimension may be summed
//   in any order as long as Q^T is laid out alike.  Row m of the first / second product is key 8 (m / 4) + (m % 4), + 4
//   for the second: a lane's 8 scores are then the keys 8 g .. 8 g + 7, exactly the ones it has to hold as operand of
//   the second product, and the probabilities never leave their lane.
//   Output O^T = V^T P^T: lane (m, g) needs columns [m D/16, (m + 1) D/16) of keys 8 g .. + 7.  The cache keeps V in that
//   order (tmx_fp4.h): one or two 16-byte loads, 32 conversions and 32 byte permutes turn them into operands.  No LDS.
//   Probabilities are held as two bf16 terms (16 significant bits; one term alone would cost as much accuracy as the
//   rounding of the output).  Up to 8 rows, columns 8..15 repeat the rows and carry the second term: no extra product.
//   fp16 queries are split into two bf16 terms as well (exact: 11 bits in 8 + 8).
//   The running maximum is raised only when a score exceeds it by more than 2^kSlack (factors stay below 2^8 in fp32).
//   A piece's result goes to the output row, or to partial results that a second launch joins.
#include <atomic>
#include <type_traits>

#include "tmx_common.h"
#include "tmx_decode_plan.h"
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
  int64_t q_stride_t, q_stride_h, out_stride_t, out_stride_h;  // elements
  int out_f32;
  float scale_log2;
  float* partial_o;   // [piece][row of the request][head][D]
  float* partial_ml;  // [piece][row of the request][head][2]
  int plan_slots;
};

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

// Workgroups resident per CU by the registers that the accumulators of `rows` rows leave.
constexpr int fp4_wgs_per_cu(int head_dim, int rows) { return rows <= 16 ? (head_dim == 128 ? 3 : 4) : (rows <= 32 ? 2 : 1); }

// NT column tiles of 16 rows; HALF: one tile, at most 8 rows, columns 8..15 carry the second terms
template <int D, bool BF16, int NT, bool HALF>
__global__ __launch_bounds__(256, fp4_wgs_per_cu(D, 16 * NT)) void fp4_decode_kernel(const Fp4DecodeParams p) {
  static_assert(!HALF || NT == 1, "the half form has one tile");
  constexpr int KS = D / 32;        // k-steps of the first product
  constexpr int DT = D / 16;        // row tiles of the second
  constexpr int VL = D / 64;        // 16-byte V loads per lane and tile
  constexpr bool Q2 = !BF16 && !HALF;  // a second query term in registers of its own
  constexpr int ROWS = HALF ? 8 : 16 * NT;
  constexpr int COPIES = NT == 1 ? 4 : 1;  // LDS images of the waves' sums (more than 16 rows: one, added to in turn)
  __shared__ float sm_o[COPIES][ROWS][D + 2];  // (+ 2: the 16 rows a wave writes at once start in different banks)
  __shared__ float sm_ml[4][ROWS][2];
  __shared__ int plan_sm[4 + 2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int w = (int)blockIdx.x / p.Hkv;
  const int h = (int)blockIdx.x - w * p.Hkv;
  const DcPiece dp = dc_find_piece<256>(p.seq_lens, p.batch, p.Hkv, p.plan_slots, w, plan_sm, tid);
  if (dp.b < 0) return;  // fewer pieces in this step than the grid provides for
  const int b = __builtin_amdgcn_readfirstlane(dp.b);
  const int n = __builtin_amdgcn_readfirstlane(dp.n);
  const int tile0 = __builtin_amdgcn_readfirstlane(dp.tile0);
  const int tile_end = tile0 + __builtin_amdgcn_readfirstlane(dp.ntiles);
  const int R = p.m * p.G;

  // ---- query rows: operand Q^T, lane column c16 = row, k-step i covers columns g D/4 + 8 i .. + 7.  Row r is position
  // n - m + r / G, head h G + r % G. ----
  uint4 qf[NT][KS], ql[Q2 ? NT : 1][KS];
  int pos[NT];  // the position of this lane's row
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = HALF ? (c16 & 7) : 16 * t + c16;
    const bool row = r < R;
    const int j = row ? r / p.G : 0, hd = h * p.G + (row ? r - j * p.G : 0);
    pos[t] = n - p.m + j;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + ((int64_t)b * p.m + j) * p.q_stride_t + hd * p.q_stride_h;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      uint4 x = *reinterpret_cast<const uint4*>(src + g * (D / 4) + 8 * i);
      if (!row) x = make_uint4(0, 0, 0, 0);
      if constexpr (BF16) {
        qf[t][i] = x;
      } else {
        const unsigned xs[4] = {x.x, x.y, x.z, x.w};
        unsigned hi[4], lo[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const fp4_f16x2 f = __builtin_bit_cast(fp4_f16x2, xs[y]);
          hi[y] = fp4_pack_bf16((float)f[0], (float)f[1]);
          // (an infinity has no second term)
          const float h0 = __uint_as_float(hi[y] << 16), h1 = __uint_as_float(hi[y] & 0xffff0000u);
          const float d0 = (float)f[0] - h0, d1 = (float)f[1] - h1;
          lo[y] = fp4_pack_bf16(__builtin_isinf(h0) ? 0.f : d0, __builtin_isinf(h1) ? 0.f : d1);
        }
        const uint4 a = make_uint4(hi[0], hi[1], hi[2], hi[3]), c = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if constexpr (HALF) qf[t][i] = c16 < 8 ? a : c;
        else qf[t][i] = a, ql[Q2 ? t : 0][i] = c;
      }
    }
  }

  // ---- addresses.  A tile's two 16-key halves may lie on two pages; K rows of a lane belong to half m / 8, its V keys to
  // half g / 2. ----
  const int ps = 1 << p.page_shift;
  const int64_t codes = fp4_code_bytes(p.Hkv, ps, D);
  const int64_t head_codes = (int64_t)h * ps * (D / 2);
  const int64_t head_scales = codes + (int64_t)h * ps * (D / 32);
  const int32_t* const bt = p.block_table + b * p.block_table_stride;
  const bool khalf = (c16 & 8) != 0, vhalf = (g & 2) != 0;
  const int k_lane = (8 * ((c16 >> 2) & 1) + (c16 & 3)) * (D / 2) + g * (D / 8);
  const int v_lane = (g & 1) * (8 * (D / 2)) + c16 * 16;
  const int ks_lane = (D == 128 ? g : g >> 1) * ps + 8 * ((c16 >> 2) & 1);
  const int vs_lane = (D == 128 ? c16 >> 2 : c16 >> 3) * ps + 8 * (g & 1);

  struct Raw {
    fp4_u32x4 k[2];  // D = 64: the first two words
    fp4_u32x4 v[VL];
    fp4_u32x2 ks, vs;
    unsigned bad;  // bit x: half x has no page
  };
  auto load = [&](int tile, Raw& r) {
    const int key0 = tile * kBlockN;
    const int blk0 = key0 >> p.page_shift;
    const int key1 = key0 + 16 < n ? key0 + 16 : key0;  // a half past the end reads the first one again
    const int blk1 = key1 >> p.page_shift;
    int e0 = blk0 < p.max_blocks ? fp4_sload(bt + blk0) : -1;
    int e1 = blk1 < p.max_blocks ? fp4_sload(bt + blk1) : -1;
    r.bad = ((unsigned)e0 >= (unsigned)p.num_pages ? 1u : 0u) | ((unsigned)e1 >= (unsigned)p.num_pages ? 2u : 0u);
    if (r.bad & 1) e0 = 0;
    if (r.bad & 2) e1 = 0;
    const int at0 = key0 & (ps - 1), at1 = key1 & (ps - 1);
    const int64_t o0 = e0 * p.stride_page, o1 = e1 * p.stride_page;
    const int64_t c0 = o0 + head_codes + at0 * (D / 2), c1 = o1 + head_codes + at1 * (D / 2);
    const int64_t s0 = o0 + head_scales + at0, s1 = o1 + head_scales + at1;
    const uint8_t* kp = p.k + (khalf ? c1 : c0) + k_lane;
    const uint8_t* vp = p.v + (vhalf ? c1 : c0) + v_lane;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (D == 128) {
        r.k[t] = __builtin_nontemporal_load(reinterpret_cast<const fp4_u32x4*>(kp + t * 4 * (D / 2)));
      } else {
        const fp4_u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const fp4_u32x2*>(kp + t * 4 * (D / 2)));
        r.k[t] = fp4_u32x4{x[0], x[1], 0, 0};
      }
    }
#pragma unroll
    for (int x = 0; x < VL; ++x) r.v[x] = __builtin_nontemporal_load(reinterpret_cast<const fp4_u32x4*>(vp + x * 256));
    r.ks = *reinterpret_cast<const fp4_u32x2*>(p.k + (khalf ? s1 : s0) + ks_lane);
    r.vs = *reinterpret_cast<const fp4_u32x2*>(p.v + (vhalf ? s1 : s0) + vs_lane);
  };

  f4_f32x4 o[NT][DT];
  float mx[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    mx[t] = kFp4MinusBig;
    l[t] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[t][i] = f4_f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto scale_of = [](unsigned word, int byte) -> float { return __uint_as_float(((word >> (8 * byte)) & 0xffu) << 23); };

  // ---- O^T += V^T P^T with the probabilities in pb (and their second terms in pl unless HALF), one byte of every
  // key's codes -- a pair of columns, two row tiles -- at a time ----
  auto weighted_sum = [&](const Raw& r, const uint4 (&pb)[NT], const uint4 (&pl)[NT]) {
    float sc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sc[j] = scale_of(r.vs[j >> 2], j & 3);
    auto pair = [&](auto at) {
      constexpr int B = decltype(at)::value;
      unsigned c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (D == 128) c[j] = fp4_bf16<B>(r.v[j >> 2][j & 3], sc[j]);
        else c[j] = (j & 1) ? fp4_bf16<2 + (B & 1)>(r.v[0][j >> 1], sc[j]) : fp4_bf16<B & 1>(r.v[0][j >> 1], sc[j]);
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
    if constexpr (D == 128) r.v[j >> 2][j & 3] = 0;
    else r.v[0][j >> 1] &= (j & 1) ? 0x0000ffffu : 0xffff0000u;
    r.vs[j >> 2] &= ~(0xffu << (8 * (j & 3)));
  };

  auto process = [&](Raw& r, int tile) {
    const int key0 = tile * kBlockN;
    if (r.bad) {  // keys without a page count as NaN
      if ((r.bad >> (khalf ? 1 : 0)) & 1) r.ks = fp4_u32x2{~0u, ~0u};
      if ((r.bad >> (vhalf ? 1 : 0)) & 1) r.vs = fp4_u32x2{~0u, ~0u};
    }
    // scores
    f4_f32x4 s[NT][2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const float sc = __uint_as_float(((r.ks[tt] >> (8 * (c16 & 3))) & 0xffu) << 23);
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t][tt] = f4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const unsigned word = r.k[tt][i];
        const uint4 a = make_uint4(fp4_bf16<0>(word, sc), fp4_bf16<1>(word, sc), fp4_bf16<2>(word, sc), fp4_bf16<3>(word, sc));
        const f4_bf16x8 av = __builtin_bit_cast(f4_bf16x8, a);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          s[t][tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, __builtin_bit_cast(f4_bf16x8, qf[t][i]), s[t][tt], 0, 0, 0);
          if constexpr (Q2) s[t][tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, __builtin_bit_cast(f4_bf16x8, ql[t][i]), s[t][tt], 0, 0, 0);
        }
      }
    }
    // the tile may hold keys past a row's position (or past the sequence: their V must not enter even as 0 x NaN)
    const bool tail = key0 + kBlockN > n - p.m + 1;
    if (key0 + kBlockN > n) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (key0 + 8 * g + j >= n) drop_key(r, j);
    }
    if (p.m > 1 && tail) {
      // A NaN in V at a position that only some rows may see must not reach the others as 0 x NaN: such blocks are taken
      // out, and the rows that see them set to NaN.  (Lane (c16, g) holds V of column block c16 / (512 / D) and outputs of
      // block g D / 128.)
      unsigned nan = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) nan |= ((r.vs[j >> 2] >> (8 * (j & 3))) & 0xffu) == 0xffu ? 1u << j : 0u;
      if (__any(nan != 0)) {
        const unsigned long long mine = D == 128 ? 0x000f000f000f000full << (4 * g) : 0x00ff00ff00ff00ffull << (8 * (g >> 1));
        for (int at = 0; at < p.m; ++at) {
          const int last = n - p.m + at, seen = last - key0 - 8 * g;  // the lane's keys 0 .. seen
          const unsigned upto = seen < 0 ? 0u : (seen >= 7 ? 0xffu : (2u << seen) - 1u);
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
      for (int j = 0; j < 8; ++j) {
        float v = s[t][j >> 2][j & 3];
        if constexpr (HALF && !BF16) v += fp4_other8(v);  // the query's two terms
        x[j] = v;
      }
      if (tail) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (key0 + 8 * g + j > pos[t]) x[j] = -__builtin_inff();
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
      l[t] += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
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

  // ---- the wave's tiles, the next one's loads in flight while one is computed ----
  {
    int t = tile0 + wave;
    Raw a, c;
    if (t < tile_end) {
      load(t, a);
      for (;;) {
        if (t + 4 < tile_end) load(t + 4, c);
        process(a, t);
        t += 4;
        if (t >= tile_end) break;
        if (t + 4 < tile_end) load(t + 4, a);
        process(c, t);
        t += 4;
        if (t >= tile_end) break;
      }
    }
  }

  // ---- join the waves ----
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);
    l[t] += __shfl_xor(l[t], 32, 64);
    if constexpr (HALF) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[t][i][y] += fp4_other8(o[t][i][y]);
    }
    const int r = HALF ? c16 : 16 * t + c16;
    if (g == 0 && r < ROWS) {
      sm_ml[wave][r][0] = mx[t];
      sm_ml[wave][r][1] = l[t];
    }
  }
  __syncthreads();
  // Row r's common maximum, and this wave's factor.  A wave without tiles holds (lowest, 0): factor 0 or, if no wave saw
  // a key, 1 on zeros.
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = HALF ? (c16 & 7) : 16 * t + c16;
    const float top = fmaxf(fmaxf(sm_ml[0][r][0], sm_ml[1][r][0]), fmaxf(sm_ml[2][r][0], sm_ml[3][r][0]));
    const float f = fp4_exp2(mx[t] - top);
#pragma unroll
    for (int i = 0; i < DT; ++i) o[t][i] *= f;
  }
  // O^T tile i: row 4 g + y of it is column (4 g + y) D/16 + i
  if constexpr (COPIES == 4) {
    const int r = c16;
    if (r < ROWS) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y) sm_o[wave][r][(4 * g + y) * DT + i] = o[0][i][y];
    }
    __syncthreads();
  } else {
    for (int turn = 0; turn < 4; ++turn) {
      if (wave == turn) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              float* d = &sm_o[0][16 * t + c16][(4 * g + y) * DT + i];
              *d = turn == 0 ? o[t][i][y] : *d + o[t][i][y];
            }
      }
      __syncthreads();
    }
  }
  for (int u = tid; u < R * D; u += 256) {
    const int r = u / D, d = u - r * D;
    const int j = r / p.G, hd = h * p.G + (r - j * p.G);
    if (n - p.m + j < 0) continue;  // the sequence is shorter than the step's rows: no such position
    float top = kFp4MinusBig, sum = 0.f, x = 0.f;
#pragma unroll
    for (int wv = 0; wv < 4; ++wv) top = fmaxf(top, sm_ml[wv][r][0]);
#pragma unroll
    for (int wv = 0; wv < 4; ++wv) sum += sm_ml[wv][r][1] * fp4_exp2(sm_ml[wv][r][0] - top);
#pragma unroll
    for (int y = 0; y < COPIES; ++y) x += sm_o[y][r][d];
    if (dp.pieces == 1) {
      fp4_store_out(p.out, ((int64_t)b * p.m + j) * p.out_stride_t + hd * p.out_stride_h + d, x / sum, p.out_f32 != 0, BF16);
    } else {
      const int64_t slot = ((int64_t)w * p.m + j) * p.H + hd;
      p.partial_o[slot * D + d] = x;
      if (d == 0) {
        p.partial_ml[2 * slot] = top;
        p.partial_ml[2 * slot + 1] = sum;
      }
    }
  }
}

// Joins the pieces of one output row: one workgroup per (request, row, head), D / 4 lanes along the columns, 1024 / D
// pieces at a time.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void fp4_join_kernel(const Fp4DecodeParams p) {
  constexpr int LANES = D / 4, AT_ONCE = 256 / LANES;
  __shared__ int sm[4 + 2];
  __shared__ float sm_m[AT_ONCE], sm_l[AT_ONCE];
  __shared__ float sm_o[AT_ONCE][D];
  const int tid = threadIdx.x;
  const int b = blockIdx.y, j = (int)blockIdx.x / p.H, hd = (int)blockIdx.x - j * p.H;
  const int n = p.seq_lens[b];
  if (n <= 0 || n - p.m + j < 0) return;
  // first piece of request b, and how many it has
  int before = 0, all = 0;
  for (int x = tid; x < p.batch; x += 256) all += dc_tiles_of(p.seq_lens[x]);
  const int P = dc_piece_len(dc_block_sum<256>(all, sm, tid), p.Hkv, p.plan_slots);
  const int pieces = (dc_tiles_of(n) + P - 1) / P;
  if (pieces <= 1) return;
  for (int x = tid; x < b; x += 256) before += (dc_tiles_of(p.seq_lens[x]) + P - 1) / P;
  const int first = dc_block_sum<256>(before, sm, tid);
  const int part = tid / LANES, c = tid - part * LANES;
  float top = kFp4MinusBig, sum = 0.f;
  f4_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int y = part; y < pieces; y += AT_ONCE) {
    const int64_t slot = ((int64_t)(first + y) * p.m + j) * p.H + hd;
    const float m1 = p.partial_ml[2 * slot], l1 = p.partial_ml[2 * slot + 1];
    const f4_f32x4 o1 = *reinterpret_cast<const f4_f32x4*>(p.partial_o + slot * D + 4 * c);
    const float m2 = fmaxf(top, m1);
    const float fa = fp4_exp2(top - m2), fb = fp4_exp2(m1 - m2);
    acc = acc * fa + o1 * fb;
    sum = sum * fa + l1 * fb;
    top = m2;
  }
  if (c == 0) sm_m[part] = top, sm_l[part] = sum;
  *reinterpret_cast<f4_f32x4*>(&sm_o[part][4 * c]) = acc;
  __syncthreads();
  if (tid < D) {
    float tm = kFp4MinusBig, tl = 0.f, x = 0.f;
#pragma unroll
    for (int y = 0; y < AT_ONCE; ++y) tm = fmaxf(tm, sm_m[y]);
#pragma unroll
    for (int y = 0; y < AT_ONCE; ++y) {
      const float f = fp4_exp2(sm_m[y] - tm);
      tl += sm_l[y] * f;
      x += sm_o[y][tid] * f;
    }
    fp4_store_out(p.out, ((int64_t)b * p.m + j) * p.out_stride_t + hd * p.out_stride_h + tid, x / tl, p.out_f32 != 0, BF16);
  }
}

// Workgroup slots of the chip for the plan: the workgroups that are resident together.
static int fp4_plan_slots(int head_dim, int64_t rows, int cus) { return cus * fp4_wgs_per_cu(head_dim, (int)(rows > 64 ? 64 : rows)); }

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
static void fp4_launch(const Fp4DecodeParams& p, int pieces, hipStream_t s) {
  const unsigned grid = (unsigned)pieces * (unsigned)p.Hkv;
  const int R = p.m * p.G;
  if (R <= 8) fp4_decode_kernel<D, BF16, 1, true><<<grid, 256, 0, s>>>(p);
  else if (R <= 16) fp4_decode_kernel<D, BF16, 1, false><<<grid, 256, 0, s>>>(p);
  else if (R <= 32) fp4_decode_kernel<D, BF16, 2, false><<<grid, 256, 0, s>>>(p);
  else fp4_decode_kernel<D, BF16, 4, false><<<grid, 256, 0, s>>>(p);
  fp4_join_kernel<D, BF16><<<dim3((unsigned)(p.m * p.H), (unsigned)p.batch), 256, 0, s>>>(p);
}

}  // namespace tmx

extern "C" int64_t tmx_decode_fp4_workspace_rows(int batch, int rows_per_request, int num_heads, int num_kv_heads, int head_dim, int num_cus) {
  using namespace tmx;
  if (batch <= 0 || rows_per_request <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0) return 0;
  if (num_cus <= 0 && fp4_cus(&num_cus) != TMX_OK) return -1;
  const int64_t R = (int64_t)rows_per_request * (num_heads / num_kv_heads);
  const int slots = fp4_plan_slots(head_dim, R, num_cus);
  const int64_t pieces = (slots + num_kv_heads - 1) / num_kv_heads + (int64_t)batch;  // bound of the step's pieces
  return pieces * rows_per_request * num_heads;
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
  TMX_CHECK_SUPPORTED(a->num_kv_heads <= 1024, "tmx_decode_attention_fp4: more than 1024 K/V heads");
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
  int cus = 0;
  {
    const int rc = fp4_cus(&cus);
    if (rc != TMX_OK) return rc;
  }
  Fp4DecodeParams p{};
  p.plan_slots = fp4_plan_slots(a->head_dim, R, cus);
  const int64_t pieces = (p.plan_slots + a->num_kv_heads - 1) / a->num_kv_heads + (int64_t)a->batch;
  const int64_t rows = pieces * a->rows_per_request * a->num_heads;
  TMX_CHECK_ARG(a->partial_o != nullptr && a->partial_ml != nullptr && ((uintptr_t)a->partial_o % 16 == 0),
                "tmx_decode_attention_fp4: the work area is missing (tmx_decode_fp4_workspace_rows)");
  TMX_CHECK_ARG(a->workspace_rows >= rows,
                "tmx_decode_attention_fp4: the work area holds %lld rows, this batch size needs %lld (tmx_decode_fp4_workspace_rows)",
                (long long)a->workspace_rows, (long long)rows);
  TMX_CHECK_SUPPORTED(pieces * a->num_kv_heads <= 0x7fffffff, "tmx_decode_attention_fp4: too many workgroups");
  p.q = a->q;
  p.out = a->out;
  p.k = (const uint8_t*)a->k;
  p.v = (const uint8_t*)a->v;
  p.stride_page = a->kv_stride_page;
  p.num_pages = (int)a->num_pages;
  p.block_table = a->block_table;
  p.block_table_stride = a->block_table_stride;
  p.max_blocks = a->max_blocks;
  p.page_shift = __builtin_ctz(a->page_size);
  p.seq_lens = a->seq_lens;
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
  hipStream_t s = (hipStream_t)stream;
  const bool bf16 = a->io_dtype == TMX_BF16;
  if (a->head_dim == 128) {
    if (bf16) fp4_launch<128, true>(p, (int)pieces, s);
    else fp4_launch<128, false>(p, (int)pieces, s);
  } else {
    if (bf16) fp4_launch<64, true>(p, (int)pieces, s);
    else fp4_launch<64, false>(p, (int)pieces, s);
  }
  TMX_CHECK_HIP(hipGetLastError());
  return TMX_OK;
}
