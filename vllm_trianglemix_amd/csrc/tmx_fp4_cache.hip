// 4-bit (MXFP4) paged K/V cache: the quantising write of a step's rows and the read-back of whole sequences as 16-bit
// rows (what reshape_and_cache_flash and the descale around the attention call are for the reference's 16-bit and fp8
// caches, csrc/cache_kernels.cu:282-355, vllm/v1/attention/backends/rocm_attn.py:345-358).  Both are bound by the
// bytes they move; the layout of a page is described in tmx_fp4.h.
#include "tmx_common.h"
#include "tmx_fp4.h"

namespace tmx {

// One wave quantises twice n = 512 / D consecutive tokens of one head of K or of V (8192 tokens x 8 heads: 8.7 us, 4.9 TB/s
// read + written, against 10.2 with n at a time and 8.5 with four times n, which costs single steps 0.8 us more): a lane holds 8 columns (16
// bytes), four neighbouring lanes a block of 32.  K lanes run along the row, V lanes along the tokens first: in both cases
// the wave's stores form runs (K the rows of D / 2 bytes, V the n tokens of a 16-byte unit side by side).
template <int D>
__global__ __launch_bounds__(256) void fp4_write_kernel(
    const uint16_t* __restrict__ key, const uint16_t* __restrict__ value, int64_t key_stride_t, int64_t key_stride_h,
    int64_t value_stride_t, int64_t value_stride_h, uint8_t* __restrict__ key_cache, uint8_t* __restrict__ value_cache,
    int64_t stride_page, const int64_t* __restrict__ slot_mapping, int num_tokens, int kv_heads, int page_shift,
    int64_t num_slots, int bf16) {
  constexpr int n = 512 / D, chunks = D / 8, GROUPS = 2;
  const int lane = threadIdx.x & 63;
  const unsigned unit = blockIdx.x * 4u + (threadIdx.x >> 6);
  const int h = (int)(unit % (unsigned)kv_heads);
  const int64_t grp = unit / (unsigned)kv_heads;
  const bool is_v = blockIdx.y != 0;
  const int tok = is_v ? lane % n : lane / chunks, ch = is_v ? lane / n : lane % chunks;
  const uint16_t* rows_in = (is_v ? value + (int64_t)h * value_stride_h : key + (int64_t)h * key_stride_h) + ch * 8;
  const int64_t stride_t = is_v ? value_stride_t : key_stride_t;
  const int ps = 1 << page_shift;
  uint8_t* const cache = is_v ? value_cache : key_cache;
  const int64_t head_codes = (int64_t)h * ps * (D / 2);
  const int64_t scales = fp4_code_bytes(kv_heads, ps, D) + ((int64_t)h * (D / 32) + (ch >> 2)) * ps;
  uint4 x[GROUPS];
  int64_t slot[GROUPS];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const int64_t t = (grp * GROUPS + i) * n + tok;
    x[i] = make_uint4(0, 0, 0, 0);
    slot[i] = -1;
    if (t < num_tokens) {
      slot[i] = slot_mapping[t];
      x[i] = *reinterpret_cast<const uint4*>(rows_in + t * stride_t);
    }
  }
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    // the block's largest magnitude: four lanes hold it
    unsigned m = fp4_amax8(x[i]);
    const int step = is_v ? n : 1;
    m = max(m, (unsigned)__shfl_xor((int)m, step, 64));
    m = max(m, (unsigned)__shfl_xor((int)m, 2 * step, 64));
    if (slot[i] < 0 || slot[i] >= num_slots) continue;
    const unsigned byte = fp4_scale_byte(m, bf16 != 0);
    const unsigned codes = fp4_codes8(x[i], byte, bf16 != 0);
    const int at = (int)(slot[i] & (ps - 1));
    uint8_t* page = cache + (slot[i] >> page_shift) * stride_page;
    uint8_t* rows = page + head_codes;
    if (!is_v) {
      *reinterpret_cast<unsigned*>(rows + at * (D / 2) + ch * 4) = codes;
    } else if (D == 128) {
      *reinterpret_cast<unsigned*>(rows + (at / n) * 256 + ch * 16 + (at % n) * 4) = codes;
    } else {  // 8 columns are two units' worth
      uint8_t* u = rows + (at / n) * 256 + ch * 32 + (at % n) * 2;
      *reinterpret_cast<uint16_t*>(u) = (uint16_t)codes;
      *reinterpret_cast<uint16_t*>(u + 16) = (uint16_t)(codes >> 16);
    }
    if ((ch & 3) == 0) page[scales + at] = (uint8_t)byte;
  }
}

// Eight codes as eight 16-bit values.  bf16 holds every value that the write makes (scale bytes up to 252); fp16 does not:
// magnitudes from 65536 on saturate at 65504 (a value of 65504 is stored as 4 x 2^14), NaN stays NaN.
__device__ __forceinline__ uint4 fp4_values8(unsigned w, unsigned byte, bool bf16) {
  const float s = __uint_as_float(byte << 23);
  if (bf16) return make_uint4(fp4_bf16<0>(w, s), fp4_bf16<1>(w, s), fp4_bf16<2>(w, s), fp4_bf16<3>(w, s));
  uint4 r = make_uint4(fp4_f16<0>(w, s), fp4_f16<1>(w, s), fp4_f16<2>(w, s), fp4_f16<3>(w, s));
  if (byte >= 127 + 14 && byte != 255) {  // 4 x 2^14 and up: an infinity's bits become those of 65504
    unsigned* v = reinterpret_cast<unsigned*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((v[i] & 0x7fffu) == 0x7c00u) v[i] -= 1u;
      if ((v[i] & 0x7fff0000u) == 0x7c000000u) v[i] -= 0x10000u;
    }
  }
  return r;
}

// One wave converts 16 consecutive tokens (part of one page) of one head of K or of V: a lane 4 code bytes at a time, the
// lanes in the order of the output row, so that every store instruction writes whole rows.  Bound by the rows it writes;
// they go past the caches (2 x 32768 tokens x 8 heads: 49 us, 6.9 TB/s, against 65 with cached stores).
template <int D>
__global__ __launch_bounds__(256) void fp4_gather_kernel(
    const uint8_t* __restrict__ key_cache, const uint8_t* __restrict__ value_cache, int64_t stride_page, int num_pages,
    const int32_t* __restrict__ block_table, int64_t block_table_stride, int max_blocks, int page_shift,
    const int32_t* __restrict__ seq_lens, const int32_t* __restrict__ cu_k, int64_t total_rows, uint16_t* __restrict__ k_out,
    uint16_t* __restrict__ v_out, int kv_heads, int bf16) {
  constexpr int n = 512 / D, chunks = D / 8, steps = 16 / n;
  const int lane = threadIdx.x & 63;
  const unsigned unit = blockIdx.x * 4u + (threadIdx.x >> 6);
  const int h = (int)(unit % (unsigned)kv_heads);
  const int64_t first = (int64_t)(unit / (unsigned)kv_heads) * 16;
  const int b = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const uint8_t* const cache = is_v ? value_cache : key_cache;
  uint16_t* const out = is_v ? v_out : k_out;
  const int len = seq_lens[b];
  if (first >= len) return;
  const int tok0 = (int)first;
  const int ps = 1 << page_shift;
  const int tl = lane / chunks, ch = lane % chunks;
  const int blk = tok0 >> page_shift;
  const int page = blk < max_blocks ? block_table[b * block_table_stride + blk] : -1;
  const bool good = page >= 0 && page < num_pages;  // no such page: its rows read as NaN
  const int at0 = tok0 & (ps - 1);
  const int64_t off = (good ? (int64_t)page : 0) * stride_page;
  const int64_t code0 = off + (int64_t)h * ps * (D / 2) + at0 * (D / 2);
  const int64_t scale0 = off + fp4_code_bytes(kv_heads, ps, D) + ((int64_t)h * (D / 32) + (ch >> 2)) * ps + at0 + tl;
  unsigned code[steps], byte[steps];
#pragma unroll
  for (int i = 0; i < steps; ++i) {
    if (!is_v) {
      code[i] = *reinterpret_cast<const unsigned*>(cache + code0 + i * 256 + lane * 4);
    } else if (D == 128) {
      code[i] = *reinterpret_cast<const unsigned*>(cache + code0 + i * 256 + ch * 16 + tl * 4);
    } else {
      const uint8_t* u = cache + code0 + i * 256 + ch * 32 + tl * 2;
      code[i] = *reinterpret_cast<const uint16_t*>(u) | (unsigned)*reinterpret_cast<const uint16_t*>(u + 16) << 16;
    }
    byte[i] = good ? cache[scale0 + i * n] : 255u;
  }
  const int64_t row0 = cu_k[b];
#pragma unroll
  for (int i = 0; i < steps; ++i) {
    const int t = tok0 + i * n + tl;
    const int64_t row = row0 + t;
    if (t >= len || row < 0 || row >= total_rows) continue;
    const int64_t dst = (row * kv_heads + h) * D + ch * 8;
    __builtin_nontemporal_store(__builtin_bit_cast(fp4_u32x4, fp4_values8(code[i], byte[i], bf16 != 0)), reinterpret_cast<fp4_u32x4*>(out + dst));
  }
}

static int fp4_check_cache(const char* fn, const void* k, const void* v, int64_t stride_page, int64_t num_pages, int kv_heads,
                           int head_dim, int page_size) {
  TMX_CHECK_ARG(kv_heads > 0 && head_dim > 0 && num_pages >= 0, "%s: bad sizes", fn);
  TMX_CHECK_SUPPORTED(head_dim == 64 || head_dim == 128, "%s: head_dim %d not covered (64 and 128 are)", fn, head_dim);
  TMX_CHECK_SUPPORTED(page_size >= 16 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0,
                      "%s: page_size %d not supported (powers of two from 16 to 2^20 are)", fn, page_size);
  TMX_CHECK_SUPPORTED(num_pages <= 0x7fffffff, "%s: more than 2^31 - 1 pages", fn);
  TMX_CHECK_SUPPORTED(kv_heads <= 1024 && fp4_page_bytes(kv_heads, page_size, head_dim) <= 0x7fffffff,
                      "%s: more than 1024 K/V heads, or a page of 2^31 bytes or more", fn);
  TMX_CHECK_ARG(stride_page >= fp4_page_bytes(kv_heads, page_size, head_dim) && stride_page % 16 == 0,
                "%s: the page stride %lld must be a multiple of 16 bytes and hold a page of %lld", fn, (long long)stride_page,
                (long long)fp4_page_bytes(kv_heads, page_size, head_dim));
  TMX_CHECK_ARG(((uintptr_t)k % 16 == 0) && ((uintptr_t)v % 16 == 0), "%s: the caches must be 16-byte aligned", fn);
  return TMX_OK;
}

}  // namespace tmx

extern "C" int tmx_reshape_and_cache_fp4(const void* key, const void* value, int64_t key_stride_t, int64_t key_stride_h,
                                         int64_t value_stride_t, int64_t value_stride_h, void* key_cache, void* value_cache,
                                         int64_t stride_page, int64_t num_pages, const int64_t* slot_mapping,
                                         int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                         int32_t in_dtype, void* stream) {
  using namespace tmx;
  TMX_CHECK_ARG(num_tokens >= 0, "tmx_reshape_and_cache_fp4: bad sizes");
  TMX_CHECK_SUPPORTED(in_dtype == TMX_BF16 || in_dtype == TMX_F16,
                      "tmx_reshape_and_cache_fp4: key / value must be bf16 or fp16 (dtype %d)", in_dtype);
  const int rc = fp4_check_cache("tmx_reshape_and_cache_fp4", key_cache, value_cache, stride_page, num_pages, num_kv_heads,
                                 head_dim, page_size);
  if (rc != TMX_OK) return rc;
  if (num_tokens == 0 || num_pages == 0) return TMX_OK;
  TMX_CHECK_ARG(key && value && key_cache && value_cache && slot_mapping, "tmx_reshape_and_cache_fp4: NULL pointer");
  TMX_CHECK_ARG(key_stride_t % 8 == 0 && key_stride_h % 8 == 0 && value_stride_t % 8 == 0 && value_stride_h % 8 == 0,
                "tmx_reshape_and_cache_fp4: key / value strides must be multiples of 8 elements");
  TMX_CHECK_ARG(((uintptr_t)key % 16 == 0) && ((uintptr_t)value % 16 == 0),
                "tmx_reshape_and_cache_fp4: key / value must be 16-byte aligned");
  const int n = 512 / head_dim;
  const int64_t units = ((int64_t)num_tokens + 2 * n - 1) / (2 * n) * num_kv_heads;
  TMX_CHECK_SUPPORTED((units + 3) / 4 <= 0x3fffffff, "tmx_reshape_and_cache_fp4: too many tokens for one launch");
  const dim3 grid((unsigned)((units + 3) / 4), 2);
  auto* kernel = head_dim == 128 ? fp4_write_kernel<128> : fp4_write_kernel<64>;
  kernel<<<grid, 256, 0, (hipStream_t)stream>>>(
      (const uint16_t*)key, (const uint16_t*)value, key_stride_t, key_stride_h, value_stride_t, value_stride_h,
      (uint8_t*)key_cache, (uint8_t*)value_cache, stride_page, slot_mapping, num_tokens, num_kv_heads,
      __builtin_ctz(page_size), num_pages * page_size, in_dtype == TMX_BF16);
  TMX_CHECK_HIP(hipGetLastError());
  return TMX_OK;
}

extern "C" int tmx_gather_dequant_kv_fp4(const void* key_cache, const void* value_cache, int64_t stride_page, int64_t num_pages,
                                         const int32_t* block_table, int64_t block_table_stride, int32_t max_blocks,
                                         int32_t page_size, const int32_t* seq_lens, const int32_t* cu_seqlens_k, int32_t batch,
                                         int32_t max_seq_len, int32_t num_kv_heads, int32_t head_dim, void* k_out, void* v_out,
                                         int64_t total_rows, int32_t out_dtype, void* stream) {
  using namespace tmx;
  TMX_CHECK_ARG(batch >= 0 && max_seq_len >= 0 && max_blocks >= 0 && total_rows >= 0 && block_table_stride >= 0,
                "tmx_gather_dequant_kv_fp4: bad sizes");
  TMX_CHECK_SUPPORTED(out_dtype == TMX_BF16 || out_dtype == TMX_F16,
                      "tmx_gather_dequant_kv_fp4: output must be bf16 or fp16 (dtype %d)", out_dtype);
  const int rc = fp4_check_cache("tmx_gather_dequant_kv_fp4", key_cache, value_cache, stride_page, num_pages, num_kv_heads,
                                 head_dim, page_size);
  if (rc != TMX_OK) return rc;
  if (batch == 0 || max_seq_len == 0 || total_rows == 0) return TMX_OK;
  TMX_CHECK_ARG(num_pages > 0, "tmx_gather_dequant_kv_fp4: the cache has no pages");
  TMX_CHECK_SUPPORTED(batch <= 65535, "tmx_gather_dequant_kv_fp4: more than 65535 requests");
  TMX_CHECK_ARG(key_cache && value_cache && block_table && seq_lens && cu_seqlens_k && k_out && v_out,
                "tmx_gather_dequant_kv_fp4: NULL pointer");
  TMX_CHECK_ARG(((uintptr_t)k_out % 16 == 0) && ((uintptr_t)v_out % 16 == 0),
                "tmx_gather_dequant_kv_fp4: outputs must be 16-byte aligned");
  const int64_t units = ((int64_t)max_seq_len + 15) / 16 * num_kv_heads;
  TMX_CHECK_SUPPORTED(units <= 0x7ffffff0, "tmx_gather_dequant_kv_fp4: too many tokens for one launch");
  const dim3 grid((unsigned)((units + 3) / 4), (unsigned)batch, 2);
  auto* kernel = head_dim == 128 ? fp4_gather_kernel<128> : fp4_gather_kernel<64>;
  kernel<<<grid, 256, 0, (hipStream_t)stream>>>(
      (const uint8_t*)key_cache, (const uint8_t*)value_cache, stride_page, (int)num_pages, block_table, block_table_stride,
      max_blocks, __builtin_ctz(page_size), seq_lens, cu_seqlens_k, total_rows, (uint16_t*)k_out, (uint16_t*)v_out,
      num_kv_heads, out_dtype == TMX_BF16);
  TMX_CHECK_HIP(hipGetLastError());
  return TMX_OK;
}
