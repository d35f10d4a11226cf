// The 4-bit K/V cache format (OCP MXFP4), shared by the kernels that write and read it.
//
// 32 neighbouring columns of a row share a power of two 2^e, stored as the byte e + 127; a value is one of 0, 0.5, 1,
// 1.5, 2, 3, 4, 6 with a sign (e2m1), times 2^e.  The byte 255 marks a block that held an infinity or a NaN: it reads
// back as NaN.
//
// A page of page_size tokens of K (or V) of one layer, page_bytes(...) bytes in one run:
//   codes   K  [head][token][D / 2]                              two codes to a byte, the even column in the low half
//           V  [head][token / n][16][token % n][D / 32]          n = 512 / D tokens
//   scales     [head][D / 32][token]                             one byte per 32 columns of a token
// A (page, head) is a contiguous run of both, so a workgroup that reads one head of a page reads whole cache lines; the
// V order hands a lane of the decode kernel, in one 16-byte load, the D / 16 columns of n tokens that it needs as
// matrix operand rows, so that V reaches the matrix cores without a pass through LDS (see tmx_fp4_decode.hip).
#pragma once

#include "tmx_common.h"

namespace tmx {

constexpr int kFp4Block = 32;          // columns per scale
constexpr int kFp4MaxByte = 125 + 127;  // the largest scale byte that the write makes, 255 apart

TMX_HD int64_t fp4_code_bytes(int kv_heads, int page_size, int head_dim) { return (int64_t)kv_heads * page_size * (head_dim / 2); }
TMX_HD int64_t fp4_page_bytes(int kv_heads, int page_size, int head_dim) {
  return fp4_code_bytes(kv_heads, page_size, head_dim) + (int64_t)kv_heads * page_size * (head_dim / kFp4Block);
}

#if defined(__HIPCC__)
typedef __attribute__((ext_vector_type(2))) __bf16 fp4_bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 fp4_f16x2;
typedef __attribute__((ext_vector_type(4))) unsigned fp4_u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned fp4_u32x2;

// Largest of eight 16-bit magnitudes (sign bit cleared): bit patterns of bf16 and fp16 order like the values, with
// infinities and NaNs above every finite one.
__device__ __forceinline__ unsigned fp4_amax8(uint4 x) {
  const unsigned w[4] = {x.x, x.y, x.z, x.w};
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
    m = max(m, max(lo, hi));
  }
  return m;
}

// The scale byte of a block whose largest magnitude has these 16 bits: e = floor(log2(amax)) - 2, one more from 1.75 *
// 2^floor(log2(amax)) on.  With it amax / 2^e lies in [3.5, 7): every value of the block is within half a step of its
// code (7 would be the midpoint above 6), none saturates.  e stays at or above -126, the smallest normal float, and at or
// below 125: 6 x 2^125 is the largest value a block can stand for that bf16 and fp32 hold, and what a block with amax >=
// 1.75 x 2^127 (bf16 only) would round to otherwise is 2^128.  There the codes saturate: values past 5 x 2^125 become
// 6 x 2^125, off by less than 2 x 2^125.
__device__ __forceinline__ unsigned fp4_scale_byte(unsigned amax, bool bf16) {
  unsigned bits;
  if (bf16) {
    bits = amax << 16;
  } else {
    bits = __float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)amax));
  }
  const int ex = (int)(bits >> 23);
  if (ex == 255) return 255u;
  const int e = ex - 2 + ((bits & 0x7fffffu) >= 0x600000u ? 1 : 0);
  return (unsigned)imin(imax(e, 1), kFp4MaxByte);
}

// Eight 16-bit values as eight codes (the conversion instruction rounds to nearest, ties to even, and saturates at 6).  A block with scale
// byte 255 gets zeros.
__device__ __forceinline__ unsigned fp4_codes8(uint4 x, unsigned byte, bool bf16) {
  const float s = __uint_as_float(byte << 23);
  unsigned r = 0;
  if (bf16) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf16x2, x.x), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf16x2, x.y), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf16x2, x.z), s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf16x2, x.w), s, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(fp4_f16x2, x.x), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(fp4_f16x2, x.y), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(fp4_f16x2, x.z), s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(fp4_f16x2, x.w), s, 3);
  }
  return byte == 255u ? 0u : r;
}

// Two codes (byte SEL of w) times 2^e as two bf16: exact, a code has one fraction bit.  scale = the byte in a float's
// exponent field; 255 gives NaN.
template <int SEL>
__device__ __forceinline__ unsigned fp4_bf16(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
template <int SEL>
__device__ __forceinline__ unsigned fp4_f16(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
}
#endif

}  // namespace tmx
