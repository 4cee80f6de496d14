// Microscaled 4-bit floating point (MXFP4): blocks of 32 consecutive values, each an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// their negatives; two to a byte, the even one in the low half) under one E8M0 scale byte E, a power of two s = 2^(E - 127).
// Codec written from the OCP microscaling specification's formats; the rule of the scale is this library's:
//
//   a = max|x|,  s the smallest power of two with a < 7 s, E kept in [2, 252];   code = nearest e2m1 of x / s, ties to even
//
// A quotient of 6 .. 7 rounds to 6 within half the step of its binade, so no value of a block is off by more than that; the
// specification's s = 2^(floor(log2 a) - 2) cuts 7 .. 8 to 6 as well.  x / s is exact.  E's bounds keep s and every code's
// value normal and finite in fp32 and bf16.  A block that holds a NaN or an infinity: E = 255 and zero codes, which reads back
// as NaN.
#pragma once

#include "wf_common.hpp"

namespace wf {
namespace mx {

constexpr int kBlock = 32;       // values of a block
constexpr int kMinE = 2, kMaxE = 252;
constexpr int kNanE = 255;

// Scale byte of a block from the bits of its largest magnitude as bf16 (infinities and NaN order above all others).  Adding a
// quarter of the exponent's unit carries where the significand is 1.75 or more.
__host__ __device__ inline int scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f80u) return kNanE;
  const int e = static_cast<int>((amax_bits + 0x20u) >> 7) - 2;
  return e < kMinE ? kMinE : e > kMaxE ? kMaxE : e;
}

#if defined(__HIPCC__)
// 2^(E - 127); infinity for 255, which the conversions below take for NaN, and 0 for 0, which they take for 2^-127 (all
// checked over every code and every byte).
__device__ inline float scale_of(int e) { return bits_f32(static_cast<uint32_t>(e) << 23); }

// The larger of each half's magnitude bits, of two words of two bf16.
__device__ inline uint32_t max_bits2(uint32_t a, uint32_t b) {
  typedef unsigned short u2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u2, a & 0x7fff7fffu), __builtin_bit_cast(u2, b & 0x7fff7fffu)));
}
__device__ inline uint32_t max_half(uint32_t a) { return max(a & 0xffffu, a >> 16); }

// v of the lane that a DPP control names.
template <int CTRL>
__device__ inline uint32_t dpp_u32(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
}

// 8 bf16 (four words) as 8 codes under s (v_cvt_scalef32_pk_fp4_bf16: nearest, ties to even, saturated at 6; equal to the
// definition for every finite bf16).
__device__ inline uint32_t encode8(const uint32_t* w, float s) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(b2, w[0]), s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(b2, w[1]), s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(b2, w[2]), s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(b2, w[3]), s, 3);
  return c;
}

// 8 codes as 8 bf16, exact (two significant bits) where s is of a byte 2 .. 252.
__device__ inline uint4 decode8(uint32_t c, float s) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3)));
}
#endif

}  // namespace mx
}  // namespace wf
