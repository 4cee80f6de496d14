// One cached (token, head) row of 128 values: e4m3 quantization and dequantization, and its 16-byte accesses
// (arithmetic and error argument: kv_pages.hip).
#pragma once

#include "fp8_codec.hpp"
#include "wf_common.hpp"

namespace wf {

constexpr int kHeadDim = 128;

// Four e4m3 codes of bf16-exact values x[0..3] with scale s (r within one ulp of 1/s).
__device__ inline uint32_t quant4f(const float* x, float s, float r) {
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float ax = fabsf(x[i]);
    float qi = ax * r;
    const float e = fmaf(-qi, s, ax);
    qi = fmaf(e, r, qi);
    qi = fminf(qi, kE4M3Max);
    q[i] = bits_f32(f32_bits(qi) | (f32_bits(x[i]) & 0x80000000u));
  }
  return e4m3_pack4_hw(q[0], q[1], q[2], q[3]);
}

// bf16(amax / 448) as bf16(amax * RN(1/448)) (kv_pages.hip), floored at bf16(1e-8).
constexpr float kInvE4M3Max = 1.0f / kE4M3Max;
__device__ inline float scale_from_amax(float amax) {
  const float s = bf16_bits_to_f32(static_cast<uint16_t>(pack_bf16x2_hw(amax * kInvE4M3Max, 0.f)));
  return fmaxf(s, bf16_bits_to_f32(kScaleFloorBf16Bits));
}

__device__ inline uint2 dequant4(uint32_t w, float s) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  float v0, v1, v2, v3;
  e4m3_unpack4_hw(w, v0, v1, v2, v3);
  const f2 lo = {v0 * s, v1 * s};
  const f2 hi = {v2 * s, v3 * s};
  const b2 blo = __builtin_convertvector(lo, b2);
  const b2 bhi = __builtin_convertvector(hi, b2);
  return make_uint2(__builtin_bit_cast(uint32_t, blo), __builtin_bit_cast(uint32_t, bhi));
}

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <bool NT>
__device__ inline uint4 ld16(const uint4* p) {
  if constexpr (NT) {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    return make_uint4(v[0], v[1], v[2], v[3]);
  } else {
    return *p;
  }
}

template <bool NT>
__device__ inline void st16(uint4* p, const uint4& v) {
  if constexpr (NT) {
    const u32x4 w = {v.x, v.y, v.z, v.w};
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
  } else {
    *p = v;
  }
}

}  // namespace wf
