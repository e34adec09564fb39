// Device helpers of the 4-bit weight format (mx4.hip, mx4_gemm.hip, ce_pieces.hip).
#pragma once
#include "mfma.h"

namespace mft {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

// scale byte -> the fp32 whose exponent field it is; 255 -> NaN
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}

// 8 codes (one 32-bit word, low half-byte first) -> 8 bf16 values
__device__ __forceinline__ bf16x8_t mx4_cvt8(uint32_t w, float s) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 4 or 8 columns of a result row at any 2-byte address, as one store: rows of a width that is no multiple of 8 (24000 x 3268 x 128
// y 55 us, with 2-byte stores 143 us)
__device__ __forceinline__ void store4_any(bf16_t* p, f32x4_t v) {
  const uint2 q = {pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])};
  __builtin_memcpy(p, &q, 8);
}
__device__ __forceinline__ void store8_any(bf16_t* p, const float* v) {
  const uint4 q = {pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7])};
  __builtin_memcpy(p, &q, 16);
}

// the same with a scale for each code: a byte is converted under both its scales, the halves picked
__device__ __forceinline__ bf16x8_t mx4_cvt8(uint32_t w, f32x4_t s0, f32x4_t s1) {
  auto pick = [](bf16x2_t lo, bf16x2_t hi) {
    return (__builtin_bit_cast(uint32_t, lo) & 0xffffu) | (__builtin_bit_cast(uint32_t, hi) & 0xffff0000u);
  };
  const u32x4_t r = {pick(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s0[0], 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s0[1], 0)),
                     pick(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s0[2], 1), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s0[3], 1)),
                     pick(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s1[0], 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s1[1], 2)),
                     pick(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s1[2], 3), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s1[3], 3))};
  return __builtin_bit_cast(bf16x8_t, r);
}

}  // namespace mft
