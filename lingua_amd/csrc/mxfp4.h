// What the MXFP4 kernels share: the format's arithmetic and the interface between their files.
#pragma once
#include "l8_common.h"

namespace l8 {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kMxBlock = 32;   // elements per scale

// A product of few tokens (M <= 64).  x: bf16, ldx in elements, or codes with scales sx, ldx in bytes.
struct MxFewArgs {
  const void *x;
  const uint8_t *sx, *qw, *sw;
  int64_t ldx, ldsx, ldqw, ldsw;
  const uint16_t *bias;
  uint16_t *y;
  int64_t ldy;
  int M, N, K, blocks;
};

#if defined(__HIP_DEVICE_COMPILE__)
// byte of a block whose largest magnitude has the bf16 bits `amax`
L8_DEV uint32_t mx_byte(uint32_t amax) {
  const uint32_t e = amax >> 7;
  return e == 255u ? 255u : (e < 2u ? 0u : e - 2u);
}
// 2^(byte - 127) as fp32: what the conversion divides by (byte 0 is the subnormal 2^-127)
L8_DEV float mx_scale(uint32_t byte) { return __uint_as_float(byte == 0u ? 0x00400000u : byte << 23); }

// eight bf16 (four packed pairs) -> eight codes, the first in the low nibble
L8_DEV uint32_t mx_codes8(uint32_t p0, uint32_t p1, uint32_t p2, uint32_t p3, float scale) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, p0), scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, p1), scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, p2), scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, p3), scale, 3);
  return r;
}
L8_DEV uint32_t amax8(v4i v) {
  uint32_t m = pk_absmax_u16(0, (uint32_t)v[0]);
#pragma unroll
  for (int k = 1; k < 4; ++k) m = pk_absmax_u16(m, (uint32_t)v[k]);
  return max(m & 0xffffu, m >> 16);
}
template <int CTRL>
L8_DEV uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true); }
// maximum over the four lanes of a quad
L8_DEV uint32_t quad_max(uint32_t v) {
  v = max(v, dpp<0xB1>(v));    // quad_perm [1,0,3,2]
  return max(v, dpp<0x4E>(v)); // quad_perm [2,3,0,1]
}
#endif

}  // namespace l8
