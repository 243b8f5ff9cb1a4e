// Device-side pieces of the microscaled 4-bit format shared by the row operators and the convolution (gfx950 only).
#pragma once

#include "scn_device.hpp"

namespace scn {

// max over the lanes whose numbers differ in the lowest log2(W) bits (W = 2, 4 or 8)
template <int W>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if (W >= 2) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));   // quad_perm 1,0,3,2
  if (W >= 4) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));   // quad_perm 2,3,0,1
  if (W >= 8) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));  // row_half_mirror
  return v;
}

// Scale byte of a block from the fp32 bits of its largest magnitude (255: not finite).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top_bits) {
  const uint32_t f = top_bits >> 23;
  return f == 255u ? 255u : f > 2u ? f - 2u : 0u;
}

// 8 fp32 values times `up` -> 8 codes (the conversion instruction rounds to nearest even and saturates).
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8], float up) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0] * up, v[1] * up, 1.f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2] * up, v[3] * up, 1.f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4] * up, v[5] * up, 1.f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6] * up, v[7] * up, 1.f, 3);
  return r;
}

}  // namespace scn
