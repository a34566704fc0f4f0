// Rows in 4 bits: the format of the decode caches of dil_fp4_write, dil_fp4_read and
// dil_decode_step_fp4 (include/dilution_hip.h).
//
// A row of D elements is D / 2 bytes of codes, two a byte (the even element in the low half),
// and one scale byte for each block of min(32, D) elements.  A code is a sign and one of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 (2 exponent bits, 1 mantissa bit); an element is its code times
// 2^(s - 127).  The block's largest magnitude, 1.m 2^E, gives s - 127 = E - 2, or E - 1 from
// 1.75 on, where the nearest code would be 8: so every element is off by at most half a step
// of its own code.  s lies in [2, 252] (products with codes are then neither denormal nor
// infinite; a block past 6 * 2^125 saturates), is 255 for a block that holds a NaN or an
// infinity, all NaN then, and 0 in a row that was never written, all 0.
//
// gfx950 converts two codes an instruction, exactly (v_cvt_scalef32_pk_f32_fp4, and
// v_cvt_scalef32_pk_fp4_f32 back, nearest, ties to even).
#pragma once

#include "dil_common.hpp"

namespace dil {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int D> struct Fp4Row {
  static constexpr int kBlock = D < 32 ? D : 32;      // elements of a scale
  static constexpr int kBlocks = D / kBlock;
};

// The scale bytes of a row, as one load
template <int N> struct ScaleWord;
template <> struct ScaleWord<1> { using type = uint8_t; };
template <> struct ScaleWord<2> { using type = uint16_t; };
template <> struct ScaleWord<4> { using type = uint32_t; };
template <> struct ScaleWord<8> { using type = uint64_t; };

__device__ __forceinline__ float fp4_factor(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7fc00000u : s << 23);
}

// Bits of the largest of 8 magnitudes, as fp32 (a NaN's lie above those of every number)
template <int DT, typename R>
__device__ __forceinline__ uint32_t top_bits(const R& r) {
  uint32_t top = 0;
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(r[e]) & 0x7fffffffu);
    return top;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, static_cast<uint32_t>(r[e] & 0x7fff));
    return DT == DT_BF16 ? top << 16 : __float_as_uint(f16_bits_to_f32(static_cast<uint16_t>(top)));
  }
}

// The scale byte of a block whose largest magnitude has these fp32 bits
__device__ __forceinline__ uint32_t fp4_scale(uint32_t top) {
  const int s = static_cast<int>((top + 0x200000u) >> 23) - 2;
  return top >= 0x7f800000u ? 255u : static_cast<uint32_t>(min(max(s, 2), 252));
}

// The largest over the lanes (2 or 4 neighbours) that hold a block's elements, 8 each
template <int D>
__device__ __forceinline__ uint32_t block_top(uint32_t top) {
  constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E;   // quad_perm [1, 0, 3, 2], [2, 3, 0, 1]
  top = max(top, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(top), kQuadXor1, 0xF, 0xF, true)));
  if constexpr (Fp4Row<D>::kBlock == 32)
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(top), kQuadXor2, 0xF, 0xF, true)));
  return top;
}

// 8 elements as their codes under scale byte s
template <int DT, typename R>
__device__ __forceinline__ uint32_t fp4_codes8(const R& r, uint32_t s) {
  if (s == 255u) return 0u;
  const float inv = __uint_as_float((254u - s) << 23);       // exact: the products are the scaled elements
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (DT == DT_F32) y[e] = r[e] * inv;
    else y[e] = (DT == DT_BF16 ? bf16_bits_to_f32(r[e]) : f16_bits_to_f32(r[e])) * inv;
  }
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[0], y[1], 1.f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2], y[3], 1.f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[4], y[5], 1.f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[6], y[7], 1.f, 3);
  return c;
}

// The 8 values of a word of codes, unscaled
__device__ __forceinline__ void fp4_values8(uint32_t c, float (&v)[8]) {
  const floatx2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1);
  const floatx2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
  v[4] = d[0]; v[5] = d[1]; v[6] = e[0]; v[7] = e[1];
}

}  // namespace dil
