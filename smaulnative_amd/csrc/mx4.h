// mx4.h -- blocks of 32 4-bit floating point values with a shared power of two.
//
// A row of K values is ceil(K / 32) blocks; block b is 16 bytes of codes (value
// 2 j in the low half of byte j, value 2 j + 1 in the high half) and one scale
// byte.  Code c stands for {0, .5, 1, 1.5, 2, 3, 4, 6}[c & 7], negative with bit 3
// (E2M1), times 2^(scale - 127) (E8M0; 255: the block is NaN).  Values past K in
// the last block are code 0.
#ifndef SMAUL_MX4_H
#define SMAUL_MX4_H

#include "e4m3.h"
#include "smaul_common.h"

namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int MX4_BLOCK = 32;

__host__ __device__ __forceinline__ int64_t mx4_blocks(int64_t K) { return (K + MX4_BLOCK - 1) / MX4_BLOCK; }

// 2^(byte - 127) as fp32: byte 0 is the subnormal 2^-127, 255 NaN
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
  return __uint_as_float(byte == 255 ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}

// The scale byte of a block from the bits of its largest magnitude: the exponent
// of that, less 2 (the exponent of the largest code, 6), so that the scaled values
// are below 8.  Infinities and NaN have the largest bits, and give 255.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}

// 8 values -> 8 codes.  The conversion divides by the scale and rounds to
// nearest, ties to the even code, past 6 to 6.
__device__ __forceinline__ uint32_t mx4_encode8(const float* v, uint32_t byte) {
  if (byte == 255) return 0;
  const float s = mx4_scale(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
  return w;
}

// 8 codes -> 8 bf16 (exact: two significant bits; four dwords), times s
__device__ __forceinline__ uint4 mx4_decode8(uint32_t w, float s) {
  uint4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
  return r;
}

}  // namespace

#endif  // SMAUL_MX4_H
