// fp8_block.h -- rows in blocks of 128 E4M3 codes with a shared power of two.
//
// A row of K values is n = ceil(K / 128) blocks: 128 n code bytes, and 4 ceil(n / 4)
// scale bytes, so that four blocks' scales are one dword.  Code c of a block stands for
// its E4M3 value times 2^(scale - 127) (E8M0; 255: the block is NaN).  Codes past K and
// scales past n are 0.  The scale is the least power of two (from 2^-127) that the
// block's largest magnitude over it does not pass 448 with: every quotient is exact, and
// a code's rounding, to nearest with ties to the even code, the only one.
#ifndef SMAUL_FP8_BLOCK_H
#define SMAUL_FP8_BLOCK_H

#include "e4m3.h"
#include "smaul_common.h"

namespace {

constexpr int FB_BLOCK = 128;

__host__ __device__ __forceinline__ int64_t fb_blocks(int64_t K) { return (K + FB_BLOCK - 1) / FB_BLOCK; }
__host__ __device__ __forceinline__ int64_t fb_width(int64_t K) { return fb_blocks(K) * FB_BLOCK; }  // a row's codes
__host__ __device__ __forceinline__ int64_t fb_words(int64_t K) { return (fb_blocks(K) + 3) / 4; }   // of its scales

// 2^(byte - 127): byte 0 is the subnormal 2^-127, 255 NaN
__device__ __forceinline__ float fb_scale(uint32_t byte) {
  return __uint_as_float(byte == 255 ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}

// From the bits of the largest magnitude: its exponent less 8 (448 = 1.75 * 2^8), one
// more where its mantissa is past 1.75.  Infinities and NaN have the largest bits, from
// `infinity` on: 255.
__device__ __forceinline__ uint32_t fb_scale_byte(uint32_t amax_bits, uint32_t infinity = 0x7f800000u) {
  if (amax_bits >= infinity) return 255u;
  return (uint32_t)max((int)((amax_bits + 0x1fffffu) >> 23) - 8, 0);
}

// 8 values -> 8 codes
__device__ __forceinline__ uint2 fb_encode8(const float* v, uint32_t byte) {
  if (byte == 255) return make_uint2(0, 0);
  const float s = fb_scale(byte);
  typedef short s16x2_t __attribute__((ext_vector_type(2)));
  s16x2_t lo = {0, 0}, hi = {0, 0};
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, v[0], v[1], s, false);
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, v[2], v[3], s, true);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, v[4], v[5], s, false);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, v[6], v[7], s, true);
  return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// 4 codes -> 4 values, exact (scaled by a product: the conversion's own scale gives no subnormals)
__device__ __forceinline__ void fb_decode4(uint32_t w, float s, float* v) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, false);
  const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, true);
  v[0] = a.x * s; v[1] = a.y * s; v[2] = b.x * s; v[3] = b.y * s;
}

// 16 bytes from an address of no more than the values' own alignment
typedef uint32_t fb_u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t fb_u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));

// NT: past the caches, for rows that are larger than they are
constexpr int64_t FB_NT_BYTES = 128LL << 20;  // half of the last cache
struct FbAt2 { typedef fb_u32x4_at2 T; };  // (a template argument would lose the alignment)
struct FbAt4 { typedef fb_u32x4_at4 T; };
template <class At, bool NT>
__device__ __forceinline__ uint4 fb_ld16(const void* p) {
  typedef typename At::T T;
  T v;
  if constexpr (NT) v = __builtin_nontemporal_load((const T*)p);
  else v = *(const T*)p;
  return make_uint4(v.x, v.y, v.z, v.w);
}
template <class At, bool NT>
__device__ __forceinline__ void fb_st16(void* p, uint4 v) {
  typedef typename At::T T;
  const T w = {v.x, v.y, v.z, v.w};
  if constexpr (NT) __builtin_nontemporal_store(w, (T*)p);
  else *(T*)p = w;
}
// 8 consecutive values of a row of K from column c0, 0 past K
template <bool BF16, bool NT = false>
__device__ __forceinline__ void fb_load8(const void* x, int64_t row, int64_t K, int64_t c0, float (&v)[8]) {
  const int64_t i = row * K + c0;
  if (c0 + 8 <= K) {
    if constexpr (BF16) {
      const uint4 q = fb_ld16<FbAt2, NT>((const uint16_t*)x + i);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 q = fb_ld16<FbAt4, NT>((const float*)x + i + 4 * h);
        v[4 * h] = __uint_as_float(q.x); v[4 * h + 1] = __uint_as_float(q.y);
        v[4 * h + 2] = __uint_as_float(q.z); v[4 * h + 3] = __uint_as_float(q.w);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = c0 + j < K ? (BF16 ? bf2f(((const uint16_t*)x)[i + j]) : ((const float*)x)[i + j]) : 0.0f;
  }
}

// ... and to it, nothing past K
template <bool BF16, bool NT = false>
__device__ __forceinline__ void fb_store8(void* y, int64_t row, int64_t K, int64_t c0, const float (&v)[8]) {
  const int64_t i = row * K + c0;
  if constexpr (BF16) {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
    if (c0 + 8 <= K) {
      fb_st16<FbAt2, NT>((uint16_t*)y + i, make_uint4(u[0], u[1], u[2], u[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j < K) ((uint16_t*)y)[i + j] = (uint16_t)(u[j / 2] >> (16 * (j & 1)));
    }
  } else {
    if (c0 + 8 <= K) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        fb_st16<FbAt4, NT>((float*)y + i + 4 * h,
                           make_uint4(__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]),
                                      __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3])));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j < K) ((float*)y)[i + j] = v[j];
    }
  }
}

// the largest magnitude's bits (as integers: the order of magnitudes, then Inf, NaN)
__device__ __forceinline__ uint32_t fb_amax8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  return m;
}

// a block is 16 neighbouring lanes of 8 values: its largest bits, in each of them
__device__ __forceinline__ uint32_t fb_block_max(uint32_t m) {
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d, 16));
  return m;
}

// Chunk `chunk` (8 values) of row `row` as codes, called by the 16 lanes of a block at
// once; the first writes the block's scale, and the last block's the scales past it.
__device__ __forceinline__ void fb_write8(uint8_t* codes, uint8_t* scales, int64_t row, int64_t nb, int64_t chunk,
                                          const float (&v)[8], uint32_t infinity = 0x7f800000u) {
  const uint32_t byte = fb_scale_byte(fb_block_max(fb_amax8(v)), infinity);
  *(uint2*)(codes + row * nb * FB_BLOCK + chunk * 8) = fb_encode8(v, byte);
  if ((chunk & 15) == 0) {
    const int64_t b = chunk / 16, ns = (nb + 3) / 4 * 4;
    uint8_t* s = scales + row * ns;
    s[b] = (uint8_t)byte;
    if (b + 1 == nb)
      for (int64_t j = nb; j < ns; ++j) s[j] = 0;
  }
}

constexpr int64_t fb_align256(int64_t v) { return (v + 255) / 256 * 256; }
inline bool fb_aligned(const void* p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }
inline bool fb_dtype_ok(int d) { return d == SMAUL_DTYPE_F32 || d == SMAUL_DTYPE_BF16; }

}  // namespace

#endif  // SMAUL_FP8_BLOCK_H
