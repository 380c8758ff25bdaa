// mx4.hip -- blocks of 32 4-bit values on MI355X (gfx950): quantisation, the
// product with such a weight, its input gradient, and the routed experts.
//
//   y[r, n]  = sum_k x[r, k] W[n, k]           W[n, k] = code value * 2^(scale - 127)
//   dx[r, k] = sum_n g[r, n] W[n, k]
//   moe: out[t] = sum over t's experts of w (silu(x Wg^T) * (x Wu^T)) Wd^T
//
// A code and its scale are exact in bf16, so every product of the matrix cores is
// exact for bf16 activations and for activations in the format itself, and its
// sums are fp32; fp32 activations are two bf16 terms (hi + lo).
#include "mx4.h"

using smaul::check_launch;
using smaul::cu_count;
using smaul::fail;

namespace {

// ---------------------------------------------------------------------------
// quantisation: 4 lanes a block, 8 values a lane
// ---------------------------------------------------------------------------
// 8 consecutive values of a row from column c0, 0 past K
template <bool BF16, bool VEC>
__device__ __forceinline__ void mx4_load8(const void* x, int64_t row, int64_t K, int64_t c0, float (&v)[8]) {
  const int64_t i = row * K + c0;
  if constexpr (VEC) {
    if constexpr (BF16) {
      const uint4 w = *(const uint4*)((const uint16_t*)x + i);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(u[j] << 16);
        v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
      }
    } else {
      const float4 a = *(const float4*)((const float*)x + i), b = *(const float4*)((const float*)x + i + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = c0 + j < K ? (BF16 ? bf2f(((const uint16_t*)x)[i + j]) : ((const float*)x)[i + j]) : 0.0f;
  }
}

// the largest magnitude's bits (as integers: the order of magnitudes, then Inf, NaN)
__device__ __forceinline__ uint32_t mx4_amax8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  return m;
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256)
mx4_quantize_kernel(const void* __restrict__ x, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales,
                    int64_t rows, int64_t K) {
  const int64_t nb = mx4_blocks(K);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t blk = i >> 2;
  if (blk >= rows * nb) return;  // whole quads
  const int64_t row = blk / nb, b = blk - row * nb;
  const int q = (int)(i & 3);
  float v[8];
  mx4_load8<BF16, VEC>(x, row, K, b * MX4_BLOCK + q * 8, v);
  uint32_t m = mx4_amax8(v);
  m = max(m, (uint32_t)__shfl_xor((int)m, 1, 4));
  m = max(m, (uint32_t)__shfl_xor((int)m, 2, 4));
  const uint32_t byte = mx4_scale_byte(m);
  codes[i] = mx4_encode8(v, byte);
  if (q == 0) scales[blk] = (uint8_t)byte;
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256)
mx4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ y,
                      int64_t rows, int64_t K) {
  const int64_t nb = mx4_blocks(K);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t blk = i >> 2;
  if (blk >= rows * nb) return;
  const int64_t row = blk / nb, c0 = (blk - row * nb) * MX4_BLOCK + (i & 3) * 8;
  const uint4 d = mx4_decode8(codes[i], mx4_scale(scales[blk]));
  const uint32_t u[4] = {d.x, d.y, d.z, d.w};
  const int64_t o = row * K + c0;
  if constexpr (VEC) {
    if constexpr (BF16) {
      *(uint4*)((uint16_t*)y + o) = d;
    } else {
      float4* p = (float4*)((float*)y + o);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        p[j] = make_float4(__uint_as_float(u[2 * j] << 16), __uint_as_float(u[2 * j] & 0xffff0000u),
                           __uint_as_float(u[2 * j + 1] << 16), __uint_as_float(u[2 * j + 1] & 0xffff0000u));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + j < K) {
        const uint32_t b = j & 1 ? u[j / 2] >> 16 : u[j / 2] & 0xffffu;
        if constexpr (BF16) ((uint16_t*)y)[o + j] = (uint16_t)b;
        else ((float*)y)[o + j] = __uint_as_float(b << 16);
      }
  }
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
// Activations: A_BF16, A_F32 (hi + lo) or A_MX4 (codes and scales).
enum { A_BF16 = 0, A_F32 = 1, A_MX4 = 2 };
// What a tile's sums become: rounded to bf16, fp32, or blocks of the format.
enum { O_BF16 = 0, O_F32 = 1, O_MX4 = 2 };

struct Mx4Args {
  const void* x;           // rows of K values (A_MX4: codes, 16 bytes a block)
  const uint8_t* xs;       // A_MX4: scales
  const int32_t* row_idx;  // logical row -> x row (null: the same)
  const uint8_t* w;        // [E] [N][nb 16] codes
  const uint8_t* s;        // [E] [N][nb] scales
  const uint8_t* w2;       // SwiGLU: up's (w, s are gate's)
  const uint8_t* s2;
  void* y;                 // [rows][N] (O_MX4: codes)
  uint8_t* ys;             // O_MX4: scales
  int64_t R, K, N;
  const int32_t* seg_off;  // null: dense, R rows of one expert
  const int32_t* tile_off;
  int E;
  int xvec;                // x rows may be read 16 bytes at a time
};

// the rows of m-tile mt: its expert, first logical row and row count (uniform);
// false past the last tile
template <int BM>
__device__ __forceinline__ bool mx4_tile(const Mx4Args& p, int mt, int lane, int& e, int64_t& row0, int& rows) {
  if (!p.seg_off) {
    e = 0;
    row0 = (int64_t)mt * BM;
    rows = (int)min<int64_t>(BM, p.R - row0);
    return rows > 0;
  }
  const bool live = lane < p.E;
  const int to0 = live ? p.tile_off[lane] : 0, to1 = live ? p.tile_off[lane + 1] : 0x7fffffff;
  const int so0 = live ? p.seg_off[lane] : 0, so1 = live ? p.seg_off[lane + 1] : 0;
  if (mt >= __builtin_amdgcn_readlane(to1, p.E - 1)) return false;
  e = (int)__popcll(__ballot(to1 <= mt));
  const int r0 = __builtin_amdgcn_readlane(so0, e) + (mt - __builtin_amdgcn_readlane(to0, e)) * BM;
  row0 = r0;
  rows = min(BM, __builtin_amdgcn_readlane(so1, e) - r0);
  return rows > 0;
}

// silu(g) * u in fp32 (as the FP8 experts' epilogue)
__device__ __forceinline__ float mx4_swiglu(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-g * 1.4426950408889634f)) * u;
}

// The kernel for every shape: 64 x 64 outputs, K in steps of one block, operands
// decoded to bf16 in LDS and multiplied by v_mfma_f32_32x32x16_bf16, a quarter of
// the tile a wave.  TRANS: the sum runs over the weight's rows (the input
// gradient), x is g and the outputs are the weight's columns.
template <int AT, int OT, bool SWIGLU, bool TRANS>
__global__ void __launch_bounds__(256) mx4_tile_kernel(Mx4Args p) {
  constexpr int LD = MX4_BLOCK + 8;
  constexpr int AP = AT == A_F32 ? 2 : 1, BP = SWIGLU ? 2 : 1;
  __shared__ __attribute__((aligned(16))) uint16_t sa[AP][64 * LD];
  __shared__ __attribute__((aligned(16))) uint16_t sb[BP][64 * LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int e, rows;
  int64_t row0;
  const int n_tiles = (int)((p.N + 63) / 64);
  if (!mx4_tile<64>(p, blockIdx.x / n_tiles, lane, e, row0, rows)) return;
  const int64_t n0 = (int64_t)(blockIdx.x % n_tiles) * 64;
  // TRANS: the weight has p.K rows (the sum) of p.N columns
  const int64_t nb = mx4_blocks(TRANS ? p.N : p.K), wrows = TRANS ? p.K : p.N;
  const uint8_t* W[2] = {p.w + (int64_t)e * wrows * nb * 16, SWIGLU ? p.w2 + (int64_t)e * wrows * nb * 16 : nullptr};
  const uint8_t* S[2] = {p.s + (int64_t)e * wrows * nb, SWIGLU ? p.s2 + (int64_t)e * wrows * nb : nullptr};

  const int ar = tid >> 2, ac = (tid & 3) * 8;  // this thread's row and columns of A (and of W)
  const bool arow = ar < rows;
  const int64_t xr = arow ? (p.row_idx ? p.row_idx[row0 + ar] : row0 + ar) : 0;
  const int wm = wave >> 1, wn = wave & 1;
  f32x16_t acc[BP];
#pragma unroll
  for (int q = 0; q < BP; ++q)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[q][r] = 0.0f;

  const int64_t steps = mx4_blocks(p.K);
  for (int64_t kb = 0; kb < steps; ++kb) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    if constexpr (AT == A_MX4) {
      uint4 d = zero;
      if (arow) {
        const int64_t b = xr * steps + kb;
        d = mx4_decode8(((const uint32_t*)p.x)[b * 4 + (tid & 3)], mx4_scale(p.xs[b]));
      }
      *(uint4*)&sa[0][ar * LD + ac] = d;
    } else {
      float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      const int64_t c0 = kb * MX4_BLOCK + ac;
      if (arow) {
        if (p.xvec && c0 + 8 <= p.K) mx4_load8<AT == A_BF16, true>(p.x, xr, p.K, c0, v);
        else mx4_load8<AT == A_BF16, false>(p.x, xr, p.K, c0, v);
      }
      uint4 hi = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
      *(uint4*)&sa[0][ar * LD + ac] = hi;
      if constexpr (AT == A_F32) {
        const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w};
        uint32_t lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          lo[j] = pack_bf16(v[2 * j] - __uint_as_float(h[j] << 16),
                            v[2 * j + 1] - __uint_as_float(h[j] & 0xffff0000u));
        *(uint4*)&sa[AP - 1][ar * LD + ac] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
#pragma unroll
    for (int q = 0; q < BP; ++q) {
      uint4 d = zero;
      if constexpr (TRANS) {
        // 32 rows of the weight by 64 columns: 8 codes of a row, written column by column
        const int o = tid >> 3, c = (tid & 7) * 8;
        const int64_t wr = kb * MX4_BLOCK + o, wc = n0 + c;
        if (wr < wrows && wc < nb * MX4_BLOCK) {
          const int64_t b = wr * nb + wc / MX4_BLOCK;
          d = mx4_decode8(*(const uint32_t*)(W[q] + b * 16 + (wc % MX4_BLOCK) / 2), mx4_scale(S[q][b]));
        }
        const uint32_t u[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) sb[q][(c + j) * LD + o] = (uint16_t)(u[j / 2] >> (16 * (j & 1)));
      } else {
        if (n0 + ar < p.N) {
          const int64_t b = (n0 + ar) * nb + kb;
          d = mx4_decode8(*(const uint32_t*)(W[q] + b * 16 + ac / 2), mx4_scale(S[q][b]));
        }
        *(uint4*)&sb[q][ar * LD + ac] = d;
      }
    }
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int k = ks * 16 + (lane >> 5) * 8;
#pragma unroll
      for (int a = 0; a < AP; ++a) {
        const bf16x8_t af = *(const bf16x8_t*)&sa[a][(wm * 32 + (lane & 31)) * LD + k];
#pragma unroll
        for (int q = 0; q < BP; ++q)
          acc[q] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              af, *(const bf16x8_t*)&sb[q][(wn * 32 + (lane & 31)) * LD + k], acc[q], 0, 0, 0);
      }
    }
    __syncthreads();
  }

  // register r of lane: row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32
  const int64_t n = n0 + wn * 32 + (lane & 31);
  const int64_t onb = mx4_blocks(p.N);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = wm * 32 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
    const float v = SWIGLU ? mx4_swiglu(acc[0][r], acc[BP - 1][r]) : acc[0][r];
    const int64_t o = (row0 + row) * p.N + n;
    if constexpr (OT == O_MX4) {
      // the 32 lanes of a half hold one row's block (columns past N are zeros)
      uint32_t m = __float_as_uint(v) & 0x7fffffffu;
      for (int d = 16; d >= 1; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d, 32));
      const uint32_t byte = mx4_scale_byte(m);
      uint32_t c = byte == 255 ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v, 0.0f, mx4_scale(byte), 0) & 15u;
      c |= (uint32_t)__shfl_xor((int)c, 1, 64) << 4;  // even lanes: a byte of two codes
      const int64_t b = (row0 + row) * onb + n / MX4_BLOCK;
      if (row < rows && n / MX4_BLOCK < onb) {
        if (!(lane & 1)) ((uint8_t*)p.y)[b * 16 + (lane & 31) / 2] = (uint8_t)c;
        if ((lane & 31) == 0) p.ys[b] = (uint8_t)byte;
      }
    } else if (row < rows && n < p.N) {
      if constexpr (OT == O_BF16) ((__bf16*)p.y)[o] = (__bf16)v;
      else ((float*)p.y)[o] = v;
    }
  }
}

template <int AT, int OT, bool SWIGLU, bool TRANS>
int launch_tiles(const Mx4Args& p, int64_t m_tiles, hipStream_t stream) {
  const int64_t n_tiles = (p.N + 63) / 64;
  if (m_tiles * n_tiles > 2147483647LL) return fail(SMAUL_ERR_UNSUPPORTED, "mx4 product: too many tiles");
  hipLaunchKernelGGL((mx4_tile_kernel<AT, OT, SWIGLU, TRANS>), dim3((unsigned)(m_tiles * n_tiles)), dim3(256), 0,
                     stream, p);
  return check_launch("mx4_tile_kernel");
}

constexpr int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
bool aligned(const void* p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }
bool dtype_ok(int d) { return d == SMAUL_DTYPE_F32 || d == SMAUL_DTYPE_BF16; }

int launch_quantize(const void* x, int dtype, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t K,
                    hipStream_t stream) {
  const int64_t threads = rows * mx4_blocks(K) * 4;
  if (threads > 256LL * 2147483647LL) return fail(SMAUL_ERR_UNSUPPORTED, "mx4_quantize: too many values");
  const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
  const bool vec = K % MX4_BLOCK == 0 && aligned(x, 16), bf16 = dtype == SMAUL_DTYPE_BF16;
#define SMAUL_Q(B, V) \
  hipLaunchKernelGGL((mx4_quantize_kernel<B, V>), grid, block, 0, stream, x, (uint32_t*)codes, scales, rows, K)
  if (bf16) { if (vec) SMAUL_Q(true, true); else SMAUL_Q(true, false); }
  else { if (vec) SMAUL_Q(false, true); else SMAUL_Q(false, false); }
#undef SMAUL_Q
  return check_launch("mx4_quantize_kernel");
}

// activations with a weight: y of `out` type
int launch_linear(Mx4Args p, int at, int out, int64_t m_tiles, hipStream_t stream) {
  if (at == A_MX4)
    return out == O_BF16 ? launch_tiles<A_MX4, O_BF16, false, false>(p, m_tiles, stream)
                         : launch_tiles<A_MX4, O_F32, false, false>(p, m_tiles, stream);
  return at == A_BF16 ? launch_tiles<A_BF16, O_BF16, false, false>(p, m_tiles, stream)
                      : launch_tiles<A_F32, O_F32, false, false>(p, m_tiles, stream);
}

}  // namespace

extern "C" {

int smaul_mx4_quantize(const void* x, int dtype, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t K,
                       hipStream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || K <= 0) return fail(SMAUL_ERR_INVALID, "mx4_quantize: bad sizes or dtype");
  if (rows == 0) return SMAUL_OK;
  if (!x || !codes || !scales) return fail(SMAUL_ERR_INVALID, "mx4_quantize: null pointer");
  if (!aligned(codes, 4)) return fail(SMAUL_ERR_INVALID, "mx4_quantize: codes must be 4-byte aligned");
  return launch_quantize(x, dtype, codes, scales, rows, K, stream);
}

int smaul_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, void* y, int dtype, int64_t rows, int64_t K,
                         hipStream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || K <= 0) return fail(SMAUL_ERR_INVALID, "mx4_dequantize: bad sizes or dtype");
  if (rows == 0) return SMAUL_OK;
  if (!codes || !scales || !y) return fail(SMAUL_ERR_INVALID, "mx4_dequantize: null pointer");
  if (!aligned(codes, 4)) return fail(SMAUL_ERR_INVALID, "mx4_dequantize: codes must be 4-byte aligned");
  const int64_t threads = rows * mx4_blocks(K) * 4;
  if (threads > 256LL * 2147483647LL) return fail(SMAUL_ERR_UNSUPPORTED, "mx4_dequantize: too many values");
  const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
  const bool vec = K % MX4_BLOCK == 0 && aligned(y, 16), bf16 = dtype == SMAUL_DTYPE_BF16;
#define SMAUL_D(B, V) \
  hipLaunchKernelGGL((mx4_dequantize_kernel<B, V>), grid, block, 0, stream, (const uint32_t*)codes, scales, y, rows, K)
  if (bf16) { if (vec) SMAUL_D(true, true); else SMAUL_D(true, false); }
  else { if (vec) SMAUL_D(false, true); else SMAUL_D(false, false); }
#undef SMAUL_D
  return check_launch("mx4_dequantize_kernel");
}

int64_t smaul_mx4_linear_workspace_size(int64_t rows, int64_t in_f, int64_t out_f, int act) {
  if (rows < 0 || in_f <= 0 || out_f <= 0) return -1;
  return act == SMAUL_ACT_MX4 ? align256(rows * mx4_blocks(in_f) * 16) + align256(rows * mx4_blocks(in_f)) : 0;
}

int smaul_mx4_linear(const void* x, int dtype, const uint8_t* w, const uint8_t* s, void* y, int64_t rows,
                     int64_t in_f, int64_t out_f, int act, void* workspace, int64_t workspace_bytes,
                     hipStream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || in_f <= 0 || out_f <= 0 || (act != SMAUL_ACT_KEEP && act != SMAUL_ACT_MX4))
    return fail(SMAUL_ERR_INVALID, "mx4_linear: bad sizes, dtype or act");
  if (rows == 0) return SMAUL_OK;
  if (!x || !w || !s || !y) return fail(SMAUL_ERR_INVALID, "mx4_linear: null pointer");
  if (!aligned(w, 16)) return fail(SMAUL_ERR_INVALID, "mx4_linear: codes must be 16-byte aligned");
  const int64_t need = smaul_mx4_linear_workspace_size(rows, in_f, out_f, act);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned(workspace, 16))))
    return fail(SMAUL_ERR_INVALID, "mx4_linear: workspace %lld < %lld bytes, or unaligned", (long long)workspace_bytes,
                (long long)need);
  Mx4Args p{};
  p.x = x;
  p.w = w;
  p.s = s;
  p.y = y;
  p.R = rows;
  p.K = in_f;
  p.N = out_f;
  p.E = 1;
  const bool bf16 = dtype == SMAUL_DTYPE_BF16;
  p.xvec = aligned(x, 16) && in_f % (bf16 ? 8 : 4) == 0;
  int at = bf16 ? A_BF16 : A_F32;
  if (act == SMAUL_ACT_MX4) {
    uint8_t* codes = (uint8_t*)workspace;
    uint8_t* scales = codes + align256(rows * mx4_blocks(in_f) * 16);
    const int rc = launch_quantize(x, dtype, codes, scales, rows, in_f, stream);
    if (rc) return rc;
    p.x = codes;
    p.xs = scales;
    at = A_MX4;
  }
  return launch_linear(p, at, bf16 ? O_BF16 : O_F32, (rows + 63) / 64, stream);
}

int smaul_mx4_backward_input(const void* g, int dtype, const uint8_t* w, const uint8_t* s, void* dx, int64_t rows,
                             int64_t in_f, int64_t out_f, hipStream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || in_f <= 0 || out_f <= 0)
    return fail(SMAUL_ERR_INVALID, "mx4_backward_input: bad sizes or dtype");
  if (rows == 0) return SMAUL_OK;
  if (!g || !w || !s || !dx) return fail(SMAUL_ERR_INVALID, "mx4_backward_input: null pointer");
  if (!aligned(w, 16)) return fail(SMAUL_ERR_INVALID, "mx4_backward_input: codes must be 16-byte aligned");
  Mx4Args p{};
  p.x = g;
  p.w = w;
  p.s = s;
  p.y = dx;
  p.R = rows;
  p.K = out_f;
  p.N = in_f;
  p.E = 1;
  const bool bf16 = dtype == SMAUL_DTYPE_BF16;
  p.xvec = aligned(g, 16) && out_f % (bf16 ? 8 : 4) == 0;
  return bf16 ? launch_tiles<A_BF16, O_BF16, false, true>(p, (rows + 63) / 64, stream)
              : launch_tiles<A_F32, O_F32, false, true>(p, (rows + 63) / 64, stream);
}

// The experts' workspace, each part 256-byte aligned: the dispatch's tables and
// scratch, the rounded rows of x (act mx4), the hidden rows, the slots' outputs.
struct Mx4MoeParts {
  int64_t seg_off, tile_off, perm_row, perm_w, inv, scratch, scratch_bytes, xc, xs, hc, hs, y, total;
};
static Mx4MoeParts mx4_moe_parts(int64_t T, int64_t d, int64_t h, int64_t E, int64_t k, int dtype, int act) {
  Mx4MoeParts q{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  const int64_t size = dtype == SMAUL_DTYPE_BF16 ? 2 : 4;
  const bool mx4 = act == SMAUL_ACT_MX4;
  q.seg_off = take((E + 1) * 4);
  q.tile_off = take((E + 1) * 4);
  q.perm_row = take(T * k * 4);
  q.perm_w = take(T * k * 4);
  q.inv = take(T * k * 4);
  q.scratch_bytes = smaul_moe_dispatch_workspace_size(T, E);
  q.scratch = take(q.scratch_bytes);
  q.xc = take(mx4 ? T * mx4_blocks(d) * 16 : 0);
  q.xs = take(mx4 ? T * mx4_blocks(d) : 0);
  q.hc = take(mx4 ? T * k * mx4_blocks(h) * 16 : T * k * h * size);
  q.hs = take(mx4 ? T * k * mx4_blocks(h) : 0);
  q.y = take(T * k * d * size);
  q.total = at;
  return q;
}

int64_t smaul_mx4_moe_workspace_size(int64_t T, int64_t d, int64_t h, int64_t E, int64_t k, int dtype, int act) {
  if (T < 0 || d <= 0 || h <= 0 || E < 1 || k < 1 || !dtype_ok(dtype)) return -1;
  return mx4_moe_parts(T, d, h, E, k, dtype, act).total;
}

int smaul_mx4_moe_forward(const void* x, int dtype, const int64_t* topi, const float* topw, const uint8_t* gate_w,
                          const uint8_t* gate_s, const uint8_t* up_w, const uint8_t* up_s, const uint8_t* down_w,
                          const uint8_t* down_s, void* out, int32_t* counts, int64_t T, int64_t d, int64_t h,
                          int64_t E, int64_t k, int act, void* workspace, int64_t workspace_bytes,
                          hipStream_t stream) {
  if (!dtype_ok(dtype) || T < 0 || d <= 0 || h <= 0 || (act != SMAUL_ACT_KEEP && act != SMAUL_ACT_MX4))
    return fail(SMAUL_ERR_INVALID, "mx4_moe: bad sizes, dtype or act");
  if (E < 1 || E > 64 || k < 1 || k > E || k > 8)
    return fail(SMAUL_ERR_INVALID, "mx4_moe: need 1 <= k <= min(E, 8) and E <= 64");
  if (d % 8 != 0) return fail(SMAUL_ERR_UNSUPPORTED, "mx4_moe: d must be a multiple of 8");
  if (act == SMAUL_ACT_MX4 && dtype != SMAUL_DTYPE_BF16)
    return fail(SMAUL_ERR_UNSUPPORTED, "mx4_moe: rounded activations are for bf16 x");
  if (T * k > 2147483647LL) return fail(SMAUL_ERR_UNSUPPORTED, "mx4_moe: T * k exceeds int32");
  if (T == 0) return SMAUL_OK;
  if (!x || !topi || !topw || !gate_w || !gate_s || !up_w || !up_s || !down_w || !down_s || !out || !counts)
    return fail(SMAUL_ERR_INVALID, "mx4_moe: null pointer");
  if (!aligned(gate_w, 16) || !aligned(up_w, 16) || !aligned(down_w, 16) || !aligned(out, 16))
    return fail(SMAUL_ERR_INVALID, "mx4_moe: codes and out must be 16-byte aligned");
  const Mx4MoeParts q = mx4_moe_parts(T, d, h, E, k, dtype, act);
  if (workspace_bytes < q.total || !workspace || !aligned(workspace, 256))
    return fail(SMAUL_ERR_INVALID, "mx4_moe: workspace %lld < %lld bytes, or unaligned", (long long)workspace_bytes,
                (long long)q.total);
  char* ws = (char*)workspace;
  int32_t* seg_off = (int32_t*)(ws + q.seg_off);
  int32_t* tile_off = (int32_t*)(ws + q.tile_off);
  int32_t* perm_row = (int32_t*)(ws + q.perm_row);
  int32_t* inv = (int32_t*)(ws + q.inv);
  const bool bf16 = dtype == SMAUL_DTYPE_BF16, mx4 = act == SMAUL_ACT_MX4;
  const int64_t R = T * k, m_tiles = (R + 63) / 64 + E;
  int rc = smaul_moe_dispatch(topi, topw, counts, seg_off, tile_off, perm_row, (float*)(ws + q.perm_w), inv, T, E, k,
                              64, ws + q.scratch, q.scratch_bytes, stream);
  if (rc) return rc;
  if (mx4) {
    rc = launch_quantize(x, dtype, (uint8_t*)ws + q.xc, (uint8_t*)ws + q.xs, T, d, stream);
    if (rc) return rc;
  }
  Mx4Args p{};
  p.x = mx4 ? ws + q.xc : x;
  p.xs = mx4 ? (uint8_t*)ws + q.xs : nullptr;
  p.row_idx = perm_row;
  p.w = gate_w;
  p.s = gate_s;
  p.w2 = up_w;
  p.s2 = up_s;
  p.y = ws + q.hc;
  p.ys = mx4 ? (uint8_t*)ws + q.hs : nullptr;
  p.K = d;
  p.N = h;
  p.seg_off = seg_off;
  p.tile_off = tile_off;
  p.E = (int)E;
  p.xvec = aligned(x, 16) && d % 8 == 0;
  rc = mx4 ? launch_tiles<A_MX4, O_MX4, true, false>(p, m_tiles, stream)
           : bf16 ? launch_tiles<A_BF16, O_BF16, true, false>(p, m_tiles, stream)
                  : launch_tiles<A_F32, O_F32, true, false>(p, m_tiles, stream);
  if (rc) return rc;
  Mx4Args dn{};
  dn.x = ws + q.hc;
  dn.xs = p.ys;
  dn.w = down_w;
  dn.s = down_s;
  dn.y = ws + q.y;
  dn.K = h;
  dn.N = d;
  dn.seg_off = seg_off;
  dn.tile_off = tile_off;
  dn.E = (int)E;
  dn.xvec = h % (bf16 ? 8 : 4) == 0;
  rc = launch_linear(dn, mx4 ? A_MX4 : bf16 ? A_BF16 : A_F32, bf16 ? O_BF16 : O_F32, m_tiles, stream);
  if (rc) return rc;
  return smaul_moe_combine(ws + q.y, dtype, topi, topw, inv, out, T, d, k, stream);
}

}  // extern "C"
