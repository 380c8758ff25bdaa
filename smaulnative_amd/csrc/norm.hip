// norm.hip -- the residual's addition, the root-mean-square norm of the sum and its
// output as rows or in blocks of 8-bit codes, and that norm's gradients (gfx950).
//
//   s = round(x + r), y = s / rms(s) * w, rms(s) = sqrt(mean(s^2) + eps)
//   dx = ds + (w dy - s (sum(w dy s) / d) / rms^2) / rms,   dw = sum over rows of dy s / rms
#include <cmath>

#include "fp8_block.h"

using smaul::check_launch;
using smaul::fail;
using smaul::grid_fits;

namespace {

// the sum over a row's NW waves, in each of their lanes (red: NW floats of the row's own)
template <int NW>
__device__ __forceinline__ float row_sum(float v, float* red, int wave) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  if constexpr (NW > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w];
  }
  return v;
}

__device__ __forceinline__ float inv_rms(float ss, int64_t d, float eps) {
  return 1.0f / __fsqrt_rn(ss / (float)d + eps);
}

// A row is NW waves', a lane has 8 values of every NW * 512, the first CH of them kept in
// registers (the rest are read again).
template <bool BF16, bool CODES, int NW, int CH>
__global__ void __launch_bounds__(256)
add_rms_norm_kernel(const void* __restrict__ x, const void* __restrict__ r, const float* __restrict__ weight,
                    void* __restrict__ sum, void* __restrict__ out, uint8_t* __restrict__ scales, int64_t T, int64_t d,
                    float eps) {
  constexpr int ROWS = 4 / NW;
  __shared__ float red[4];
  const int lane = threadIdx.x & 63, w4 = threadIdx.x >> 6, wave = w4 % NW;
  const int64_t t = (int64_t)blockIdx.x * ROWS + w4 / NW;
  if (NW == 1 && t >= T) return;  // a workgroup of more waves has one row
  const int64_t nb = fb_blocks(d), chunks = nb * 16;
  float keep[CH][8];
  // s of the chunk that begins at column c, and what is stored of it
  auto load = [&](int64_t c, float (&v)[8]) {
    fb_load8<BF16>(x, t, d, c, v);
    if (r) {
      float q[8];
      fb_load8<BF16>(r, t, d, c, q);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = BF16 ? (float)(__bf16)(v[j] + q[j]) : v[j] + q[j];
    }
  };
  float ss = 0.0f;
  auto add = [&](int64_t c, const float (&v)[8]) {
    if (r && c < d) fb_store8<BF16>(sum, t, d, c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
  };
  auto chunk = [&](int i) -> int64_t { return (int64_t)i * (NW * 64) + wave * 64 + lane; };
#pragma unroll
  for (int i = 0; i < CH; ++i) load(chunk(i) * 8, keep[i]);
#pragma unroll
  for (int i = 0; i < CH; ++i) add(chunk(i) * 8, keep[i]);
  for (int i = CH; chunk(i) - lane < chunks; ++i) {
    float v[8];
    load(chunk(i) * 8, v);
    add(chunk(i) * 8, v);
  }
  const float rstd = inv_rms(row_sum<NW>(ss, red, wave), d, eps);
  auto put = [&](int64_t c, float (&v)[8]) {  // whole blocks of lanes
    if (c >= chunks * 8) return;
    float wv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) wv[j] = 1.0f;
    if (weight) fb_load8<false>(weight, 0, d, c, wv);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * rstd * wv[j];
    if constexpr (CODES) fb_write8((uint8_t*)out, scales, t, nb, c / 8, v);
    else if (c < d) fb_store8<BF16>(out, t, d, c, v);
  };
#pragma unroll
  for (int i = 0; i < CH; ++i) put(chunk(i) * 8, keep[i]);
  for (int i = CH; chunk(i) - lane < chunks; ++i) {
    float v[8];
    load(chunk(i) * 8, v);
    put(chunk(i) * 8, v);
  }
}

// Rows blockIdx.x, + gridDim.x, ...: a workgroup's share of dw stays in registers until
// its rows are done.  Columns from CH * 2048 on take another pass of the kernel's loop
// for their part of dw (col0).
template <bool BF16, int CH>
__global__ void __launch_bounds__(256)
add_rms_norm_backward_kernel(const void* __restrict__ dy, const void* __restrict__ s, const void* __restrict__ ds,
                             const float* __restrict__ weight, void* __restrict__ dx, float* __restrict__ part,
                             int64_t T, int64_t d, float eps) {
  __shared__ float red[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t chunks = (d + 7) / 8;
  for (int64_t c0 = 0; c0 < chunks; c0 += CH * 256) {  // of dw's columns
    float acc[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = 0.0f;
    for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
      float ss = 0.0f, sd = 0.0f;
      for (int64_t c = threadIdx.x; c < chunks; c += 256) {
        float v[8], g[8], w[8];
        fb_load8<BF16>(s, t, d, c * 8, v);
        fb_load8<BF16>(dy, t, d, c * 8, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 1.0f;
        if (weight) fb_load8<false>(weight, 0, d, c * 8, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ss = fmaf(v[j], v[j], ss);
          sd = fmaf(w[j] * g[j], v[j], sd);
        }
      }
      const float rstd = inv_rms(row_sum<4>(ss, red, wave), d, eps);
      const float dot = row_sum<4>(sd, red, wave) / (float)d * rstd * rstd;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int64_t c = c0 + i * 256 + threadIdx.x;
        if (c < chunks) {
          float v[8], g[8];
          fb_load8<BF16>(s, t, d, c * 8, v);
          fb_load8<BF16>(dy, t, d, c * 8, g);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(g[j], v[j] * rstd, acc[i][j]);
        }
      }
      for (int64_t c = threadIdx.x; c0 == 0 && c < chunks; c += 256) {
        float v[8], g[8], w[8], o[8];
        fb_load8<BF16>(s, t, d, c * 8, v);
        fb_load8<BF16>(dy, t, d, c * 8, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          w[j] = 1.0f;
          o[j] = 0.0f;
        }
        if (weight) fb_load8<false>(weight, 0, d, c * 8, w);
        if (ds) fb_load8<BF16>(ds, t, d, c * 8, o);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += (w[j] * g[j] - v[j] * dot) * rstd;
        fb_store8<BF16>(dx, t, d, c * 8, o);
      }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int64_t c = c0 + i * 256 + threadIdx.x;
      if (part && c < chunks) fb_store8<false>(part, blockIdx.x, d, c * 8, acc[i]);
    }
  }
}

// dw: the workgroups' parts, in their order
__global__ void __launch_bounds__(256)
norm_weight_sum_kernel(const float* __restrict__ part, float* __restrict__ dw, int parts, int64_t d) {
  __shared__ float sh[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float a = 0.0f;
  if (c < d)
    for (int p = wave; p < parts; p += 4) a += part[p * d + c];
  sh[wave][lane] = a;
  __syncthreads();
  if (wave == 0 && c < d) dw[c] = sh[0][lane] + sh[1][lane] + sh[2][lane] + sh[3][lane];
}

int norm_parts(int64_t T) { return (int)(T < 512 ? T : 512); }

}  // namespace

extern "C" {

int smaul_add_rms_norm(const void* x, const void* residual, int dtype, const float* weight, float eps, void* sum,
                       void* out, uint8_t* scales, int64_t T, int64_t d, hipStream_t stream) {
  if (!fb_dtype_ok(dtype) || T < 0 || d <= 0) return fail(SMAUL_ERR_INVALID, "add_rms_norm: bad sizes or dtype");
  if (!(eps > 0.0f) || !std::isfinite(eps)) return fail(SMAUL_ERR_INVALID, "add_rms_norm: eps must be positive finite");
  if (T == 0) return SMAUL_OK;
  if (!x || !out || (residual && !sum)) return fail(SMAUL_ERR_INVALID, "add_rms_norm: null pointer");
  if (scales && !fb_aligned(out, 8)) return fail(SMAUL_ERR_INVALID, "add_rms_norm: codes must be 8-byte aligned");
  const bool bf16 = dtype == SMAUL_DTYPE_BF16;
  const int64_t blocks = d <= 2048 ? (T + 3) / 4 : T;
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "add_rms_norm: too many rows");
  const dim3 grid((unsigned)blocks), block(256);
#define SMAUL_N(B, C, NW) \
  hipLaunchKernelGGL((add_rms_norm_kernel<B, C, NW, 4>), grid, block, 0, stream, x, residual, weight, sum, out, scales, \
                     T, d, eps)
  if (d <= 2048) {
    if (bf16 && scales) SMAUL_N(true, true, 1);
    else if (bf16) SMAUL_N(true, false, 1);
    else if (scales) SMAUL_N(false, true, 1);
    else SMAUL_N(false, false, 1);
  } else {
    if (bf16 && scales) SMAUL_N(true, true, 4);
    else if (bf16) SMAUL_N(true, false, 4);
    else if (scales) SMAUL_N(false, true, 4);
    else SMAUL_N(false, false, 4);
  }
#undef SMAUL_N
  return check_launch("add_rms_norm_kernel");
}

int64_t smaul_add_rms_norm_backward_workspace_size(int64_t T, int64_t d) {
  if (T < 0 || d <= 0) return -1;
  return norm_parts(T) * d * 4;
}

int smaul_add_rms_norm_backward(const void* dy, const void* s, const void* ds, int dtype, const float* weight,
                                float eps, void* dx, float* dw, int64_t T, int64_t d, void* workspace,
                                int64_t workspace_bytes, hipStream_t stream) {
  if (!fb_dtype_ok(dtype) || T < 0 || d <= 0)
    return fail(SMAUL_ERR_INVALID, "add_rms_norm_backward: bad sizes or dtype");
  if (!(eps > 0.0f) || !std::isfinite(eps))
    return fail(SMAUL_ERR_INVALID, "add_rms_norm_backward: eps must be positive finite");
  if (T == 0 && !dw) return SMAUL_OK;
  if (T > 0 && (!dy || !s || !dx)) return fail(SMAUL_ERR_INVALID, "add_rms_norm_backward: null pointer");
  const int64_t need = dw ? smaul_add_rms_norm_backward_workspace_size(T, d) : 0;
  if (workspace_bytes < need || (need > 0 && (!workspace || !fb_aligned(workspace, 256))))
    return fail(SMAUL_ERR_INVALID, "add_rms_norm_backward: workspace %lld < %lld bytes, or unaligned",
                (long long)workspace_bytes, (long long)need);
  if (!grid_fits((d + 63) / 64, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "add_rms_norm_backward: rows too wide");
  const int parts = norm_parts(T);
  float* part = dw ? (float*)workspace : nullptr;
  if (T > 0) {
    auto* kernel = dtype == SMAUL_DTYPE_BF16 ? &add_rms_norm_backward_kernel<true, 4>
                                             : &add_rms_norm_backward_kernel<false, 4>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)parts), dim3(256), 0, stream, dy, s, ds, weight, dx, part, T, d, eps);
    if (int rc = check_launch("add_rms_norm_backward_kernel")) return rc;
  }
  if (!dw) return SMAUL_OK;
  hipLaunchKernelGGL(norm_weight_sum_kernel, dim3((unsigned)((d + 63) / 64)), dim3(256), 0, stream, part, dw, parts, d);
  return check_launch("norm_weight_sum_kernel");
}

}  // extern "C"
