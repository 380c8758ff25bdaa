// norm.hip -- the residual's addition, the root-mean-square norm of the sum and its
// output as rows or in blocks of 8-bit codes, and that norm's gradients (gfx950).
//
//   s = round(x + r), y = s / rms(s) * w, rms(s) = sqrt(mean(s^2) + eps)
//   dx = ds + (w dy - s (sum(w dy s) / d) / rms^2) / rms,   dw = sum over rows of dy s / rms
#include <cmath>

#include "fp8_block.h"

using smaul::check_launch;
using smaul::cu_count;
using smaul::fail;
using smaul::grid_fits;

namespace {

// The sum over a row's NW waves, in each of their lanes (red: NW values of the row's own).
template <int NW>
__device__ __forceinline__ double row_sum(double v, double* red, int wave) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  if constexpr (NW > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w];
  }
  return v;
}

// 1 / sqrt(m): the 32-bit root with one step of Newton in 64
__device__ __forceinline__ double inv_root(double m) {
  if (!(m > 1e-30 && m < 1e30)) return 1.0 / sqrt(m);
  const double r = (double)__builtin_amdgcn_rsqf((float)m);
  return r * (1.5 - 0.5 * m * r * r);
}

// (as fp32 it keeps 22 bits for the largest rms there is, 3.4e38: no scaling, which would cost
// the forward pass 2 us of 92 by a product a value, 13 by a branch)
__device__ __forceinline__ double row_root(double ss, int64_t d, float eps) { return inv_root(ss / (double)d + (double)eps); }

// of 8 values, in 64 bits
__device__ __forceinline__ double sum_squares(const float (&v)[8]) {
  double a = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = fma((double)v[j], (double)v[j], a);
  return a;
}
__device__ __forceinline__ double sum_products(const float (&w)[8], const float (&g)[8], const float (&v)[8]) {
  double a = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = fma((double)(w[j] * g[j]), (double)v[j], a);
  return a;
}

// A row is NW waves', a lane has 8 values of every NW * 512, the first CH of them kept in
// registers (the rest are read again).  Memory bounds it: 32768 x 2048 bf16 to codes 99 us, 4.8
// TB/s, to rows 94.
//
// The squares, their sum and the root are in 64 bits (in 32, rows past 1.8e19 would overflow;
// 1 % of the time, 4 of the gradients'), and the two products with 1 / rms and the weight carry
// their errors along (1 / rms as two floats).  Towards codes y is rounded to odd, so that one
// that fp32 would round to the middle of two codes goes to its own side of it: a code is the
// neighbouring one of what 64 bits give once in 30 million (2 % of the time; y to nearest once
// in 2 million, in 32 bits throughout in 250000).
template <bool BF16, bool CODES, bool NT, int NW, int CH>
__global__ void __launch_bounds__(256)
add_rms_norm_kernel(const void* __restrict__ x, const void* __restrict__ r, const float* __restrict__ weight,
                    void* __restrict__ sum, void* __restrict__ out, uint8_t* __restrict__ scales, int64_t T, int64_t d,
                    float eps) {
  constexpr int ROWS = 4 / NW;
  __shared__ double red[4];
  const int lane = threadIdx.x & 63, w4 = threadIdx.x >> 6, wave = w4 % NW;
  const int64_t t = (int64_t)blockIdx.x * ROWS + w4 / NW;
  if (NW == 1 && t >= T) return;  // a workgroup of more waves has one row
  const int64_t nb = fb_blocks(d), chunks = nb * 16;
  float keep[CH][8], extra[CH][8];
  auto chunk = [&](int i) -> int64_t { return (int64_t)i * (NW * 64) + wave * 64 + lane; };
  double ss = 0.0;
  // s of the chunk that begins at column c
  auto add = [&](int64_t c, float (&v)[8], const float (&q)[8]) {
    if (r) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = BF16 ? (float)(__bf16)(v[j] + q[j]) : v[j] + q[j];
    }
  };
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    fb_load8<BF16, NT>(x, t, d, chunk(i) * 8, keep[i]);
    if (r) fb_load8<BF16, NT>(r, t, d, chunk(i) * 8, extra[i]);
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    add(chunk(i) * 8, keep[i], extra[i]);
    if (r && chunk(i) * 8 < d) fb_store8<BF16, NT>(sum, t, d, chunk(i) * 8, keep[i]);
    ss += sum_squares(keep[i]);
  }
  for (int i = CH; chunk(i) - lane < chunks; ++i) {
    float v[8], q[8];
    fb_load8<BF16, NT>(x, t, d, chunk(i) * 8, v);
    if (r) fb_load8<BF16, NT>(r, t, d, chunk(i) * 8, q);
    add(chunk(i) * 8, v, q);
    if (r && chunk(i) * 8 < d) fb_store8<BF16, NT>(sum, t, d, chunk(i) * 8, v);
    ss += sum_squares(v);
  }
  const double root = row_root(row_sum<NW>(ss, red, wave), d, eps);
  const float rh = (float)root, rl = (float)(root - (double)rh);
  auto put = [&](int64_t c, float (&v)[8]) {  // whole blocks of lanes
    if (c >= chunks * 8) return;
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 1.0f;
    if (weight) fb_load8<false>(weight, 0, d, c, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = v[j] * rh, ae = fmaf(v[j], rl, fmaf(v[j], rh, -a));
      const float y = a * w[j], ye = fmaf(ae, w[j], fmaf(a, w[j], -y));
      if constexpr (CODES) {
        const int less = (int)__float_as_uint(fmaf(ye, y, 0.0f)) >> 31;  // -1: |y + ye| < |y| (never of 0)
        v[j] = __uint_as_float((__float_as_uint(y) + (uint32_t)less) | 1u);
      } else {
        const float z = y + ye;
        v[j] = z == z ? z : y;  // an infinity has no error to carry
      }
    }
    // (an infinity less one is fp32's largest)
    if constexpr (CODES) fb_write8((uint8_t*)out, scales, t, nb, c / 8, v, 0x7f7fffffu);
    else if (c < d) fb_store8<BF16, NT>(out, t, d, c, v);
  };
#pragma unroll
  for (int i = 0; i < CH; ++i) put(chunk(i) * 8, keep[i]);
  for (int i = CH; chunk(i) - lane < chunks; ++i) {
    float v[8], q[8];
    fb_load8<BF16, NT>(x, t, d, chunk(i) * 8, v);
    if (r) fb_load8<BF16, NT>(r, t, d, chunk(i) * 8, q);
    add(chunk(i) * 8, v, q);
    put(chunk(i) * 8, v);
  }
}

// One pass over the rows: a row's values and gradients stay in registers between its two
// sums and dx, the next row's are on their way meanwhile, and a workgroup's share of dw
// stays until its rows (blockIdx.x * ROWS, + gridDim.x * ROWS, ...) are done;
// norm_weight_sum_kernel adds the shares in their order.  d is no more than NW * CH * 512.
// Memory bounds it: 16384 x 2048 bf16 57 us, 4.7 TB/s (50 without dw; 178 with the rows read again).
template <bool BF16, int NW, int CH>
__global__ void __launch_bounds__(256)
add_rms_norm_backward_kernel(const void* __restrict__ dy, const void* __restrict__ s, const void* __restrict__ ds,
                             const float* __restrict__ weight, void* __restrict__ dx, float* __restrict__ part,
                             int64_t T, int64_t d, float eps) {
  constexpr int ROWS = 4 / NW;
  __shared__ double red[2][8];
  __shared__ float share[NW < 4 ? 4 * 512 : 1];
  const int lane = threadIdx.x & 63, w4 = threadIdx.x >> 6, wave = w4 % NW, first = w4 - wave;
  auto col = [&](int i) -> int64_t { return ((int64_t)i * (NW * 64) + wave * 64 + lane) * 8; };
  float w[CH][8], acc[CH][8], v[CH][8], g[CH][8], o[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[i][j] = 1.0f;
      acc[i][j] = 0.0f;
      o[i][j] = 0.0f;
    }
  if (weight) {
#pragma unroll
    for (int i = 0; i < CH; ++i) fb_load8<false>(weight, 0, d, col(i), w[i]);
  }
  auto load = [&](int64_t t, float (&a)[CH][8], float (&b)[CH][8], float (&c)[CH][8]) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      fb_load8<BF16>(s, t, d, col(i), a[i]);
      fb_load8<BF16>(dy, t, d, col(i), b[i]);
      if (ds) fb_load8<BF16>(ds, t, d, col(i), c[i]);
    }
  };
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t t = (int64_t)blockIdx.x * ROWS + w4 / NW;
  if (t < T) load(t, v, g, o);
  int turn = 0;
  for (int64_t t0 = (int64_t)blockIdx.x * ROWS; t0 < T; t0 += step, t += step, turn ^= 1) {  // of the whole workgroup
    float v2[CH][8], g2[CH][8], o2[CH][8];
    if (t + step < T) load(t + step, v2, g2, o2);
    double ss = 0.0, sd = 0.0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      ss += sum_squares(v[i]);
      sd += sum_products(w[i], g[i], v[i]);
    }
#pragma unroll
    for (int q = 32; q >= 1; q >>= 1) {
      ss += __shfl_xor(ss, q, 64);
      sd += __shfl_xor(sd, q, 64);
    }
    if constexpr (NW > 1) {  // two places by turns: one barrier a row
      if (lane == 0) {
        red[turn][w4] = ss;
        red[turn][4 + w4] = sd;
      }
      __syncthreads();
      ss = sd = 0.0;
#pragma unroll
      for (int q = 0; q < NW; ++q) {
        ss += red[turn][first + q];
        sd += red[turn][4 + first + q];
      }
    }
    if (t >= T) continue;  // a last row that is not there
    const double root = row_root(ss, d, eps);
    const float rstd = (float)root, dot = (float)(sd / (double)d * root * root);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[i][j] = fmaf(g[i][j], v[i][j] * rstd, acc[i][j]);
        o[i][j] += (w[i][j] * g[i][j] - v[i][j] * dot) * rstd;
      }
      if (col(i) < d) fb_store8<BF16>(dx, t, d, col(i), o[i]);
    }
    if (t + step < T) {
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[i][j] = v2[i][j];
          g[i][j] = g2[i][j];
          o[i][j] = ds ? o2[i][j] : 0.0f;
        }
    }
  }
  if (!part) return;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if constexpr (NW < 4) {  // its rows' waves
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) share[w4 * 512 + j * 64 + lane] = acc[i][j];
      __syncthreads();
      if (first == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float a = 0.0f;
#pragma unroll
          for (int q = 0; q < ROWS; ++q) a += share[(q * NW + wave) * 512 + j * 64 + lane];
          acc[i][j] = a;
        }
        if (col(i) < d) fb_store8<false>(part, blockIdx.x, d, col(i), acc[i]);
      }
    } else if (col(i) < d) {
      fb_store8<false>(part, blockIdx.x, d, col(i), acc[i]);
    }
  }
}

// Rows of any width: read again for dx, and for every CH * 2048 columns of dw.
template <bool BF16, int CH>
__global__ void __launch_bounds__(256)
add_rms_norm_backward_wide_kernel(const void* __restrict__ dy, const void* __restrict__ s, const void* __restrict__ ds,
                                  const float* __restrict__ weight, void* __restrict__ dx, float* __restrict__ part,
                                  int64_t T, int64_t d, float eps) {
  __shared__ double red[4];
  const int wave = threadIdx.x >> 6;
  const int64_t chunks = (d + 7) / 8;
  for (int64_t c0 = 0; c0 < (part ? chunks : 1); c0 += CH * 256) {  // of dw's columns, the first with dx
    float acc[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = 0.0f;
    for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
      double ss = 0.0, sd = 0.0;
      for (int64_t c = threadIdx.x; c < chunks; c += 256) {
        float v[8], g[8], w[8];
        fb_load8<BF16>(s, t, d, c * 8, v);
        fb_load8<BF16>(dy, t, d, c * 8, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 1.0f;
        if (weight) fb_load8<false>(weight, 0, d, c * 8, w);
        ss += sum_squares(v);
        sd += sum_products(w, g, v);
      }
      const double root = row_root(row_sum<4>(ss, red, wave), d, eps);
      const float rstd = (float)root, dot = (float)(row_sum<4>(sd, red, wave) / (double)d * root * root);
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

// dw: the workgroups' parts, 32 of them at a time, in their order
__global__ void __launch_bounds__(1024)
norm_weight_sum_kernel(const float* __restrict__ part, float* __restrict__ dw, int parts, int64_t d) {
  __shared__ float sh[32][33];
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + col;
  float a = 0.0f;
  if (c < d) {
#pragma unroll 8
    for (int p = row; p < parts; p += 32) a += part[p * d + c];
  }
  sh[row][col] = a;
  __syncthreads();
  if (row == 0 && c < d) {
    float t = 0.0f;
#pragma unroll
    for (int r = 0; r < 32; ++r) t += sh[r][col];
    dw[c] = t;
  }
}

// workgroups of the backward pass, each with a part of dw: as many as run, four a CU, of 2049
// to 4096 columns two (16384 x 2048 62 us, of two a CU 82, of eight 68; 8192 x 4096 78, of four 90)
int64_t norm_parts(int64_t T, int64_t d) {
  const int64_t rows = d <= 512 ? (T + 3) / 4 : d <= 1024 ? (T + 1) / 2 : T;
  const int64_t most = (d > 2048 && d <= 4096 ? 2 : 4) * (int64_t)cu_count();
  return rows < most ? rows : most;
}

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
  // rows past the caches (32768 x 2048 bf16 93 us for 100 by way of them)
  const bool nt = T * d * (bf16 ? 2 : 4) >= FB_NT_BYTES;
  // a workgroup a row from 2048 columns on, and for so few rows that a wave a row would
  // leave most of the chip idle (250 x 2048 3.6 us for 6.4, 64 x 1024 3.5 for 4.1)
  const bool wide = d > 2048 || T <= cu_count();
  const int64_t blocks = wide ? T : (T + 3) / 4;
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "add_rms_norm: too many rows");
#define SMAUL_N(B, C, N)                                                                                             \
  do {                                                                                                               \
    auto* kernel = wide ? (d <= 2048 ? &add_rms_norm_kernel<B, C, false, 4, 1> : &add_rms_norm_kernel<B, C, N, 4, 4>) \
                   : d <= 512  ? &add_rms_norm_kernel<B, C, N, 1, 1>                                                  \
                   : d <= 1024 ? &add_rms_norm_kernel<B, C, N, 1, 2>                                                  \
                               : &add_rms_norm_kernel<B, C, N, 1, 4>;                                                 \
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, x, residual, weight, sum, out, scales,  \
                       T, d, eps);                                                                                   \
  } while (0)
#define SMAUL_NT(B, C)           \
  do {                           \
    if (nt) SMAUL_N(B, C, true); \
    else SMAUL_N(B, C, false);   \
  } while (0)
  if (bf16 && scales) SMAUL_NT(true, true);
  else if (bf16) SMAUL_NT(true, false);
  else if (scales) SMAUL_NT(false, true);
  else SMAUL_NT(false, false);
#undef SMAUL_NT
#undef SMAUL_N
  return check_launch("add_rms_norm_kernel");
}

int64_t smaul_add_rms_norm_backward_workspace_size(int64_t T, int64_t d) {
  if (T < 0 || d <= 0) return -1;
  return norm_parts(T, d) * d * 4;
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
  if (!grid_fits((d + 31) / 32, 1024)) return fail(SMAUL_ERR_UNSUPPORTED, "add_rms_norm_backward: rows too wide");
  const int parts = (int)norm_parts(T, d);
  float* part = dw ? (float*)workspace : nullptr;
  if (T > 0) {
    const bool bf16 = dtype == SMAUL_DTYPE_BF16;
    auto* kernel = bf16 ? &add_rms_norm_backward_wide_kernel<true, 4> : &add_rms_norm_backward_wide_kernel<false, 4>;
#define SMAUL_B(NW, CH) \
  kernel = bf16 ? &add_rms_norm_backward_kernel<true, NW, CH> : &add_rms_norm_backward_kernel<false, NW, CH>
    if (d <= 512) SMAUL_B(1, 1);
    else if (d <= 1024) SMAUL_B(2, 1);
    else if (d <= 2048) SMAUL_B(4, 1);
    else if (d <= 4096) SMAUL_B(4, 2);
#undef SMAUL_B
    hipLaunchKernelGGL(kernel, dim3((unsigned)parts), dim3(256), 0, stream, dy, s, ds, weight, dx, part, T, d, eps);
    if (int rc = check_launch("add_rms_norm_backward_kernel")) return rc;
  }
  if (!dw) return SMAUL_OK;
  hipLaunchKernelGGL(norm_weight_sum_kernel, dim3((unsigned)((d + 31) / 32)), dim3(1024), 0, stream, part, dw, parts, d);
  return check_launch("norm_weight_sum_kernel");
}

}  // extern "C"
