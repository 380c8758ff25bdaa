// fp8_block.hip -- rows in blocks of 128 E4M3 codes on MI355X (gfx950): quantisation,
// the product of such rows with such a weight, its input gradient, and the gated
// feed-forward block with its gradients.
//
//   y[r, n]  = sum_k x[r, k] W[n, k]
//   dx[r, k] = sum_n g[r, n] W[n, k]
//   block:   h = Q(silu(x Wg^T) * (x Wu^T)),  y = h Wd^T
//   its gradients, straight through the roundings: dh = dy Wd, dg = dh u silu'(g),
//   du = dh silu(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
#include "fp8_block.h"

using smaul::check_launch;
using smaul::cu_count;
using smaul::fail;
using smaul::grid_fits;

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------
// quantisation: 16 lanes a block, 8 values a lane
// ---------------------------------------------------------------------------
template <bool BF16>
__global__ void __launch_bounds__(256)
fb_quantize_kernel(const void* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t rows,
                   int64_t K) {
  const int64_t nb = fb_blocks(K), i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (nb * 16), c = i - row * nb * 16;
  if (row >= rows) return;  // whole blocks
  float v[8];
  fb_load8<BF16>(x, row, K, c * 8, v);
  fb_write8(codes, scales, row, nb, c, v);
}

template <bool BF16>
__global__ void __launch_bounds__(256)
fb_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ y,
                     int64_t rows, int64_t K) {
  const int64_t nb = fb_blocks(K), i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (nb * 16), c = i - row * nb * 16;
  if (row >= rows || c * 8 >= K) return;
  const uint2 w = *(const uint2*)(codes + row * nb * FB_BLOCK + c * 8);
  const float s = fb_scale(scales[row * ((nb + 3) / 4 * 4) + c / 16]);
  float v[8];
  fb_decode4(w.x, s, v);
  fb_decode4(w.y, s, v + 4);
  fb_store8<BF16>(y, row, K, c * 8, v);
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
enum { F_F32 = 0, F_BF16 = 1, F_CODES = 2 };

// a matrix of rows of ld values (codes: with scales of ld / 128 blocks), or with
// `turned` its transpose
struct FbMat {
  const void* p;
  const uint8_t* s;
  int64_t ld;
  int fmt, turned;
};

__device__ __forceinline__ float fb_at(const FbMat& m, int64_t r, int64_t c) {
  if (m.turned) {
    const int64_t t = r;
    r = c;
    c = t;
  }
  const int64_t i = r * m.ld + c;
  if (m.fmt == F_F32) return ((const float*)m.p)[i];
  if (m.fmt == F_BF16) return bf2f(((const uint16_t*)m.p)[i]);
  const uint32_t code = ((const uint8_t*)m.p)[i];
  float v[4];
  fb_decode4(code, fb_scale(m.s[r * ((m.ld / FB_BLOCK + 3) / 4 * 4) + c / FB_BLOCK]), v);
  return v[0];
}

struct FbProduct {
  FbMat a[2], b[2];  // c = a[0] b[0]^T + a[1] b[1]^T (pairs of them)
  int pairs, bf16;   // c's type
  void* c;
  int64_t M, N, K, ldc;
};

// 64 x 64 outputs a workgroup, in fp32
__global__ void __launch_bounds__(256) fb_product_kernel(FbProduct p) {
  __shared__ float sa[16][66], sb[16][66];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5, l32 = lane & 31;
  const int64_t nt = (p.N + 63) / 64, m0 = (int64_t)blockIdx.x / nt * 64, n0 = (int64_t)blockIdx.x % nt * 64;
  const int wm = wave >> 1, wn = wave & 1;
  f32x16_t acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
  for (int q = 0; q < p.pairs; ++q)
    for (int64_t k0 = 0; k0 < p.K; k0 += 16) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = j * 256 + tid, r = i >> 4, k = i & 15;
        const bool in = k0 + k < p.K;
        sa[k][r] = in && m0 + r < p.M ? fb_at(p.a[q], m0 + r, k0 + k) : 0.0f;
        sb[k][r] = in && n0 + r < p.N ? fb_at(p.b[q], n0 + r, k0 + k) : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; k += 2)
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(sa[k + g][wm * 32 + l32], sb[k + g][wn * 32 + l32], acc, 0, 0, 0);
    }
  const int64_t n = n0 + wn * 32 + l32;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t m = m0 + wm * 32 + (r & 3) + 8 * (r >> 2) + 4 * g;
    if (m < p.M && n < p.N) {
      if (p.bf16) ((__bf16*)p.c)[m * p.ldc + n] = (__bf16)acc[r];
      else ((float*)p.c)[m * p.ldc + n] = acc[r];
    }
  }
}

int launch_product(const FbProduct& p, hipStream_t stream) {
  const int64_t blocks = (p.M + 63) / 64 * ((p.N + 63) / 64);
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block product: too many tiles");
  hipLaunchKernelGGL(fb_product_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p);
  return check_launch("fb_product_kernel");
}

// gate's and up's sums [T, h] -> the hidden rows' codes and, to keep, u silu'(g) and
// silu(g) in their place
__global__ void __launch_bounds__(256)
fb_gated_kernel(float* __restrict__ g, float* __restrict__ u, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                int64_t T, int64_t h, int keep) {
  const int64_t nb = fb_blocks(h), i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (nb * 16), c = i - row * nb * 16;
  if (row >= T) return;
  float a[8], b[8], v[8];
  fb_load8<false>(g, row, h, c * 8, a);
  fb_load8<false>(u, row, h, c * 8, b);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float sig = 1.0f / (1.0f + expf(-a[j])), si = a[j] * sig;
    v[j] = si * b[j];
    a[j] = b[j] * sig * (1.0f + a[j] * (1.0f - sig));
    b[j] = si;
  }
  fb_write8(codes, scales, row, nb, c, v);
  if (keep && c * 8 < h) {
    fb_store8<false>(g, row, h, c * 8, a);
    fb_store8<false>(u, row, h, c * 8, b);
  }
}

// dh -> dg and du, by the factors that the forward pass kept
__global__ void __launch_bounds__(256)
fb_gated_backward_kernel(const float* __restrict__ dh, const float* __restrict__ a, const float* __restrict__ b,
                         float* __restrict__ dg, float* __restrict__ du, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  dg[i] = dh[i] * a[i];
  du[i] = dh[i] * b[i];
}

// a workspace laid out part by part
struct Parts {
  int64_t at = 0;
  int64_t take(int64_t bytes) {
    const int64_t here = at;
    at += fb_align256(bytes);
    return here;
  }
};

bool x_ok(int d) { return fb_dtype_ok(d) || d == SMAUL_DTYPE_FP8_BLOCK; }

int launch_quantize(const void* x, int dtype, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t K,
                    hipStream_t stream) {
  const int64_t blocks = (rows * fb_blocks(K) * 16 + 255) / 256;
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block_quantize: too many values");
  auto* kernel = dtype == SMAUL_DTYPE_BF16 ? &fb_quantize_kernel<true> : &fb_quantize_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, x, codes, scales, rows, K);
  return check_launch("fb_quantize_kernel");
}

struct FfnParts {
  int64_t xc, xs, hc, hs, keep, total;
};
// what the caller keeps for the gradients stands in `saved` (save), the rest in the workspace
FfnParts ffn_parts(int64_t T, int64_t d, int64_t h, int x_dtype, bool save) {
  FfnParts q{};
  Parts w;
  const bool rows = x_dtype != SMAUL_DTYPE_FP8_BLOCK && !save;
  q.xc = w.take(rows ? T * fb_width(d) : 0);
  q.xs = w.take(rows ? T * fb_words(d) * 4 : 0);
  q.hc = w.take(save ? 0 : T * fb_width(h));
  q.hs = w.take(save ? 0 : T * fb_words(h) * 4);
  q.keep = w.take(save ? 0 : T * h * 8);
  q.total = w.at;
  return q;
}

struct FfnBackParts {
  int64_t dh, dg, du, total;
};
FfnBackParts ffn_back_parts(int64_t T, int64_t h) {
  FfnBackParts q{};
  Parts w;
  q.dh = w.take(T * h * 4);
  q.dg = w.take(T * h * 4);
  q.du = w.take(T * h * 4);
  q.total = w.at;
  return q;
}

FbMat codes_mat(const void* p, const uint8_t* s, int64_t K, int turned = 0) {
  return FbMat{p, s, fb_width(K), F_CODES, turned};
}
FbMat float_mat(const void* p, int64_t ld, int fmt, int turned = 0) { return FbMat{p, nullptr, ld, fmt, turned}; }

}  // namespace

extern "C" {

int smaul_fp8_block_quantize(const void* x, int dtype, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t K,
                             hipStream_t stream) {
  if (!fb_dtype_ok(dtype) || rows < 0 || K <= 0)
    return fail(SMAUL_ERR_INVALID, "fp8_block_quantize: bad sizes or dtype");
  if (rows == 0) return SMAUL_OK;
  if (!x || !codes || !scales) return fail(SMAUL_ERR_INVALID, "fp8_block_quantize: null pointer");
  if (!fb_aligned(codes, 8)) return fail(SMAUL_ERR_INVALID, "fp8_block_quantize: codes must be 8-byte aligned");
  return launch_quantize(x, dtype, codes, scales, rows, K, stream);
}

int smaul_fp8_block_dequantize(const uint8_t* codes, const uint8_t* scales, void* y, int dtype, int64_t rows, int64_t K,
                               hipStream_t stream) {
  if (!fb_dtype_ok(dtype) || rows < 0 || K <= 0)
    return fail(SMAUL_ERR_INVALID, "fp8_block_dequantize: bad sizes or dtype");
  if (rows == 0) return SMAUL_OK;
  if (!codes || !scales || !y) return fail(SMAUL_ERR_INVALID, "fp8_block_dequantize: null pointer");
  if (!fb_aligned(codes, 8)) return fail(SMAUL_ERR_INVALID, "fp8_block_dequantize: codes must be 8-byte aligned");
  const int64_t blocks = (rows * fb_blocks(K) * 16 + 255) / 256;
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block_dequantize: too many values");
  auto* kernel = dtype == SMAUL_DTYPE_BF16 ? &fb_dequantize_kernel<true> : &fb_dequantize_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, codes, scales, y, rows, K);
  return check_launch("fb_dequantize_kernel");
}

int64_t smaul_fp8_block_linear_workspace_size(int64_t rows, int64_t in_f, int64_t out_f, int x_dtype) {
  if (rows < 0 || in_f <= 0 || out_f <= 0 || !x_ok(x_dtype)) return -1;
  Parts w;
  if (x_dtype != SMAUL_DTYPE_FP8_BLOCK) {
    w.take(rows * fb_width(in_f));
    w.take(rows * fb_words(in_f) * 4);
  }
  return w.at;
}

int smaul_fp8_block_linear(const void* x, int x_dtype, const uint8_t* xs, const uint8_t* w, const uint8_t* s, void* y,
                           int y_dtype, int64_t rows, int64_t in_f, int64_t out_f, void* workspace,
                           int64_t workspace_bytes, hipStream_t stream) {
  if (!x_ok(x_dtype) || !fb_dtype_ok(y_dtype) || rows < 0 || in_f <= 0 || out_f <= 0)
    return fail(SMAUL_ERR_INVALID, "fp8_block_linear: bad sizes or dtype");
  if (rows == 0) return SMAUL_OK;
  const bool given = x_dtype == SMAUL_DTYPE_FP8_BLOCK;
  if (!x || !w || !s || !y || (given && !xs)) return fail(SMAUL_ERR_INVALID, "fp8_block_linear: null pointer");
  if (!fb_aligned(x, 16) || !fb_aligned(w, 16) || !fb_aligned(y, 16) || !fb_aligned(s, 4) || (given && !fb_aligned(xs, 4)))
    return fail(SMAUL_ERR_INVALID, "fp8_block_linear: x, y and the codes must be 16-byte aligned, the scales 4-byte");
  const int64_t need = smaul_fp8_block_linear_workspace_size(rows, in_f, out_f, x_dtype);
  if (workspace_bytes < need || (need > 0 && (!workspace || !fb_aligned(workspace, 256))))
    return fail(SMAUL_ERR_INVALID, "fp8_block_linear: workspace %lld < %lld bytes, or unaligned",
                (long long)workspace_bytes, (long long)need);
  if (!given) {
    uint8_t* c = (uint8_t*)workspace;
    uint8_t* cs = c + fb_align256(rows * fb_width(in_f));
    if (int rc = launch_quantize(x, x_dtype, c, cs, rows, in_f, stream)) return rc;
    x = c;
    xs = cs;
  }
  FbProduct p{};
  p.a[0] = codes_mat(x, xs, in_f);
  p.b[0] = codes_mat(w, s, in_f);
  p.pairs = 1;
  p.bf16 = y_dtype == SMAUL_DTYPE_BF16;
  p.c = y;
  p.M = rows;
  p.N = out_f;
  p.K = in_f;
  p.ldc = out_f;
  return launch_product(p, stream);
}

int64_t smaul_fp8_block_backward_input_workspace_size(int64_t rows, int64_t in_f, int64_t out_f, int dtype) {
  if (rows < 0 || in_f <= 0 || out_f <= 0 || !fb_dtype_ok(dtype)) return -1;
  return 0;
}

int smaul_fp8_block_backward_input(const void* g, int dtype, const uint8_t* w, const uint8_t* s, void* dx, int64_t rows,
                                   int64_t in_f, int64_t out_f, void* workspace, int64_t workspace_bytes,
                                   hipStream_t stream) {
  if (!fb_dtype_ok(dtype) || rows < 0 || in_f <= 0 || out_f <= 0)
    return fail(SMAUL_ERR_INVALID, "fp8_block_backward_input: bad sizes or dtype");
  if (rows == 0) return SMAUL_OK;
  if (!g || !w || !s || !dx) return fail(SMAUL_ERR_INVALID, "fp8_block_backward_input: null pointer");
  if (!fb_aligned(g, 16) || !fb_aligned(w, 16) || !fb_aligned(dx, 16))
    return fail(SMAUL_ERR_INVALID, "fp8_block_backward_input: g, dx and the codes must be 16-byte aligned");
  const int64_t need = smaul_fp8_block_backward_input_workspace_size(rows, in_f, out_f, dtype);
  if (workspace_bytes < need || (need > 0 && (!workspace || !fb_aligned(workspace, 256))))
    return fail(SMAUL_ERR_INVALID, "fp8_block_backward_input: workspace %lld < %lld bytes, or unaligned",
                (long long)workspace_bytes, (long long)need);
  const bool bf16 = dtype == SMAUL_DTYPE_BF16;
  FbProduct p{};
  p.a[0] = float_mat(g, out_f, bf16 ? F_BF16 : F_F32);
  p.b[0] = codes_mat(w, s, in_f, 1);
  p.pairs = 1;
  p.bf16 = bf16;
  p.c = dx;
  p.M = rows;
  p.N = in_f;
  p.K = out_f;
  p.ldc = in_f;
  return launch_product(p, stream);
}

int64_t smaul_fp8_block_ffn_saved_size(int64_t T, int64_t h) {
  if (T < 0 || h <= 0) return -1;
  return T * h * 8;
}

int64_t smaul_fp8_block_ffn_workspace_size(int64_t T, int64_t d, int64_t h, int x_dtype, int save) {
  if (T < 0 || d <= 0 || h <= 0 || (x_dtype != SMAUL_DTYPE_BF16 && x_dtype != SMAUL_DTYPE_FP8_BLOCK)) return -1;
  return ffn_parts(T, d, h, x_dtype, save != 0).total;
}

int smaul_fp8_block_ffn_forward(const void* x, int x_dtype, const uint8_t* xs, const uint8_t* gate_w,
                                const uint8_t* gate_s, const uint8_t* up_w, const uint8_t* up_s, const uint8_t* down_w,
                                const uint8_t* down_s, void* y, uint8_t* x_codes, uint8_t* x_scales, uint8_t* h_codes,
                                uint8_t* h_scales, void* saved, int64_t T, int64_t d, int64_t h, void* workspace,
                                int64_t workspace_bytes, hipStream_t stream) {
  const bool given = x_dtype == SMAUL_DTYPE_FP8_BLOCK, save = saved != nullptr;
  if ((x_dtype != SMAUL_DTYPE_BF16 && !given) || T < 0 || d <= 0 || h <= 0)
    return fail(SMAUL_ERR_INVALID, "fp8_block_ffn: bad sizes or dtype");
  if (T == 0) return SMAUL_OK;
  if (!x || !gate_w || !gate_s || !up_w || !up_s || !down_w || !down_s || !y || (given && !xs) ||
      (save && (!h_codes || !h_scales || (!given && (!x_codes || !x_scales)))))
    return fail(SMAUL_ERR_INVALID, "fp8_block_ffn: null pointer");
  for (const void* p : {x, (const void*)gate_w, (const void*)up_w, (const void*)down_w, (const void*)y,
                        (const void*)x_codes, (const void*)h_codes, (const void*)saved})
    if (!fb_aligned(p, 16)) return fail(SMAUL_ERR_INVALID, "fp8_block_ffn: rows and codes must be 16-byte aligned");
  for (const void* p : {(const void*)xs, (const void*)gate_s, (const void*)up_s, (const void*)down_s,
                        (const void*)x_scales, (const void*)h_scales})
    if (!fb_aligned(p, 4)) return fail(SMAUL_ERR_INVALID, "fp8_block_ffn: scales must be 4-byte aligned");
  const FfnParts q = ffn_parts(T, d, h, x_dtype, save);
  if (workspace_bytes < q.total || (q.total > 0 && (!workspace || !fb_aligned(workspace, 256))))
    return fail(SMAUL_ERR_INVALID, "fp8_block_ffn: workspace %lld < %lld bytes, or unaligned",
                (long long)workspace_bytes, (long long)q.total);
  uint8_t* ws = (uint8_t*)workspace;
  if (!given) {
    uint8_t* xc = save ? x_codes : ws + q.xc;
    uint8_t* xcs = save ? x_scales : ws + q.xs;
    if (int rc = launch_quantize(x, x_dtype, xc, xcs, T, d, stream)) return rc;
    x = xc;
    xs = xcs;
  }
  uint8_t* hc = save ? h_codes : ws + q.hc;
  uint8_t* hs = save ? h_scales : ws + q.hs;
  float* g = save ? (float*)saved : (float*)(ws + q.keep);
  float* u = g + T * h;
  FbProduct p{};
  p.pairs = 1;
  p.a[0] = codes_mat(x, xs, d);
  p.b[0] = codes_mat(gate_w, gate_s, d);
  p.c = g;
  p.M = T;
  p.N = h;
  p.K = d;
  p.ldc = h;
  if (int rc = launch_product(p, stream)) return rc;
  p.b[0] = codes_mat(up_w, up_s, d);
  p.c = u;
  if (int rc = launch_product(p, stream)) return rc;
  const int64_t blocks = (T * fb_blocks(h) * 16 + 255) / 256;
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block_ffn: too many values");
  hipLaunchKernelGGL(fb_gated_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, g, u, hc, hs, T, h, (int)save);
  if (int rc = check_launch("fb_gated_kernel")) return rc;
  p.a[0] = codes_mat(hc, hs, h);
  p.b[0] = codes_mat(down_w, down_s, h);
  p.c = y;
  p.bf16 = 1;
  p.N = d;
  p.K = h;
  p.ldc = d;
  return launch_product(p, stream);
}

int64_t smaul_fp8_block_ffn_backward_workspace_size(int64_t T, int64_t d, int64_t h) {
  if (T < 0 || d <= 0 || h <= 0) return -1;
  return ffn_back_parts(T, h).total;
}

int smaul_fp8_block_ffn_backward(const void* dy, const uint8_t* gate_w, const uint8_t* gate_s, const uint8_t* up_w,
                                 const uint8_t* up_s, const uint8_t* down_w, const uint8_t* down_s,
                                 const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* h_codes,
                                 const uint8_t* h_scales, const void* saved, void* dx, void* dgate, void* dup,
                                 void* ddown, int64_t T, int64_t d, int64_t h, void* workspace, int64_t workspace_bytes,
                                 hipStream_t stream) {
  if (T < 0 || d <= 0 || h <= 0) return fail(SMAUL_ERR_INVALID, "fp8_block_ffn_backward: bad sizes");
  const bool weights = dgate != nullptr;
  if (weights != (dup != nullptr) || weights != (ddown != nullptr))
    return fail(SMAUL_ERR_INVALID, "fp8_block_ffn_backward: all weights' gradients or none");
  if (!weights && (!dx || T == 0)) return SMAUL_OK;
  if (T > 0 && (!dy || !gate_w || !gate_s || !up_w || !up_s || !down_w || !down_s || !saved ||
                (weights && (!x_codes || !x_scales || !h_codes || !h_scales))))
    return fail(SMAUL_ERR_INVALID, "fp8_block_ffn_backward: null pointer");
  for (const void* p : {dy, (const void*)gate_w, (const void*)up_w, (const void*)down_w, (const void*)x_codes,
                        (const void*)h_codes, saved, (const void*)dx, (const void*)dgate, (const void*)dup,
                        (const void*)ddown})
    if (!fb_aligned(p, 16))
      return fail(SMAUL_ERR_INVALID, "fp8_block_ffn_backward: rows and codes must be 16-byte aligned");
  const FfnBackParts q = ffn_back_parts(T, h);
  if (workspace_bytes < q.total || (q.total > 0 && (!workspace || !fb_aligned(workspace, 256))))
    return fail(SMAUL_ERR_INVALID, "fp8_block_ffn_backward: workspace %lld < %lld bytes, or unaligned",
                (long long)workspace_bytes, (long long)q.total);
  char* ws = (char*)workspace;
  float *dh = (float*)(ws + q.dh), *dg = (float*)(ws + q.dg), *du = (float*)(ws + q.du);
  const float* a = (const float*)saved;
  FbProduct p{};
  p.pairs = 1;
  p.a[0] = float_mat(dy, d, F_BF16);
  p.b[0] = codes_mat(down_w, down_s, h, 1);
  p.c = dh;
  p.M = T;
  p.N = h;
  p.K = d;
  p.ldc = h;
  if (T > 0) {
    if (int rc = launch_product(p, stream)) return rc;
    const int64_t blocks = (T * h + 255) / 256;
    if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block_ffn_backward: too many values");
    hipLaunchKernelGGL(fb_gated_backward_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, dh, a, a + T * h, dg, du,
                       T * h);
    if (int rc = check_launch("fb_gated_backward_kernel")) return rc;
  }
  p.bf16 = 1;
  if (dx && T > 0) {
    p.pairs = 2;
    p.a[0] = float_mat(dg, h, F_F32);
    p.b[0] = codes_mat(gate_w, gate_s, d, 1);
    p.a[1] = float_mat(du, h, F_F32);
    p.b[1] = codes_mat(up_w, up_s, d, 1);
    p.c = dx;
    p.N = d;
    p.K = h;
    p.ldc = d;
    if (int rc = launch_product(p, stream)) return rc;
  }
  if (!weights) return SMAUL_OK;
  p.pairs = 1;
  p.K = T;
  p.M = h;
  p.N = d;
  p.ldc = d;
  p.a[0] = float_mat(dg, h, F_F32, 1);
  p.b[0] = codes_mat(x_codes, x_scales, d, 1);
  p.c = dgate;
  if (int rc = launch_product(p, stream)) return rc;
  p.a[0] = float_mat(du, h, F_F32, 1);
  p.c = dup;
  if (int rc = launch_product(p, stream)) return rc;
  p.a[0] = float_mat(dy, d, F_BF16, 1);
  p.b[0] = codes_mat(h_codes, h_scales, h, 1);
  p.c = ddown;
  p.M = d;
  p.N = h;
  p.ldc = h;
  return launch_product(p, stream);
}

}  // extern "C"
