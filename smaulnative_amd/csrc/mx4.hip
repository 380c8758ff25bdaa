// mx4.hip -- blocks of 32 4-bit values on MI355X (gfx950): quantisation, the
// product with such a weight, its input gradient, and the routed experts.
//
//   y[r, n]  = sum_k x[r, k] W[n, k]           W[n, k] = code value * 2^(scale - 127)
//   dx[r, k] = sum_n g[r, n] W[n, k]
//   moe: out[t] = sum over t's experts of w (silu(x Wg^T) * (x Wu^T)) Wd^T
//
// A code and its scale are exact in bf16, so every product of the matrix cores is
// exact for bf16 activations and for activations in the format itself, and its
// sums are fp32; fp32 activations are three bf16 terms, all of their 24 bits.
#include "lds_dma.h"
#include "mx4.h"

using smaul::check_launch;
using smaul::cu_count;
using smaul::fail;
using smaul::grid_fits;

namespace {

// ---------------------------------------------------------------------------
// quantisation: 4 lanes a block, 8 values a lane
// ---------------------------------------------------------------------------
// 16 bytes from an address of no more than the values' own alignment
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void mx4_widen(const uint32_t (&u)[4], float* v) {  // 8 bf16
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(u[j] << 16);
    v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
  }
}

// 16 bytes that nobody reads again soon, past the caches
typedef uint32_t u32x4_nt __attribute__((ext_vector_type(4)));
template <bool NT>
__device__ __forceinline__ uint4 mx4_ld16(const void* p) {
  if constexpr (!NT) return *(const uint4*)p;
  const u32x4_nt v = __builtin_nontemporal_load((const u32x4_nt*)p);
  return make_uint4(v.x, v.y, v.z, v.w);
}
template <bool NT>
__device__ __forceinline__ void mx4_st16(void* p, uint4 v) {
  if constexpr (!NT) *(uint4*)p = v;
  else __builtin_nontemporal_store((u32x4_nt){v.x, v.y, v.z, v.w}, (u32x4_nt*)p);
}

// 8 consecutive values of a row from column c0, 0 past K.  VEC: whole, 16-byte aligned.
template <bool BF16, bool VEC, bool NT = false>
__device__ __forceinline__ void mx4_load8(const void* x, int64_t row, int64_t K, int64_t c0, float (&v)[8]) {
  const int64_t i = row * K + c0;
  if constexpr (VEC) {
    if constexpr (BF16) {
      const uint4 w = mx4_ld16<NT>((const uint16_t*)x + i);
      mx4_widen({w.x, w.y, w.z, w.w}, v);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 w = mx4_ld16<NT>((const float*)x + i + 4 * h);
        v[4 * h] = __uint_as_float(w.x); v[4 * h + 1] = __uint_as_float(w.y);
        v[4 * h + 2] = __uint_as_float(w.z); v[4 * h + 3] = __uint_as_float(w.w);
      }
    }
  } else if (c0 + 8 <= K) {
    if constexpr (BF16) {
      const u32x4_at2 w = *(const u32x4_at2*)((const uint16_t*)x + i);
      mx4_widen({w.x, w.y, w.z, w.w}, v);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4_at4 w = *(const u32x4_at4*)((const float*)x + i + 4 * h);
        v[4 * h] = __uint_as_float(w.x); v[4 * h + 1] = __uint_as_float(w.y);
        v[4 * h + 2] = __uint_as_float(w.z); v[4 * h + 3] = __uint_as_float(w.w);
      }
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

// the block's largest bits over its quad of lanes
__device__ __forceinline__ uint32_t mx4_quad_max(uint32_t m) {
  m = max(m, (uint32_t)__shfl_xor((int)m, 1, 4));
  return max(m, (uint32_t)__shfl_xor((int)m, 2, 4));
}

// A thread takes MX4_U groups of 8 values, all loaded first.  VEC: K is a multiple of
// 32, so that the groups, their codes and their blocks are each one run over the whole
// matrix; otherwise a row's last block is padded, and a group finds its row by a
// division (32-bit where the groups' number is).  NT: the values' side goes past the
// caches, where it is larger than they are anyway (65536 x 2048 bf16 there and back:
// 143 us through them, 108 past them, 6.3 TB/s; a smaller result is left for its reader).
constexpr int MX4_U = 4;
constexpr int64_t MX4_NT_BYTES = 128LL << 20;  // half of the last cache

// group i of rows of nb blocks: its row, and its first column
template <bool VEC>
__device__ __forceinline__ void mx4_place(int64_t i, int64_t nb, bool small, int64_t& row, int64_t& c0) {
  if constexpr (VEC) {
    row = 0;
    c0 = i * 8;
  } else if (small) {
    const uint32_t r = (uint32_t)i / (uint32_t)(nb * 4);
    row = r;
    c0 = (int64_t)((uint32_t)i - r * (uint32_t)(nb * 4)) * 8;
  } else {
    row = i / (nb * 4);
    c0 = (i - row * nb * 4) * 8;
  }
}

template <bool BF16, bool VEC, bool NT>
__global__ void __launch_bounds__(256)
mx4_quantize_kernel(const void* __restrict__ x, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales,
                    int64_t rows, int64_t K) {
  const int64_t nb = mx4_blocks(K), groups = rows * nb * 4;
  const bool small = groups < (1LL << 31);
  const int64_t i0 = (int64_t)blockIdx.x * (256 * MX4_U) + threadIdx.x;
  float v[MX4_U][8];
#pragma unroll
  for (int u = 0; u < MX4_U; ++u)
    if (i0 + u * 256 < groups) {
      int64_t row, c0;
      mx4_place<VEC>(i0 + u * 256, nb, small, row, c0);
      mx4_load8<BF16, VEC, NT>(x, row, K, c0, v[u]);
    }
#pragma unroll
  for (int u = 0; u < MX4_U; ++u) {
    const int64_t i = i0 + u * 256;
    if (i < groups) {  // whole quads
      const uint32_t byte = mx4_scale_byte(mx4_quad_max(mx4_amax8(v[u])));
      codes[i] = mx4_encode8(v[u], byte);
      if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
    }
  }
}

// 8 decoded values (bf16 pairs) to y[o ..]; whole: all of them are the row's (`left`)
template <bool BF16, bool VEC, bool NT>
__device__ __forceinline__ void mx4_store8(void* y, int64_t o, int64_t left, uint4 d) {
  const uint32_t u[4] = {d.x, d.y, d.z, d.w};
  if (VEC || left >= 8) {
    if constexpr (BF16) {
      const u32x4_at2 w = {d.x, d.y, d.z, d.w};
      if constexpr (VEC) mx4_st16<NT>((uint16_t*)y + o, d);
      else *(u32x4_at2*)((uint16_t*)y + o) = w;
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4_at4 w = {u[2 * h] << 16, u[2 * h] & 0xffff0000u, u[2 * h + 1] << 16, u[2 * h + 1] & 0xffff0000u};
        if constexpr (VEC) mx4_st16<NT>((float*)y + o + 4 * h, make_uint4(w.x, w.y, w.z, w.w));
        else *(u32x4_at4*)((float*)y + o + 4 * h) = w;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) {
        const uint32_t b = j & 1 ? u[j / 2] >> 16 : u[j / 2] & 0xffffu;
        if constexpr (BF16) ((uint16_t*)y)[o + j] = (uint16_t)b;
        else ((float*)y)[o + j] = __uint_as_float(b << 16);
      }
  }
}

template <bool BF16, bool VEC, bool NT>
__global__ void __launch_bounds__(256)
mx4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ y,
                      int64_t rows, int64_t K) {
  const int64_t nb = mx4_blocks(K), groups = rows * nb * 4;
  const bool small = groups < (1LL << 31);
  const int64_t i0 = (int64_t)blockIdx.x * (256 * MX4_U) + threadIdx.x;
  uint32_t c[MX4_U], s[MX4_U];
#pragma unroll
  for (int u = 0; u < MX4_U; ++u)
    if (i0 + u * 256 < groups) {
      c[u] = codes[i0 + u * 256];
      s[u] = scales[(i0 + u * 256) >> 2];
    }
#pragma unroll
  for (int u = 0; u < MX4_U; ++u)
    if (i0 + u * 256 < groups) {
      int64_t row, c0;
      mx4_place<VEC>(i0 + u * 256, nb, small, row, c0);
      mx4_store8<BF16, VEC, NT>(y, row * K + c0, K - c0, mx4_decode8(c[u], mx4_scale(s[u])));
    }
}

// ---------------------------------------------------------------------------
// operands of the larger products, one launch for all of a call's
// ---------------------------------------------------------------------------
// Scales go to [group of 128 values][row] dwords (four blocks' bytes): a stage's
// scales of consecutive rows are then whole cache lines (a dword from every row of
// the stored layout costs the GEMM as many line requests as a stage's codes).
// Activations are rounded to the format straight into that form, and rows whose
// width is no whole number of stages are copied to padded ones: codes 0.
// Widths are padded to whole stages of the widest kind, MX4_STAGE.
constexpr int MX4_GROUP = 128, MX4_STAGE = 256;
__host__ __device__ __forceinline__ int64_t mx4_groups(int64_t K) {
  return (K + MX4_STAGE - 1) / MX4_STAGE * (MX4_STAGE / MX4_GROUP);
}

struct Mx4Weight {
  const uint8_t* w;
  const uint8_t* s;
  uint32_t* st;    // [E][groups][N] dwords
  uint4* wp;       // padded codes [E N][groups * 4], or null: used as they are
  int64_t N, K;    // rows of an expert
  int64_t blocks;  // workgroups that the matrix takes
};
// activations: as they are, rounded, or copied to padded rows (fp32: of planes)
enum { P_NONE = 0, P_ROUND = 1, P_PAD = 2 };
// v = a + b + c, each the next 8 significant bits: exact in bf16, and all 24 of fp32.
// An infinity or NaN is a alone.
__device__ __forceinline__ void mx4_split3(const float* v, uint4 (&t)[3]) {
  uint32_t h[3][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = __builtin_canonicalizef(v[j]);  // a NaN that keeps its highest bit
    h[0][j] = __float_as_uint(a) & 0xffff0000u;
    float r = a - __uint_as_float(h[0][j]);
    r = r == r ? r : 0.0f;
    h[1][j] = __float_as_uint(r) & 0xffff0000u;
    h[2][j] = __float_as_uint(r - __uint_as_float(h[1][j]));
  }
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    uint32_t u[4];  // the high halves of pairs
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = __builtin_amdgcn_perm(h[q][2 * j + 1], h[q][2 * j], 0x07060302u);
    t[q] = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// fp32 rows as the larger products read them: three planes of bf16, 64 values of each in
// turn, [width / 64][3][64].  Split once here: split after the LDS read, each wave of a
// tile's columns did it again, 44 instructions beside three products.
__host__ __device__ __forceinline__ int64_t mx4_plane_at(int64_t c) { return c / 64 * 192 + c % 64; }

struct Mx4Prep {
  Mx4Weight m[3];
  const void* x;
  void* xo;        // codes [T][groups * 4] of 16 bytes, or padded rows
  uint32_t* xst;   // P_ROUND: scales [groups][T]
  int64_t T, K;
  int64_t xblocks;
  int xmode, xvec;
};

// a workgroup: 16 rows of one group, 16 lanes a row (16384 x 1024: 10.4 us, 11.7 of four groups)
template <bool BF16>
__device__ __forceinline__ void mx4_prep_rows(const Mx4Prep& p, int64_t block) {
  const int64_t ng = mx4_groups(p.K);
  const uint32_t rb = (uint32_t)block / (uint32_t)ng;  // both from one 32-bit grid
  const int64_t row = (int64_t)rb * 16 + (threadIdx.x >> 4), g = block - (int64_t)rb * ng;
  const int c = threadIdx.x & 15;
  if (row >= p.T) return;  // whole quads
  float v[8];
  const int64_t c0 = g * MX4_GROUP + c * 8;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.0f;
  if (c0 < p.K) {
    if (p.xvec && c0 + 8 <= p.K) mx4_load8<BF16, true>(p.x, row, p.K, c0, v);
    else mx4_load8<BF16, false>(p.x, row, p.K, c0, v);
  }
  const int64_t at = (row * ng + g) * 16 + c;  // groups of 8 values
  if (p.xmode == P_ROUND) {
    uint32_t byte = mx4_scale_byte(mx4_quad_max(mx4_amax8(v)));
    ((uint32_t*)p.xo)[at] = mx4_encode8(v, byte);
    byte <<= 8 * (c >> 2);  // the group's four blocks to one dword
    byte |= (uint32_t)__shfl_xor((int)byte, 4, 16);
    byte |= (uint32_t)__shfl_xor((int)byte, 8, 16);
    if (c == 0) p.xst[g * p.T + row] = byte;
  } else if constexpr (BF16) {
    ((uint4*)p.xo)[at] = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                                    pack_bf16(v[6], v[7]));
  } else {
    uint4 t[3];
    mx4_split3(v, t);
    uint16_t* o = (uint16_t*)p.xo + row * ng * (3 * MX4_GROUP) + mx4_plane_at(c0);
#pragma unroll
    for (int k = 0; k < 3; ++k) *(uint4*)(o + 64 * k) = t[k];
  }
}

// a thread: the four blocks of one group of one row, rows fastest
__device__ __forceinline__ void mx4_prep_weight(const Mx4Weight& m, int64_t E, int64_t block) {
  const int64_t ng = mx4_groups(m.K), nb = mx4_blocks(m.K);
  const int64_t i = block * 256 + threadIdx.x, all = E * ng * m.N;
  if (i >= all) return;
  int64_t q, e;
  if (all < 1LL << 32) {  // 64-bit divisions take as long as the loads
    q = (uint32_t)i / (uint32_t)m.N;
    e = (uint32_t)q / (uint32_t)ng;
  } else {
    q = i / m.N;
    e = q / ng;
  }
  const int64_t n = i - q * m.N, g = q - e * ng, row = e * m.N + n;
  const uint8_t* s = m.s + row * nb + g * 4;
  uint32_t d = 0;
  if (g * 4 + 4 <= nb && nb % 4 == 0 && ((uintptr_t)m.s & 3) == 0) {
    d = *(const uint32_t*)s;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) d |= (g * 4 + j < nb ? (uint32_t)s[j] : 127u) << (8 * j);
  }
  m.st[i] = d;
  if (m.wp) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      m.wp[(row * ng + g) * 4 + j] =
          g * 4 + j < nb ? ((const uint4*)m.w)[row * nb + g * 4 + j] : make_uint4(0, 0, 0, 0);
  }
}

template <bool BF16>
__global__ void __launch_bounds__(256) mx4_prep_kernel(Mx4Prep p, int64_t E) {
  int64_t b = blockIdx.x;
  if (b < p.xblocks) {
    mx4_prep_rows<BF16>(p, b);
    return;
  }
  b -= p.xblocks;
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    if (b < p.m[j].blocks) {
      mx4_prep_weight(p.m[j], E, b);
      return;
    }
    b -= p.m[j].blocks;
  }
}

// The weight turned round, for the input gradient: wt[i][o] = W[o][i] in bf16, rows of
// ldo values (zeros from O on).  A workgroup: 64 o by 64 i, through LDS.  The first
// workgroups lay out the gradient's rows where that has to be.
template <bool BF16>
__global__ void __launch_bounds__(256)
mx4_turn_kernel(Mx4Prep p, const uint8_t* __restrict__ w, const uint8_t* __restrict__ s, uint16_t* __restrict__ wt,
                int64_t O, int64_t I, int64_t ldo) {
  if (blockIdx.x < p.xblocks) {
    mx4_prep_rows<BF16>(p, blockIdx.x);
    return;
  }
  const uint32_t block = blockIdx.x - (uint32_t)p.xblocks;
  constexpr int LD = 72;  // 16-byte rows of 64 o, off the banks' period
  __shared__ __attribute__((aligned(16))) uint16_t sh[64 * LD];
  const int64_t nb = mx4_blocks(I);
  const uint32_t ti = (uint32_t)((I + 63) / 64), ot = block / ti;
  const int64_t i0 = (int64_t)(block - ot * ti) * 64, o0 = (int64_t)ot * 64;
  {
    const int o = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
    const int64_t b = (i0 + c) / MX4_BLOCK;
    uint2 codes = make_uint2(0, 0);
    float sc = 1.0f;
    if (o0 + o < O && b < nb) {
      codes = *(const uint2*)(w + ((o0 + o) * nb + b) * 16 + (c & 16) / 2);
      sc = mx4_scale(s[(o0 + o) * nb + b]);
    }
    const uint4 lo = mx4_decode8(codes.x, sc), hi = mx4_decode8(codes.y, sc);
    const uint32_t u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int j = 0; j < 16; ++j) sh[(c + j) * LD + o] = (uint16_t)(u[j / 2] >> (16 * (j & 1)));
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int at = threadIdx.x + q * 256, i = at >> 3, c = (at & 7) * 8;
    if (i0 + i < I) *(uint4*)(wt + (i0 + i) * ldo + o0 + c) = *(const uint4*)&sh[i * LD + c];
  }
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
// Activations: A_BF16, A_F32 (three bf16 terms) or A_MX4 (codes and scales).
enum { A_BF16 = 0, A_F32 = 1, A_MX4 = 2 };
// The weight: codes and scales, or (mx4_gemm_kernel) rows already decoded to bf16.
enum { W_MX4 = 0, W_BF16 = 1 };
// What a tile's sums become: rounded to bf16, fp32, or blocks of the format.
enum { O_BF16 = 0, O_F32 = 1, O_MX4 = 2, O_PLANES = 3 };

struct Mx4Args {
  const void* x;           // rows of K values (A_MX4: codes, 16 bytes a block)
  const uint8_t* xs;       // A_MX4: scales
  const int32_t* row_idx;  // logical row -> x row (null: the same)
  const uint8_t* w;        // [E] [N] rows of codes
  const uint8_t* s;        // [E] [N][nb] scales
  const uint8_t* w2;       // SwiGLU: up's (w, s are gate's)
  const uint8_t* s2;
  void* y;                 // [rows][N] (O_MX4: codes)
  uint8_t* ys;             // O_MX4: scales
  int64_t R, K, N;
  // the larger products: scales are [group][row] dwords (w's of each expert, xs and ys over
  // xrows and yrows rows); row strides of x and y in values (planes: of all three;
  // codes: blocks), of W in blocks
  int64_t ldx, ldw, ldy, xrows, yrows;
  const int32_t* seg_off;  // null: dense, R rows of one expert
  const int32_t* tile_off;
  int E;
  int tile;                // the larger products: which of the kernels' tiles
  int xvec;                // mx4_stream_kernel: x rows may be read 16 bytes at a time,
  int svec;                // and four scales of W
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

constexpr int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
bool aligned(const void* p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }
bool dtype_ok(int d) { return d == SMAUL_DTYPE_F32 || d == SMAUL_DTYPE_BF16; }

// The two kernels of larger calls: K in stages of KS, activations, codes and scales
// brought to LDS by DMA, NSTAGE stages in flight, WM x WN waves over BM rows x BN
// columns.
//
// Roles: the weight's rows are the matrix instruction's rows and the activations its
// columns, and row i of a 32 x 32 tile is given weight row 16 ((i / 4) % 2) + 4 (i / 8)
// + i % 4, so that the 16 sums of a lane are 16 consecutive outputs of one activation
// row: whole 16-byte pieces, and a block of the format has its largest value in 8
// instructions and one exchange.
template <int AT, int WF, int BM, int BN, int WM, int WN, int KS, int NSTAGE>
struct Mx4Cfg {
  static constexpr int NW = WM * WN;
  static constexpr int XP = AT == A_F32 ? 3 : 1;  // planes of x, each BM rows of XROW bytes
  static constexpr int XROW = AT == A_MX4 ? KS / 2 : KS * 2;
  static constexpr int WROW = WF == W_BF16 ? KS * 2 : KS / 2;
  static constexpr int XB = XP * BM * XROW, WB = BN * WROW;
  static constexpr int SROWS = WF == W_BF16 ? 0 : BN + (AT == A_MX4 ? BM : 0);  // of scales
  static constexpr int SG = KS < 128 ? 1 : KS / 128;                            // dwords of each
  static constexpr int STAGE = XB + WB + SROWS * SG * 4;
  // DMA instructions: a wave's of x and W, all of the scales
  static constexpr int X_INS = XB / (1024 * NW), W_INS = WB / (1024 * NW), S_INS = SROWS * SG / 64;
  static constexpr int DMA_MIN = X_INS + W_INS + S_INS / NW;
  static constexpr int SI = (S_INS + NW - 1) / NW < 1 ? 1 : (S_INS + NW - 1) / NW, SP = SROWS < 64 ? 1 : SROWS / 64;
  static constexpr int SD = NW % SP == 0 ? 1 : SI;  // different rows of a wave's scale instructions
  static constexpr int TT = BM / WM / 32, WT = BN / WN / 32;  // 32 x 32 tiles of a wave
  static constexpr int ROWS = BM, COLS = BN, KW = KS;
  static constexpr int LDS = NSTAGE * STAGE;
  static constexpr int XS = AT == A_MX4 ? 16 : 2;  // bytes of a unit of ldx
  static_assert(AT != A_F32 || KS == 64, "planes take turns every 64 values");
  static_assert(XB % (1024 * NW) == 0 && WB % (1024 * NW) == 0 && SROWS % 64 == 0, "whole DMA instructions");
  static_assert(DMA_MIN * (NSTAGE - 2) < 64 && LDS <= 160 * 1024, "pipeline depth");
};

// the weight row of row i of a 32-row tile
__device__ __forceinline__ int mx4_perm(int i) { return ((i >> 2) & 1) * 16 + (i >> 3) * 4 + (i & 3); }

// the place of chunk c (16 bytes) of LDS row r, rows of ROW bytes (as swz_a and swz_b)
template <int ROW>
__device__ __forceinline__ int mx4_swz(int r, int c) {
  if constexpr (ROW == 32) return c ^ (((r >> 2) ^ (r >> 3)) & 1);
  else if constexpr (ROW == 64) return c ^ swz_b(r);
  else if constexpr (ROW == 128) return c ^ swz_a(r);
  else return c ^ (r & 15);
}

// columns that a product writes: past N zeros, up to the padded row
template <int OT>
__host__ __device__ __forceinline__ int64_t mx4_cols(const Mx4Args& p) {
  const int64_t c = OT == O_MX4 ? p.ldy * MX4_BLOCK : OT == O_PLANES ? p.ldy / 3 : p.ldy;
  return c > p.N ? c : p.N;
}

typedef int i32x8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8_t mx4_operand(uint4 c) {
  i32x8_t r;  // 32 codes; the instruction reads no more of the eight registers
  r[0] = (int)c.x; r[1] = (int)c.y; r[2] = (int)c.z; r[3] = (int)c.w;
  r[4] = r[5] = r[6] = r[7] = 0;
  return r;
}

// Where a lane's DMA instructions of a tile read, and the tile's first rows.
template <class C, int WF, bool SWIGLU>
struct Mx4Source {
  const char* X;
  const uint8_t *W1, *W2, *S1, *S2;
  uint32_t x_off[C::X_INS], w_off[C::W_INS], s_off[C::SD];
};

// 32-bit offsets from the tile's first rows (gathered rows' from x's; the host checks its
// size).  Rows past the end read the last one: their sums are not stored.  row_of(r):
// x row of the tile's row r, from row0 where rows are not gathered.
template <class C, int WF, bool SWIGLU, class RowOf>
__device__ __forceinline__ void mx4_source(const Mx4Args& p, int e, int64_t row0, int64_t n0, int lane, int wave,
                                           RowOf row_of, Mx4Source<C, WF, SWIGLU>& q) {
  constexpr int XL = C::XROW / 16, XR = 64 / XL;  // lanes a row, rows an instruction
  const int64_t eblocks = (int64_t)e * p.N * p.ldw;  // ldw / 4 groups of N dwords: as many bytes as blocks
  const int64_t nw = min<int64_t>(n0, p.N - 1);      // first weight row; a tile of padding reads the last
  const int64_t w0 = (eblocks + nw * p.ldw) * 16, s0 = eblocks + nw * 4;
  q.W1 = p.w + (WF == W_BF16 ? nw * p.ldw * 2 : w0);
  q.S1 = p.s + s0;
  q.W2 = SWIGLU ? p.w2 + w0 : q.W1;
  q.S2 = SWIGLU ? p.s2 + s0 : q.S1;
  q.X = (const char*)p.x + (p.row_idx ? 0 : row0 * p.ldx * C::XS);
#pragma unroll
  for (int a = 0; a < C::X_INS; ++a) {
    const int i = (wave * C::X_INS + a) * XR + lane / XL, r = i % C::ROWS;
    q.x_off[a] =
        (uint32_t)(row_of(r) * p.ldx * C::XS + i / C::ROWS * C::XROW + mx4_swz<C::XROW>(r, lane % XL) * 16);
  }
  // staged weight row r, from the first: tiles of 32 (gate's, then up's), permuted
  const int64_t left = p.N - 1 - nw;
  auto w_row = [&](int r) -> int64_t {
    int t = r >> 5;
    if (SWIGLU) t = t >= C::COLS / 64 ? t - C::COLS / 64 : t;
    return min<int64_t>(t * 32 + mx4_perm(r & 31), left);
  };
  constexpr int WL = C::WROW / 16, WR = 64 / WL;
#pragma unroll
  for (int b = 0; b < C::W_INS; ++b) {
    const int r = (wave * C::W_INS + b) * WR + lane / WL;
    q.w_off[b] = (uint32_t)(w_row(r) * p.ldw * (WF == W_BF16 ? 2 : 16) + mx4_swz<C::WROW>(r, lane % WL) * 16);
  }
  // scale instruction i stages 64 rows of one group: of the weight's, then of x's
#pragma unroll
  for (int i = 0; i < C::SD; ++i) {
    const int r = (wave + C::NW * i) % C::SP * 64;
    q.s_off[i] = (uint32_t)(r < C::COLS ? w_row(r + lane) : (p.row_idx ? 0 : row0) + row_of(r + lane - C::COLS)) * 4;
  }
}

// the loads of stage kt into the stage buffer at LDS address l
template <class C, int WF, bool SWIGLU>
__device__ __forceinline__ void mx4_dma(const Mx4Args& p, const Mx4Source<C, WF, SWIGLU>& q, int wave, int kt,
                                        uint32_t l) {
  constexpr int WR = 64 / (C::WROW / 16);
#pragma unroll
  for (int i = 0; i < C::SI; ++i) {
    const int j = wave + C::NW * i, r = (C::SD == 1 ? wave : j) % C::SP * 64;
    if (C::S_INS > 0 && (C::S_INS % C::NW == 0 || j < C::S_INS)) {  // uniform
      const int64_t grp = C::KW < 128 ? kt / (128 / C::KW) : (int64_t)kt * C::SG + j / C::SP;
      const uint8_t* src =
          r >= C::COLS ? p.xs + grp * p.xrows * 4 : (SWIGLU && r >= C::COLS / 2 ? q.S2 : q.S1) + grp * p.N * 4;
      dma4(src, q.s_off[i % C::SD], l + C::XB + C::WB + j * 256);
    }
  }
  const char* xk = q.X + (int64_t)kt * (C::XP * C::XROW);
#pragma unroll
  for (int a = 0; a < C::X_INS; ++a) dma16(xk, q.x_off[a], l + (wave * C::X_INS + a) * 1024);
#pragma unroll
  for (int b = 0; b < C::W_INS; ++b) {
    const int r = (wave * C::W_INS + b) * WR;
    dma16((SWIGLU && r >= C::COLS / 2 ? q.W2 : q.W1) + (int64_t)kt * C::WROW, q.w_off[b],
          l + C::XB + (wave * C::W_INS + b) * 1024);
  }
}

// tile `lin` of m_tiles by n_tiles, in groups of 8 row tiles by all column tiles
__device__ __forceinline__ void mx4_tile_at(int lin, int m_tiles, int n_tiles, int& mt, int& nt) {
  constexpr int GM = 8;
  const int g = lin / (GM * n_tiles), within = lin - g * GM * n_tiles, gm = min(GM, m_tiles - g * GM);
  mt = g * GM + within % gm;
  nt = within / gm;
}

// 16 consecutive sums of row `row` from column n, cast; columns from `ld` on are not
// the row's.  whole (uniform): all of them are, and 16-byte aligned.
template <bool BF16>
__device__ __forceinline__ void mx4_store16(void* out, int64_t row, int64_t ld, int64_t n, bool whole,
                                            const float (&v)[16]) {
  const int64_t o = row * ld + n;
  if constexpr (BF16) {
    uint32_t u[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) u[r] = pack_bf16(v[2 * r], v[2 * r + 1]);
    uint16_t* y = (uint16_t*)out + o;
    if (whole) {
      ((uint4*)y)[0] = make_uint4(u[0], u[1], u[2], u[3]);
      ((uint4*)y)[1] = make_uint4(u[4], u[5], u[6], u[7]);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (n + r < ld) y[r] = (uint16_t)(u[r / 2] >> (16 * (r & 1)));
    }
  } else {
    float* y = (float*)out + o;
    if (whole) {
#pragma unroll
      for (int r = 0; r < 4; ++r) ((float4*)y)[r] = make_float4(v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (n + r < ld) y[r] = v[r];
    }
  }
}

// The sums of a wave's tiles to y.  bf16 rows leave as pieces of 64 bytes, four lanes a
// row, through 2 KB of LDS of the wave's own: a store of 16 bytes to each of 64 rows is
// 64 requests (16384 x 4096 x 4096: 203 us so, 191 through LDS; past the caches 187, but
// 4096 rows 58 us for 52, as half a line is then fetched again).
template <int OT, bool SWIGLU, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void mx4_epilogue(const Mx4Args& p, const f32x16_t (&acc)[BN / WN / 32][BM / WM / 32],
                                             int64_t row0, int rows, int64_t n0, int wm, int wn, int lane, char* own) {
  constexpr int TT = BM / WM / 32, WT = BN / WN / 32, BNO = SWIGLU ? BN / 2 : BN, OTW = SWIGLU ? WT / 2 : WT;
  const int g = lane >> 5, l32 = lane & 31;
  const bool inside = n0 + BNO <= p.N;  // of the whole workgroup: no column past N
  const bool whole = (OT == O_BF16 || OT == O_F32) && n0 + BNO <= p.ldy && p.ldy % 8 == 0;
#pragma unroll
  for (int i = 0; i < TT; ++i) {
    const int lr = wm * (BM / WM) + i * 32 + l32;
    const bool live = lr < rows;
    const int64_t row = row0 + lr;
#pragma unroll
    for (int j = 0; j < OTW; ++j) {
      const int64_t nb0 = n0 + wn * (BNO / WN) + j * 32, n = nb0 + g * 16;
      float v[16];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        v[r] = SWIGLU ? mx4_swiglu(acc[j][i][r], acc[j + WT / 2 < WT ? j + WT / 2 : j][i][r]) : acc[j][i][r];
      if (!inside) {  // padding
        const int left = (int)(p.N - n < 16 ? p.N - n : 16);
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = r < left ? v[r] : 0.0f;
      }
      if constexpr (OT == O_MX4) {
        float m = __builtin_fabsf(v[0]);  // NaN stays NaN
#pragma unroll
        for (int r = 1; r < 16; ++r) m = __builtin_elementwise_maximum(m, __builtin_fabsf(v[r]));
        m = __builtin_elementwise_maximum(m, __shfl_xor(m, 32, 64));
        const uint32_t byte = mx4_scale_byte(__float_as_uint(m) & 0x7fffffffu);
        const uint32_t lo = mx4_encode8(v, byte), hi = mx4_encode8(v + 8, byte);
        const int64_t b = row * p.ldy + nb0 / MX4_BLOCK;
        if (live && nb0 / MX4_BLOCK < p.ldy) {
          *(uint2*)((uint8_t*)p.y + b * 16 + g * 8) = make_uint2(lo, hi);
          if (g == 0) p.ys[(nb0 / MX4_GROUP * p.yrows + row) * 4 + nb0 % MX4_GROUP / MX4_BLOCK] = (uint8_t)byte;
        }
      } else if constexpr (OT == O_PLANES) {
        uint4 lo[3], hi[3];
        mx4_split3(v, lo);
        mx4_split3(v + 8, hi);
        uint16_t* y = (uint16_t*)p.y + row * p.ldy + mx4_plane_at(n);
        if (live && n < mx4_cols<OT>(p)) {
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            ((uint4*)(y + 64 * k))[0] = lo[k];
            ((uint4*)(y + 64 * k))[1] = hi[k];
          }
        }
      } else {
        if constexpr (OT == O_BF16) {
          if (whole) {
            const int m = l32 / 2 & 3;  // 8 lanes' pieces are in different banks, here and below
            *(uint4*)(own + l32 * 64 + (2 * g ^ m) * 16) =
                make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
            *(uint4*)(own + l32 * 64 + ((2 * g + 1) ^ m) * 16) = make_uint4(
                pack_bf16(v[8], v[9]), pack_bf16(v[10], v[11]), pack_bf16(v[12], v[13]), pack_bf16(v[14], v[15]));
            __builtin_amdgcn_wave_barrier();  // a wave's LDS accesses are done in order
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int r = h * 16 + lane / 4, c = lane % 4, tr = wm * (BM / WM) + i * 32 + r;
              const uint4 d = *(const uint4*)(own + r * 64 + (c ^ (r / 2 & 3)) * 16);
              uint16_t* y = (uint16_t*)p.y + (row0 + tr) * p.ldy + nb0 + c * 8;
              if (tr < rows) *(uint4*)y = d;
            }
            __builtin_amdgcn_wave_barrier();
            continue;
          }
        }
        if (live) mx4_store16<OT == O_BF16>(p.y, row, p.ldy, n, whole, v);
      }
    }
  }
}

// Activations as they are (A_BF16, A_F32): the weight is decoded.  A lane's 16 bytes of
// codes are its block g of a 64-wide step, times their scale (exact in bf16), and MFMA
// q multiplies values 32 g + 8 q and on; fp32 activations are three planes of bf16.
// W_BF16: the weight's rows are bf16 already.
template <int AT, int WF, int OT, bool SWIGLU, int BM, int BN, int WM, int WN, int KS, int NSTAGE>
__global__ void __launch_bounds__(WM * WN * 64, WM * WN < 4 ? 1 : 2) mx4_gemm_kernel(Mx4Args p) {
  using C = Mx4Cfg<AT, WF, BM, BN, WM, WN, KS, NSTAGE>;
  static_assert(AT != A_MX4 && OT != O_MX4, "mx4_codes_kernel's");
  constexpr int TT = C::TT, WT = C::WT, BNO = SWIGLU ? BN / 2 : BN, XROW = C::XROW, WROW = C::WROW;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // a contiguous band of tiles for each XCD (workgroup b runs on XCD b % 8)
  int mt, nt;
  {
    constexpr int NXCD = 8;
    const int n_tiles = (int)((mx4_cols<OT>(p) + BNO - 1) / BNO), total = gridDim.x;
    int lin = blockIdx.x;
    const int full = total / NXCD * NXCD;
    if (lin < full) lin = lin % NXCD * (full / NXCD) + lin / NXCD;
    mx4_tile_at(lin, total / n_tiles, n_tiles, mt, nt);
  }
  int e, rows;
  int64_t row0;
  if (!mx4_tile<BM>(p, mt, lane, e, row0, rows)) return;
  const int64_t n0 = (int64_t)nt * BNO;
  Mx4Source<C, WF, SWIGLU> src;
  mx4_source(p, e, row0, n0, lane, wave, [&](int r) -> int64_t {
    const int lr = min(r, rows - 1);
    return p.row_idx ? (int64_t)p.row_idx[row0 + lr] : lr;
  }, src);
  const uint32_t lds0 = lds_offset(&smem[0]);
  auto dma_stage = [&](int kt, int buf) { mx4_dma(p, src, wave, kt, lds0 + (uint32_t)(buf * C::STAGE)); };

  const int g = lane >> 5, l32 = lane & 31;
  // staged row of weight tile j of this wave: with SwiGLU its gate tiles, then its up tiles
  auto w_tile = [&](int j) -> int {
    if constexpr (SWIGLU)
      return j < WT / 2 ? wn * (BN / WN / 2) + j * 32 : BN / 2 + wn * (BN / WN / 2) + (j - WT / 2) * 32;
    else return wn * (BN / WN) + j * 32;
  };
  f32x16_t acc[WT][TT];
#pragma unroll
  for (int j = 0; j < WT; ++j)
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0.0f;

  const int nk = (int)(p.K / KS);
  auto compute = [&](int buf, int kt) {
    const char* xs_ = smem + buf * C::STAGE;
    const char* ws_ = xs_ + C::XB;
    const char* ss_ = ws_ + C::WB;
#pragma unroll
    for (int h = 0; h < KS / 64; ++h) {
      const int sh = 8 * g + 16 * (KS < 128 ? kt & 1 : h & 1);
      uint4 wc[WT];  // codes of block g of each weight row, and its scale
      float sc[WT];
#pragma unroll
      for (int j = 0; j < WT && WF == W_MX4; ++j) {
        const int r = w_tile(j) + l32;
        wc[j] = *(const uint4*)(ws_ + r * WROW + mx4_swz<WROW>(r, h * 2 + g) * 16);
        sc[j] = mx4_scale((*(const uint32_t*)(ss_ + (h / 2 * C::SROWS + r) * 4) >> sh) & 255u);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        bf16x8_t xf[TT][C::XP];
#pragma unroll
        for (int i = 0; i < TT; ++i) {
          const int r = wm * (BM / WM) + i * 32 + l32;
#pragma unroll
          for (int k = 0; k < C::XP; ++k)
            xf[i][k] = *(const bf16x8_t*)(xs_ + (k * BM + r) * XROW + mx4_swz<XROW>(r, h * 8 + g * 4 + q) * 16);
        }
#pragma unroll
        for (int j = 0; j < WT; ++j) {
          bf16x8_t wf;
          if constexpr (WF == W_BF16) {
            const int r = w_tile(j) + l32;
            wf = *(const bf16x8_t*)(ws_ + r * WROW + mx4_swz<WROW>(r, h * 8 + g * 4 + q) * 16);
          } else {
            const uint32_t c = q == 0 ? wc[j].x : q == 1 ? wc[j].y : q == 2 ? wc[j].z : wc[j].w;
            wf = __builtin_bit_cast(bf16x8_t, mx4_decode8(c, sc[j]));
          }
#pragma unroll
          for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int k = 0; k < C::XP; ++k)
              acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf, xf[i][k], acc[j][i], 0, 0, 0);
        }
      }
    }
  };
  // Stage kt is complete when at most the loads of the later stages are outstanding;
  // the barrier publishes it and frees the buffer of stage kt - 1.  Stages past the
  // end load the last one again into a buffer nobody reads.
#pragma unroll
  for (int s = 0; s + 1 < NSTAGE; ++s) dma_stage(s < nk ? s : nk - 1, s);
  int buf = 0, nbuf = NSTAGE - 1;
  for (int kt = 0; kt < nk; ++kt) {
    wait_vm<C::DMA_MIN * (NSTAGE - 2)>();
    __syncthreads();
    const int ks = kt + NSTAGE - 1;
    dma_stage(ks < nk ? ks : nk - 1, nbuf);
    compute(buf, kt);
    buf = buf + 1 == NSTAGE ? 0 : buf + 1;
    nbuf = nbuf + 1 == NSTAGE ? 0 : nbuf + 1;
  }
  wait_vm<0>();

  if constexpr (OT == O_BF16) __syncthreads();  // the stages' LDS is the waves' now
  mx4_epilogue<OT, SWIGLU, BM, BN, WM, WN>(p, acc, row0, rows, n0, wm, wn, lane, smem + wave * 2048);
}

template <int AT, int WF, int OT, bool SWIGLU, int BM, int BN, int WM, int WN, int KS, int NSTAGE>
int launch_gemm_cfg(const Mx4Args& p, int64_t m_tiles, hipStream_t stream) {
  using C = Mx4Cfg<AT, WF, BM, BN, WM, WN, KS, NSTAGE>;
  constexpr int BNO = SWIGLU ? BN / 2 : BN;
  if (BM * p.ldx * C::XS >= 1LL << 32 || BN * p.ldw * (WF == W_BF16 ? 2 : 16) >= 1LL << 32)
    return fail(SMAUL_ERR_UNSUPPORTED, "mx4 product: rows too wide");
  const int64_t n_tiles = (mx4_cols<OT>(p) + BNO - 1) / BNO;
  if (!grid_fits(m_tiles * n_tiles, WM * WN * 64)) return fail(SMAUL_ERR_UNSUPPORTED, "mx4 product: too many tiles");
  hipLaunchKernelGGL((mx4_gemm_kernel<AT, WF, OT, SWIGLU, BM, BN, WM, WN, KS, NSTAGE>),
                     dim3((unsigned)(m_tiles * n_tiles)), dim3(WM * WN * 64), 0, stream, p);
  return check_launch("mx4_gemm_kernel");
}

// Activations in the format: v_mfma_scale_f32_32x32x64_f8f6f4 on the codes as they are,
// lane i + 32 g with block g of a 64-wide step of its row and one scale byte for the 32
// values.
//
// Stages are 256 wide, 128-byte rows: what costs the loop is L2 requests, and half a line
// is one too.  The operands of a step are read from LDS while the step before is
// multiplied, the first of a stage during the last of the stage before; by then every
// wave has the rest of its stage in registers, so that one barrier frees the buffer for
// the loads of the stage after the next.
//
// A workgroup (one a CU, two of the smaller tiles) walks a band of tiles as one sequence
// of stages: the loads of the next tile's first stages leave during the last of this one
// and its operands are in registers before the epilogue, which they hide behind.  K of
// 1024 is four stages: a tile's start, its row indices and first loads, took a quarter of
// its time (16384 tokens to 2 of 8 experts, 1024 by 2560: 274 us with a workgroup a tile,
// 236 so).
template <int OT, bool SWIGLU, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64, 2) mx4_codes_kernel(Mx4Args p, int m_tiles) {
  constexpr int KS = 256, NSTAGE = 2, STEPS = KS / 64;
  using C = Mx4Cfg<A_MX4, W_MX4, BM, BN, WM, WN, KS, NSTAGE>;
  constexpr int TT = C::TT, WT = C::WT, BNO = SWIGLU ? BN / 2 : BN, XROW = C::XROW, WROW = C::WROW;
  constexpr int OWN = OT == O_BF16 ? 2048 : 0;  // bytes that a wave's rows leave through
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS + WM * WN * OWN];
  __shared__ int index[2][BM];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, g = lane >> 5, l32 = lane & 31;
  const uint32_t lds0 = lds_offset(&smem[0]);
  const int n_tiles = (int)((mx4_cols<OT>(p) + BNO - 1) / BNO);

  // every expert's tiles and segment, a lane an expert
  int to0 = 0, to1 = 0x7fffffff, so0 = 0, so1 = 0;
  if (p.seg_off) {
    if (lane < p.E) {
      to0 = p.tile_off[lane];
      to1 = p.tile_off[lane + 1];
      so0 = p.seg_off[lane];
      so1 = p.seg_off[lane + 1];
    }
    m_tiles = __builtin_amdgcn_readlane(to1, p.E - 1);  // of the bound that the host knows
  }
  // XCD x (workgroup b runs on XCD b % 8) takes a contiguous band of the tiles
  const int wgs = gridDim.x, nx = min(8, wgs), xcd = (int)blockIdx.x % nx, step = (wgs - xcd + nx - 1) / nx;
  const int total = m_tiles * n_tiles, last = (int)((int64_t)total * (xcd + 1) / nx);
  int lin = (int)((int64_t)total * xcd / nx) + (int)blockIdx.x / nx;
  if (lin >= last) return;

  auto place = [&](int at, int& e, int64_t& row0, int& rows, int64_t& n0) {
    int mt, nt;
    mx4_tile_at(at, m_tiles, n_tiles, mt, nt);
    n0 = (int64_t)nt * BNO;
    if (!p.seg_off) {
      e = 0;
      row0 = (int64_t)mt * BM;
      rows = (int)min<int64_t>(BM, p.R - row0);
      return;
    }
    e = (int)__popcll(__ballot(to1 <= mt));
    const int r0 = __builtin_amdgcn_readlane(so0, e) + (mt - __builtin_amdgcn_readlane(to0, e)) * BM;
    row0 = r0;
    rows = min(BM, __builtin_amdgcn_readlane(so1, e) - r0);
  };
  // x rows of tile `at` to LDS (from the tile's first where they are not gathered): two
  // buffers, one being filled while the other may still be read
  auto gather = [&](int at, int buf) {
    int e, rows;
    int64_t row0, n0;
    place(at, e, row0, rows, n0);
    const int r = wave * 64 + lane, lr = min(r, rows - 1);
    if (wave >= BM / 64) return;
    if (p.row_idx) dma4(p.row_idx + row0, (uint32_t)lr * 4, lds_offset(&index[buf][wave * 64]));
    else index[buf][r] = lr;
  };
  Mx4Source<C, W_MX4, SWIGLU> src;
  auto source = [&](int at, int buf) {
    int e, rows;
    int64_t row0, n0;
    place(at, e, row0, rows, n0);
    mx4_source(p, e, row0, n0, lane, wave, [&](int r) -> int64_t { return index[buf][r]; }, src);
  };
  // the loads of the sequence's next stage, of this tile or the one after
  const int nk = (int)(p.K / KS);
  int load_at = lin, load_k = nk, turn = 0;
  auto load = [&](int buf) {
    if (load_k == nk) {
      if (load_at >= last) return;
      source(load_at, turn);
      turn ^= 1;
      load_at += step;
      load_k = 0;
      if (load_at < last) gather(load_at, turn);  // there at the next stage's barrier
    }
    mx4_dma(p, src, wave, load_k, lds0 + (uint32_t)(buf * C::STAGE));
    ++load_k;
  };
  gather(lin, 0);
  wait_vm<0>();
  __syncthreads();
  load(0);
  wait_vm<0>();
  __syncthreads();
  load(1);

  // staged row of weight tile j of this wave: with SwiGLU its gate tiles, then its up tiles
  auto w_tile = [&](int j) -> int {
    if constexpr (SWIGLU)
      return j < WT / 2 ? wn * (BN / WN / 2) + j * 32 : BN / 2 + wn * (BN / WN / 2) + (j - WT / 2) * 32;
    else return wn * (BN / WN) + j * 32;
  };
  i32x8_t wf[2][WT], xf[2][TT];
  uint32_t sw[2][WT], sx[2][TT];
  const char* w_at[WT];  // fixed parts of the addresses
  const char* x_at[TT];
#pragma unroll
  for (int j = 0; j < WT; ++j) w_at[j] = smem + C::XB + (w_tile(j) + l32) * WROW;
#pragma unroll
  for (int i = 0; i < TT; ++i) x_at[i] = smem + (wm * (BM / WM) + i * 32 + l32) * XROW;
  const char* s_at = smem + C::XB + C::WB + l32 * 4;
  auto read = [&](int buf, int u) {
    const int o = buf * C::STAGE, c = u * 2 + g, to = u & 1;
    if (u % 2 == 0) {  // the scales of a group of 128
#pragma unroll
      for (int j = 0; j < WT; ++j) sw[u / 2][j] = *(const uint32_t*)(s_at + o + (u / 2 * C::SROWS + w_tile(j)) * 4);
#pragma unroll
      for (int i = 0; i < TT; ++i)
        sx[u / 2][i] = *(const uint32_t*)(s_at + o + (u / 2 * C::SROWS + BN + wm * (BM / WM) + i * 32) * 4);
    }
    // tiles are 32 rows apart, which the swizzles do not see
#pragma unroll
    for (int i = 0; i < TT; ++i) xf[to][i] = mx4_operand(*(const uint4*)(x_at[i] + o + mx4_swz<XROW>(l32, c) * 16));
#pragma unroll
    for (int j = 0; j < WT; ++j) wf[to][j] = mx4_operand(*(const uint4*)(w_at[j] + o + mx4_swz<WROW>(l32, c) * 16));
  };
  f32x16_t acc[WT][TT];
  auto multiply = [&](int u) {
    if (u % 2 == 0) {  // this lane's blocks, g and g + 2 of the four, to bytes 0 and 2
#pragma unroll
      for (int j = 0; j < WT; ++j) sw[u / 2][j] >>= 8 * g;
#pragma unroll
      for (int i = 0; i < TT; ++i) sx[u / 2][i] >>= 8 * g;
    }
#pragma unroll
    for (int j = 0; j < WT; ++j)
#pragma unroll
      for (int i = 0; i < TT; ++i)
        acc[j][i] = u % 2 == 0
            ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[0][j], xf[0][i], acc[j][i], 4, 4, 0,
                                                              (int)sw[u / 2][j], 0, (int)sx[u / 2][i])
            : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[1][j], xf[1][i], acc[j][i], 4, 4, 2,
                                                              (int)sw[u / 2][j], 2, (int)sx[u / 2][i]);
  };

  read(0, 0);
  int buf = 0;
  for (; lin < last; lin += step) {
#pragma unroll
    for (int j = 0; j < WT; ++j)
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[j][i][r] = 0.0f;
    for (int kt = 0; kt < nk; ++kt, buf ^= 1) {
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        if (u + 1 < STEPS) {
          read(buf, u + 1);
        } else {
#pragma unroll
          for (int j = 0; j < WT; ++j)  // the products so far stay before the branch
#pragma unroll
            for (int i = 0; i < TT; ++i) asm volatile("" : "+v"(acc[j][i]));
          wait_vm<0>();
          __syncthreads();
          load(buf);
          read(buf ^ 1, 0);  // behind the last tile: values that nothing uses
        }
        __builtin_amdgcn_sched_barrier(0);
        multiply(u);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    int e, rows;
    int64_t row0, n0;
    place(lin, e, row0, rows, n0);
    mx4_epilogue<OT, SWIGLU, BM, BN, WM, WN>(p, acc, row0, rows, n0, wm, wn, lane, smem + C::LDS + wave * OWN);
  }
}

template <int OT, bool SWIGLU, int BM, int BN, int WM, int WN>
int launch_codes(const Mx4Args& p, int64_t m_tiles, hipStream_t stream) {
  constexpr int BNO = SWIGLU ? BN / 2 : BN;
  const int64_t tiles = m_tiles * ((mx4_cols<OT>(p) + BNO - 1) / BNO);
  if ((BM > BN ? BM : BN) * (p.ldx > p.ldw ? p.ldx : p.ldw) * 16 >= 1LL << 32)
    return fail(SMAUL_ERR_UNSUPPORTED, "mx4 product: rows too wide");
  if (tiles > 2147483647LL) return fail(SMAUL_ERR_UNSUPPORTED, "mx4 product: too many tiles");
  // as many as LDS holds: 512 tokens to 2 of 8 experts 43 us with one a CU, 40 with two
  const int64_t wgs = cu_count() * (BM * BN <= 128 * 128 ? 2 : 1);
  hipLaunchKernelGGL((mx4_codes_kernel<OT, SWIGLU, BM, BN, WM, WN>), dim3((unsigned)(tiles < wgs ? tiles : wgs)),
                     dim3(WM * WN * 64), 0, stream, p, (int)m_tiles);
  return check_launch("mx4_codes_kernel");
}

// The kernel of few rows (up to 64): a workgroup has 32 columns of one expert, its NW
// waves a slice of K each, so that every byte of the weight is read once and all at
// the same time.  A lane's codes lie in a row of their own, but x, which comes from the
// caches for every 32 columns again, goes through LDS: a load of four rows by 256 bytes
// asks for 8 lines, one of 32 rows by 32 bytes for 32 (32 x 4096 -> 4096: 10 us, 15.4
// from registers; 64 tokens to 2 of 8 experts, 1024 by 2560: 14.5 + 9.7 us, 16.4 + 10.8;
// the weights alone are 5).  The waves' sums meet in LDS too and are added in the order
// of the waves.  Sending the first weights before the rows are known cost more
// registers than it won (19.2 us for 14.5).
//
// The experts' rows are found here, without a dispatch: a workgroup looks through the
// T k <= 512 slots for its expert's; the hidden rows and the outputs
// stand at their slots.  Two launches less than a dispatch takes, and a layer of 64
// tokens is launches and latency (84 us with the tile kernel behind a dispatch).
struct Mx4Slots {
  const int64_t* topi;  // null: dense, row r of x to row r of y
  const float* topw;
  int32_t* counts;      // by the first workgroup of each expert, or null
  int T, k;
  int by_token;         // x rows by token (else by slot)
};
constexpr int ST_ROWS = 64, ST_SLOTS = 512;

// whether slot i of (token, expert) is one that the layer runs: an expert of the E, a
// weight above 0, and the token's first slot with it (as smaul_moe_dispatch)
__device__ __forceinline__ bool mx4_slot(const int64_t* topi, const float* topw, int64_t t, int j, int k, int E,
                                         int e) {
  if (topi[t * k + j] != e || !(topw[t * k + j] > 0.0f) || e < 0 || e >= E) return false;
  for (int i = 0; i < j; ++i)
    if (topi[t * k + i] == e && topw[t * k + i] > 0.0f) return false;
  return true;
}

template <int AT, int OT, bool SWIGLU, bool VEC, int NW>
__global__ void __launch_bounds__(NW * 64) mx4_stream_kernel(Mx4Args p, Mx4Slots q) {
  constexpr int SW = SWIGLU ? 2 : 1, U = AT == A_MX4 ? 4 : 2;  // steps read at once
  constexpr int JS = 1024 + 64;  // bytes between the quarters of a wave's sums: other banks
  // x as it is: a wave's U steps of 32 rows, XP pieces of 16 bytes a row, changing places
  // by the row; the sums meet in the same LDS
  constexpr bool XL = VEC && AT != A_MX4;
  constexpr int XSZ = AT == A_BF16 ? 2 : 4, XP = U * 4 * XSZ, XI = XL ? XP / 2 : 1, XW = XL ? 32 * XP * 16 : 0;
  __shared__ __attribute__((aligned(1024))) char red[NW * (XW > 4 * JS ? XW : 4 * JS)];
  constexpr int NC = ST_SLOTS / (NW * 64);  // slots a thread
  __shared__ int s_row[ST_ROWS], s_cnt[NC * NW];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n_tiles = (int)((p.N + 31) / 32);
  const int e = blockIdx.x / n_tiles;
  const int64_t n0 = (int64_t)(blockIdx.x % n_tiles) * 32;

  int rows = (int)p.R;
  if (q.topi) {
    bool mine[NC];
    uint64_t b[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = c * NW * 64 + tid;
      mine[c] = i < q.T * q.k && mx4_slot(q.topi, q.topw, i / q.k, i % q.k, q.k, p.E, e);
      b[c] = __ballot(mine[c]);
      if (lane == 0) s_cnt[c * NW + wave] = __popcll(b[c]);
    }
    __syncthreads();
    rows = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      int before = rows;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        before += w < wave ? s_cnt[c * NW + w] : 0;
        rows += s_cnt[c * NW + w];
      }
      // at most one slot a token: rows <= T <= 64
      if (mine[c]) s_row[before + __popcll(b[c] & ((1ull << lane) - 1))] = c * NW * 64 + tid;
    }
    if (q.counts && n0 == 0 && tid == 0) q.counts[e] = rows;
    __syncthreads();
  }

  const int64_t nb = mx4_blocks(p.K);
  const int64_t wrow = n0 + mx4_perm(l32) < p.N ? n0 + mx4_perm(l32) : p.N - 1;
  const int64_t wblk = ((int64_t)e * p.N + wrow) * nb;
  const int steps = (int)((nb + 1) / 2), per = ((steps + NW - 1) / NW + 1) / 2 * 2;
  const int lo = min(wave * per, steps), hi = min(lo + per, steps);

  uint4 wc[U][SW];
  uint32_t ws[U][SW];
  auto load_w = [&](int s0) {
    uint32_t sd[(U + 1) / 2][SW];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t b = (int64_t)(s0 + u) * 2 + g;  // this lane's block of the step
      const bool in = s0 + u < hi && b < nb;
#pragma unroll
      for (int j = 0; j < SW; ++j) {
        wc[u][j] = in ? *(const uint4*)((j ? p.w2 : p.w) + (wblk + b) * 16) : make_uint4(0, 0, 0, 0);
        const uint8_t* s = (j ? p.s2 : p.s) + wblk;
        if (p.svec) {  // the four scales of 128 values at once; slices begin at a multiple
          if (u % 2 == 0) sd[u / 2][j] = in ? *(const uint32_t*)(s + (b - g)) : 0u;
          ws[u][j] = sd[u / 2][j] >> (16 * (u & 1) + 8 * g);
        } else {
          ws[u][j] = in ? s[b] : 0u;
        }
      }
    }
  };
  for (int r0 = 0; r0 < rows; r0 += 32) {  // uniform
    const int r = min(r0 + l32, rows - 1);
    const int64_t slot = q.topi ? s_row[r] : r;
    const int64_t xr = q.topi && q.by_token ? slot / q.k : slot;
    f32x16_t acc[SW];
#pragma unroll
    for (int j = 0; j < SW; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[j][i] = 0.0f;

    char* own = red + wave * XW;
    uint32_t x_at[XI];  // where this lane's piece of DMA instruction a begins, in the row
    if constexpr (XL) {
#pragma unroll
      for (int a = 0; a < XI; ++a) {
        const int rr = a * (64 / XP) + lane / XP, rc = min(r0 + rr, rows - 1);
        const int at = q.topi ? s_row[rc] : rc, row = q.topi && q.by_token ? at / q.k : at;
        x_at[a] = (uint32_t)(row * p.K * XSZ);
      }
    }
    for (int s0 = lo; s0 < hi; s0 += U) {
      if constexpr (XL) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last pieces are read
#pragma unroll
        for (int a = 0; a < XI; ++a) {
          if (a * (64 / XP) >= rows - r0) break;  // uniform; rows that nobody needs hold anything
          const int rr = a * (64 / XP) + lane / XP;
          const int64_t col = (int64_t)s0 * 64 * XSZ + (lane % XP ^ (rr & 15)) * 16, end = p.K * XSZ - 16;
          dma16(p.x, x_at[a] + (uint32_t)(col < end ? col : end), lds_offset(own + a * 1024));
        }
      }
      load_w(s0);
      uint4 xv[U];  // A_MX4
      uint32_t xsc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t b = (int64_t)(s0 + u) * 2 + g;
        const bool in = s0 + u < hi && b < nb;
        if constexpr (AT == A_MX4) {
          xv[u] = in ? *(const uint4*)((const uint8_t*)p.x + (xr * nb + b) * 16) : make_uint4(0, 0, 0, 0);
          xsc[u] = in ? p.xs[xr * nb + b] : 0u;
        }
      }
      if constexpr (XL) wait_vm<0>();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s0 + u >= hi) break;  // uniform
        if constexpr (AT == A_MX4) {
#pragma unroll
          for (int j = 0; j < SW; ++j)
            acc[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                mx4_operand(wc[u][j]), mx4_operand(xv[u]), acc[j], 4, 4, 0, (int)ws[u][j], 0, (int)xsc[u]);
        } else {
          const int64_t b = (int64_t)(s0 + u) * 2 + g;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            constexpr int NT = AT == A_F32 ? 3 : 1;
            bf16x8_t t[3];
            const int64_t c0 = b * MX4_BLOCK + v * 8;
            // piece i, whose first column is c; rows end with whole pieces, past them zeros
            auto piece = [&](int i, int64_t c) {
              const uint4 x = *(const uint4*)(own + (l32 * XP + (i ^ (l32 & 15))) * 16);
              return c < p.K ? x : make_uint4(0, 0, 0, 0);
            };
            if constexpr (XL && AT == A_BF16) {
              t[0] = __builtin_bit_cast(bf16x8_t, piece(u * 8 + g * 4 + v, c0));
            } else {
              float f[8];
              if constexpr (XL) {
                const uint4 a = piece(u * 16 + g * 8 + 2 * v, c0), c = piece(u * 16 + g * 8 + 2 * v + 1, c0 + 4);
                f[0] = __uint_as_float(a.x); f[1] = __uint_as_float(a.y);
                f[2] = __uint_as_float(a.z); f[3] = __uint_as_float(a.w);
                f[4] = __uint_as_float(c.x); f[5] = __uint_as_float(c.y);
                f[6] = __uint_as_float(c.z); f[7] = __uint_as_float(c.w);
              } else {
                mx4_load8<AT == A_BF16, false>(p.x, xr, p.K, c0, f);
              }
              uint4 h[3];
              mx4_split3(f, h);
#pragma unroll
              for (int k = 0; k < 3; ++k) t[k] = __builtin_bit_cast(bf16x8_t, h[k]);
            }
#pragma unroll
            for (int j = 0; j < SW; ++j) {
              const uint4 c = wc[u][j];
              const bf16x8_t wf = __builtin_bit_cast(
                  bf16x8_t, mx4_decode8(v == 0 ? c.x : v == 1 ? c.y : v == 2 ? c.z : c.w, mx4_scale(ws[u][j] & 255u)));
#pragma unroll
              for (int k = 0; k < NT; ++k)
                acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf, t[k], acc[j], 0, 0, 0);
            }
          }
        }
      }
    }
    // Register 4 i + 0..3 of a lane: quarter i of its 16 consecutive outputs.  Gate's
    // sums and up's go through the same LDS, for twice the workgroups on a CU.
    const int row = tid >> 3, h = (tid >> 2) & 1, i = tid & 3;  // 8 threads a row: quarter i of half h
    float v[SW][4];
#pragma unroll
    for (int j = 0; j < SW; ++j) {
      if (j || XL) __syncthreads();
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *(float4*)(red + (wave * 4 + c) * JS + lane * 16) =
            make_float4(acc[j][4 * c], acc[j][4 * c + 1], acc[j][4 * c + 2], acc[j][4 * c + 3]);
      __syncthreads();
      if (tid < 256) {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[j][c] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float4 a = *(const float4*)(red + (w * 4 + i) * JS + (h * 32 + row) * 16);
          v[j][0] += a.x;
          v[j][1] += a.y;
          v[j][2] += a.z;
          v[j][3] += a.w;
        }
      }
    }
    if (tid < 256) {
      const int64_t n = n0 + h * 16 + i * 4;
      float o[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        o[c] = SWIGLU ? mx4_swiglu(v[0][c], v[SW - 1][c]) : v[0][c];
        if (n + c >= p.N) o[c] = 0.0f;
      }
      const bool live = r0 + row < rows;
      const int64_t yr = live ? (q.topi ? s_row[r0 + row] : r0 + row) : 0;
      if constexpr (OT == O_MX4) {
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) m = max(m, __float_as_uint(o[c]) & 0x7fffffffu);
        for (int d = 4; d >= 1; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d, 8));
        const uint32_t byte = mx4_scale_byte(m);
        const float e8[8] = {o[0], o[1], o[2], o[3], 0.0f, 0.0f, 0.0f, 0.0f};
        const int64_t b = yr * mx4_blocks(p.N) + n0 / MX4_BLOCK;
        if (live) {
          *(uint16_t*)((uint8_t*)p.y + b * 16 + h * 8 + i * 2) = (uint16_t)mx4_encode8(e8, byte);
          if ((tid & 7) == 0) p.ys[b] = (uint8_t)byte;
        }
      } else if (live) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (n + c < p.N) {
            if constexpr (OT == O_BF16) ((__bf16*)p.y)[yr * p.N + n + c] = (__bf16)o[c];
            else ((float*)p.y)[yr * p.N + n + c] = o[c];
          }
      }
    }
    __syncthreads();
  }
}

// The input gradient of few rows (up to 64), in one launch: a workgroup has one block of
// columns, its NW waves a slice of the weight's rows each.  A lane reads 32 codes of one
// weight row, and the wave turns 64 such rows round through LDS of its own.  The blocks
// of a line of codes are columns of one XCD, which reads the line once.  Two launches are
// longer than the work: 1 to 32 bf16 rows 2560 -> 1024 10 to 11.5 us, 25 by way of the
// turned weight (4000 -> 4096: 15 to 17, 43).
template <int AT, bool VEC, int NW>
__global__ void __launch_bounds__(NW * 64)
mx4_dx_stream_kernel(const void* __restrict__ g, const uint8_t* __restrict__ w, const uint8_t* __restrict__ s,
                     void* __restrict__ dx, int64_t R, int64_t I, int64_t O) {
  constexpr int U = 2, LD = 72;  // steps of 64 rows read at once; rows of 64 bf16, off the banks' period
  constexpr int JS = 1024 + 64;  // as mx4_stream_kernel's
  constexpr int NT = AT == A_F32 ? 3 : 1, OWN = 32 * LD * 2 > 4 * JS ? 32 * LD * 2 : 4 * JS;
  __shared__ __attribute__((aligned(16))) char sh[NW * OWN];
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t nb = mx4_blocks(I);
  int64_t b0 = blockIdx.x;
  {
    const int64_t full = (int64_t)gridDim.x / 8 * 8;
    if (b0 < full) b0 = b0 % 8 * (full / 8) + b0 / 8;
  }
  uint16_t* own = (uint16_t*)(sh + wave * OWN);
  const int64_t steps = (O + 63) / 64, per = (steps + NW - 1) / NW;
  const int64_t lo = min((int64_t)wave * per, steps), hi = min(lo + per, steps);

  for (int64_t r0 = 0; r0 < R; r0 += 32) {  // uniform
    const int64_t r = min(r0 + l32, R - 1);
    f32x16_t acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    for (int64_t s0 = lo; s0 < hi; s0 += U) {
      uint4 wc[U];
      uint32_t ws[U];
      float v[U][4][8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t o = (s0 + u) * 64 + lane;
        const bool in = s0 + u < hi && o < O;
        wc[u] = in ? *(const uint4*)(w + (o * nb + b0) * 16) : make_uint4(0, 0, 0, 0);
        ws[u] = in ? s[o * nb + b0] : 0u;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t c = (s0 + u) * 64 + q * 16 + h * 8;
#pragma unroll
          for (int j = 0; j < 8; ++j) v[u][q][j] = 0.0f;
          if (s0 + u < hi && c < O) mx4_load8<AT == A_BF16, VEC>(g, r, O, c, v[u][q]);  // VEC: O is a multiple of 8
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s0 + u >= hi) break;  // uniform
        const float sc = mx4_scale(ws[u]);
        const uint32_t c[4] = {wc[u].x, wc[u].y, wc[u].z, wc[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4 d = mx4_decode8(c[k], sc);
          const uint32_t p[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) own[(8 * k + j) * LD + lane] = (uint16_t)(p[j / 2] >> (16 * (j & 1)));
        }
        __builtin_amdgcn_wave_barrier();  // a wave's LDS accesses are done in order
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const bf16x8_t a = *(const bf16x8_t*)&own[mx4_perm(l32) * LD + q * 16 + h * 8];
          uint4 t[3];
          if constexpr (AT == A_F32) {
            mx4_split3(v[u][q], t);
          } else {
            const float* x = v[u][q];
            t[0] = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]),
                              pack_bf16(x[6], x[7]));
          }
#pragma unroll
          for (int k = 0; k < NT; ++k)
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8_t, t[k]), acc, 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
    // the waves' sums, in the order of the waves: thread by row, half and quarter, as there
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *(float4*)(sh + (wave * 4 + c) * JS + lane * 16) =
          make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
    __syncthreads();
    if (tid < 256) {
      const int row = tid >> 3, half = (tid >> 2) & 1, i = tid & 3;
      float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int q = 0; q < NW; ++q) {
        const float4 a = *(const float4*)(sh + (q * 4 + i) * JS + (half * 32 + row) * 16);
        o[0] += a.x;
        o[1] += a.y;
        o[2] += a.z;
        o[3] += a.w;
      }
      const int64_t n = b0 * MX4_BLOCK + half * 16 + i * 4;
      if (r0 + row < R)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (n + c < I) {
            const int64_t at = (r0 + row) * I + n + c;
            if constexpr (AT == A_BF16) ((__bf16*)dx)[at] = (__bf16)o[c];
            else ((float*)dx)[at] = o[c];
          }
    }
    __syncthreads();
  }
}

template <int AT, int OT, bool SWIGLU, int NW>
int launch_stream_cfg(Mx4Args p, const Mx4Slots& q, int64_t groups, hipStream_t stream) {
  p.svec = mx4_blocks(p.K) % 4 == 0 && aligned(p.s, 4) && (!SWIGLU || aligned(p.s2, 4));
  const dim3 grid((unsigned)groups), block(NW * 64);
  if constexpr (AT != A_MX4) {
    const int64_t x_rows = q.topi ? (q.by_token ? q.T : q.T * q.k) : p.R;
    if (!p.xvec || x_rows * p.K * 4 >= 1LL << 32) {
      hipLaunchKernelGGL((mx4_stream_kernel<AT, OT, SWIGLU, false, NW>), grid, block, 0, stream, p, q);
      return check_launch("mx4_stream_kernel");
    }
  }
  hipLaunchKernelGGL((mx4_stream_kernel<AT, OT, SWIGLU, true, NW>), grid, block, 0, stream, p, q);
  return check_launch("mx4_stream_kernel");
}

template <int AT, int OT, bool SWIGLU>
int launch_stream(const Mx4Args& p, const Mx4Slots& q, hipStream_t stream) {
  const int64_t groups = (p.N + 31) / 32 * p.E;
  if (!grid_fits(groups, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "mx4 product: too many columns");
  // 4 waves where there are workgroups enough for that: then all of them run at once
  if (groups > 2 * cu_count()) return launch_stream_cfg<AT, OT, SWIGLU, 4>(p, q, groups, stream);
  return launch_stream_cfg<AT, OT, SWIGLU, 8>(p, q, groups, stream);
}

// out[t] = the sum of its slots' rows times their weights, in ascending expert order
// (fp32, product and sum rounded each, as smaul_moe_combine's), in x's type.  The
// slots' rows stay fp32 where the hidden rows were rounded to bf16 already: one
// rounding less between the experts and the sum.  With rounded activations they are bf16,
// an expert's output in x's type: as large an error as the result's own rounding (2.4e-3
// against 64 bits, 1.7e-3 of fp32 rows), beside rows of 4 bits, for half the bytes (16384
// tokens to 2 of 8 experts, 1024 by 2560: 221 us, 246 of fp32 rows).  A thread has 8
// columns; every row is read before the first is used.
template <bool YF32, bool OBF16, int KM>
__global__ void __launch_bounds__(256)
mx4_combine_kernel(const void* __restrict__ y, const int64_t* __restrict__ topi, const float* __restrict__ topw,
                   const int32_t* __restrict__ inv, void* __restrict__ out, int64_t T, int d, int k, int E) {
  const int cpt = d / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, t = i / cpt;
  if (t >= T) return;
  const int c = (int)(i - t * cpt) * 8;
  int pos[KM], key[KM];
  float w[KM];
#pragma unroll
  for (int j = 0; j < KM; ++j)
    if (j < k) {
      const int64_t e = topi[t * k + j];
      key[j] = (int)e;
      w[j] = topw[t * k + j];
      // no dispatch's rows: the outputs stand at their slots
      pos[j] = inv ? inv[t * k + j] : e >= 0 && e < E && w[j] > 0.0f ? (int)(t * k) + j : -1;
    }
  if (!inv) {  // a second slot of one expert adds nothing
#pragma unroll
    for (int j = 1; j < KM; ++j)
#pragma unroll
      for (int i = 0; i < j; ++i)
        if (j < k && pos[i] >= 0 && key[i] == key[j]) pos[j] = -1;
  }
#pragma unroll
  for (int j = 0; j < KM; ++j)
    if (j >= k || pos[j] < 0) {
      pos[j] = -1;
      key[j] = 0x7fffffff;
      w[j] = 0.0f;
    }
#pragma unroll
  for (int pass = 0; pass < KM; ++pass)
#pragma unroll
    for (int j = pass & 1; j + 1 < KM; j += 2) {
      const bool swap = key[j] > key[j + 1];
      const int k0 = key[j], p0 = pos[j];
      const float w0 = w[j];
      key[j] = swap ? key[j + 1] : k0;
      pos[j] = swap ? pos[j + 1] : p0;
      w[j] = swap ? w[j + 1] : w0;
      key[j + 1] = swap ? k0 : key[j + 1];
      pos[j + 1] = swap ? p0 : pos[j + 1];
      w[j + 1] = swap ? w0 : w[j + 1];
    }
  float v[KM][8];
#pragma unroll
  for (int j = 0; j < KM; ++j)
    if (pos[j] >= 0) mx4_load8<!YF32, true>(y, pos[j], d, c, v[j]);
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < KM; ++j)
    if (pos[j] >= 0)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float pr = v[j][q] * w[j];
        acc[q] = acc[q] + pr;
      }
  const int64_t o = t * d + c;
  if constexpr (OBF16) {
    *(uint4*)((uint16_t*)out + o) = make_uint4(pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3]),
                                               pack_bf16(acc[4], acc[5]), pack_bf16(acc[6], acc[7]));
  } else {
    ((float4*)((float*)out + o))[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    ((float4*)((float*)out + o))[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  }
}

template <bool YF32, bool OBF16>
int launch_combine(const void* y, const int64_t* topi, const float* topw, const int32_t* inv, void* out, int64_t T,
                   int64_t d, int64_t k, int64_t E, hipStream_t stream) {
  const dim3 grid((unsigned)((T * (d / 8) + 255) / 256)), block(256);
#define SMAUL_C(KM) \
  hipLaunchKernelGGL((mx4_combine_kernel<YF32, OBF16, KM>), grid, block, 0, stream, y, topi, topw, inv, out, T, \
                     (int)d, (int)k, (int)E)
  if (k <= 2) SMAUL_C(2);
  else if (k <= 4) SMAUL_C(4);
  else SMAUL_C(8);
#undef SMAUL_C
  return check_launch("mx4_combine_kernel");
}

int launch_quantize(const void* x, int dtype, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t K,
                    hipStream_t stream) {
  const bool vec = K % MX4_BLOCK == 0 && aligned(x, 16), bf16 = dtype == SMAUL_DTYPE_BF16;
  constexpr int64_t per = 256 * MX4_U;
  const int64_t blocks = (rows * mx4_blocks(K) * 4 + per - 1) / per;
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "mx4_quantize: too many values");
  const dim3 grid((unsigned)blocks), block(256);
  const bool nt = rows * K * (bf16 ? 2 : 4) >= MX4_NT_BYTES;
#define SMAUL_Q(B, V, N) \
  hipLaunchKernelGGL((mx4_quantize_kernel<B, V, N>), grid, block, 0, stream, x, (uint32_t*)codes, scales, rows, K)
  if (bf16 && vec && nt) SMAUL_Q(true, true, true);
  else if (bf16 && vec) SMAUL_Q(true, true, false);
  else if (bf16) SMAUL_Q(true, false, false);
  else if (vec && nt) SMAUL_Q(false, true, true);
  else if (vec) SMAUL_Q(false, true, false);
  else SMAUL_Q(false, false, false);
#undef SMAUL_Q
  return check_launch("mx4_quantize_kernel");
}

// Up to ST_ROWS rows (tokens of a layer) mx4_stream_kernel runs, past them the larger
// products, in tiles that fill the chip: what a round of the CUs takes (of 256 x 256 =
// 100), times the rounds.  The smaller tiles of codes run two a CU, in rounds of twice the
// CUs; a last round of no more than one a CU is `one`.  The last parts of the experts'
// segments count for half a tile.  us, by tiles of 256 x 256, 128 x 256, 128 x 128 and
// 64 x 128, rounded activations: 512 x 4096 -> 4096 32, 24, 20, 18; 1500 rows 37, 28, 28, 33;
// 6000 x 4096 -> 1024 (96, 188, 376, 752 tiles) 43, 49, 35, 39; 8192 x 4096 -> 2560 78, 75,
// 70, 84; 16384 x 1024 -> 2560 45, 47, 46, 57; tokens to 2 of 8 experts, 1024 by 2560: 700
// 53, 49, 42, 41; 16000 209, 235, 234, 296.  Of 144 products the choice is on average 1.2 % off
// the best, at most 14.  bf16 as it is, 128 x 256 and 64 x 128: 512 rows 58, 31; 1500 rows
// 65, 65; 16384 x 1024 -> 2560 80, 114.
struct Mx4Tile {
  int bm, bn, one, two;  // two: 0 where a CU takes them one by one
};
constexpr Mx4Tile CODES_TILES[] = {{256, 256, 100, 0}, {128, 256, 63, 0}, {128, 128, 40, 62}, {64, 128, 28, 39}};
constexpr Mx4Tile BF16_TILES[] = {{128, 256, 62, 0}, {64, 128, 22, 0}};
constexpr Mx4Tile F32_TILES[] = {{32, 256, 100, 0}};

struct Mx4Shape {  // of one product
  int64_t R, K, cols;
  bool swiglu;
};

int64_t tile_bm(int at, int tile) {
  return at == A_F32 ? F32_TILES[tile].bm : at == A_MX4 ? CODES_TILES[tile].bm : BF16_TILES[tile].bm;
}

// the tile for products that share their row tiles, `parts` experts
template <int N, int M>
int pick_tile(const Mx4Tile (&tiles)[N], const Mx4Shape (&products)[M], int64_t parts) {
  const int64_t cus = cu_count();
  int best = 0;
  double least = 0.0;
  for (int i = 0; i < N; ++i) {
    double cost = 0.0;
    for (const Mx4Shape& q : products) {
      const int64_t bn = q.swiglu ? tiles[i].bn / 2 : tiles[i].bn;
      const int64_t m = (q.R + tiles[i].bm - 1) / tiles[i].bm + parts / 2, n = (q.cols + bn - 1) / bn;
      const int64_t round = tiles[i].two ? 2 * cus : cus, full = m * n / round, left = m * n % round;
      const int whole = tiles[i].two ? tiles[i].two : tiles[i].one;
      cost += (double)q.K * ((double)full * whole + (left == 0 ? 0 : left <= cus ? tiles[i].one : whole));
    }
    if (i == 0 || cost < least) {
      best = i;
      least = cost;
    }
  }
  return best;
}
template <int M>
int pick_tile(int at, const Mx4Shape (&products)[M], int64_t parts) {
  return at == A_F32 ? 0 : at == A_MX4 ? pick_tile(CODES_TILES, products, parts)
                                       : pick_tile(BF16_TILES, products, parts);
}

template <int AT, int OT, bool SWIGLU>
int launch_product(const Mx4Args& p, const Mx4Slots* few, int64_t m_tiles, hipStream_t stream) {
  if (few) return launch_stream<AT, OT, SWIGLU>(p, *few, stream);
  // us, fp32, 4096 x 1024 -> 2560 and 3001 x 1000 -> 777: 77 and 47 of 32 x 256, 84 and 50
  // of 64 x 256, 87 and 47 of 64 x 128, 91 and 42 of 32 x 128
  if constexpr (AT == A_F32) {
    return launch_gemm_cfg<AT, W_MX4, SWIGLU ? O_PLANES : OT, SWIGLU, 32, 256, 1, 4, 64, 2>(p, m_tiles, stream);
  } else if constexpr (AT == A_BF16) {
    if (p.tile == 0) return launch_gemm_cfg<AT, W_MX4, OT, SWIGLU, 128, 256, 2, 2, 64, 3>(p, m_tiles, stream);
    return launch_gemm_cfg<AT, W_MX4, OT, SWIGLU, 64, 128, 2, 2, 64, 3>(p, m_tiles, stream);
  } else {
    if (p.tile == 0) return launch_codes<OT, SWIGLU, 256, 256, 4, 2>(p, m_tiles, stream);
    if (p.tile == 1) return launch_codes<OT, SWIGLU, 128, 256, 2, 4>(p, m_tiles, stream);
    if (p.tile == 2) return launch_codes<OT, SWIGLU, 128, 128, 2, 2>(p, m_tiles, stream);
    return launch_codes<OT, SWIGLU, 64, 128, 2, 2>(p, m_tiles, stream);
  }
}

// activations with a weight: y of `out` type
int launch_linear(const Mx4Args& p, int at, int out, const Mx4Slots* few, int64_t m_tiles, hipStream_t stream) {
  if (at == A_MX4)
    return out == O_BF16 ? launch_product<A_MX4, O_BF16, false>(p, few, m_tiles, stream)
                         : launch_product<A_MX4, O_F32, false>(p, few, m_tiles, stream);
  if (at == A_BF16)
    return out == O_BF16 ? launch_product<A_BF16, O_BF16, false>(p, few, m_tiles, stream)
                         : launch_product<A_BF16, O_F32, false>(p, few, m_tiles, stream);
  return launch_product<A_F32, O_F32, false>(p, few, m_tiles, stream);
}

void prep_rows(Mx4Prep& p, int dtype) {  // the workgroups of x's rows
  if (p.xmode == P_NONE) return;
  p.xblocks = (p.T + 15) / 16 * mx4_groups(p.K);
  p.xvec = aligned(p.x, 16) && p.K % (dtype == SMAUL_DTYPE_BF16 ? 8 : 4) == 0;
}

int launch_prep(Mx4Prep p, int dtype, int64_t E, hipStream_t stream) {
  prep_rows(p, dtype);
  int64_t blocks = p.xblocks;
  for (auto& m : p.m) {
    if (m.w) m.blocks = (E * mx4_groups(m.K) * m.N + 255) / 256;
    blocks += m.blocks;
  }
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "mx4 product: too many rows or weights");
  auto* kernel = dtype == SMAUL_DTYPE_BF16 ? &mx4_prep_kernel<true> : &mx4_prep_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p, E);
  return check_launch("mx4_prep_kernel");
}

// a workspace laid out part by part
struct Parts {
  int64_t at = 0;
  int64_t take(int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  }
};

// A linear's workspace: the activations rounded or in padded rows, and the weight's
// scales (and padded codes) as the GEMM reads them.  Up to ST_ROWS rows the weight is
// read as it is stored.
struct LinearParts {
  bool gemm;
  int64_t x, xs, st, wp, total;
};
LinearParts linear_parts(int64_t rows, int64_t K, int64_t N, int dtype, int act) {
  const bool mx4 = act == SMAUL_ACT_MX4;
  const int64_t ng = mx4_groups(K), nb = mx4_blocks(K);
  const bool pad = K % MX4_STAGE != 0, f32 = dtype == SMAUL_DTYPE_F32;
  LinearParts q{};
  Parts w;
  q.gemm = rows > ST_ROWS;
  if (!q.gemm) {
    q.x = w.take(mx4 ? rows * nb * 16 : 0);
    q.xs = w.take(mx4 ? rows * nb : 0);
  } else {
    q.x = w.take(mx4 ? rows * ng * 64 : f32 || pad ? rows * ng * MX4_GROUP * (f32 ? 6 : 2) : 0);
    q.xs = w.take(mx4 ? rows * ng * 4 : 0);
    q.st = w.take(N * ng * 4);
    q.wp = w.take(pad ? N * ng * 64 : 0);
  }
  q.total = w.at;
  return q;
}

// The input gradient's workspace: the weight turned round and decoded, and g's planes
// (fp32), or padded rows where its width is no whole number of stages.
struct DxParts {
  int64_t ldo, wt, g, total;
  bool gemm, lay;
};
DxParts dx_parts(int64_t rows, int64_t I, int64_t O, int dtype) {
  DxParts q{};
  Parts w;
  q.ldo = mx4_groups(O) * MX4_GROUP;
  const bool f32 = dtype == SMAUL_DTYPE_F32;
  // fp32's second 32 rows cost another pass over the weight: us, 4096 -> 4000, 32 and 33 rows
  // as few 25 and 41, by tiles 39 and 39; bf16, 33 and 64 rows, 29 and 31, by tiles 44
  q.gemm = rows > (f32 ? 32 : ST_ROWS);
  if (!q.gemm) return q;
  q.lay = f32 || O % 64 != 0;
  q.wt = w.take(I * q.ldo * 2);
  q.g = w.take(q.lay ? rows * q.ldo * (f32 ? 6 : 2) : 0);
  q.total = w.at;
  return q;
}

// The larger the tile, the less it reads, as long as every CU has one.  us, bf16, by
// tiles of 128 x 128, 128 x 256 and 256 x 256: 4096 rows 2560 -> 1024 (1, 1/2 and 1/4
// tiles a CU) 33, 44, 65; 2048 rows 4096 -> 4096 (2, 1, 1/2) 91, 77, 104; 8192 rows (8, 4,
// 2) 315, 268, 244.  Of 128 x 128 and 64 x 64: 512 rows 4000 -> 4096 (1/2 and 2 tiles a CU)
// 48, 42, 1024 rows 57, 69; 256 rows 2560 -> 1024 26, 17.6.  fp32, 512 rows 2560 -> 1024 and
// 1001 rows 777 -> 1000: 30 and 22 of 32 x 64, 31 and 25 of 64 x 64, 41 and 31 of 64 x 128
// (half the workgroups of a chip).
template <int AT, int OT>
int launch_dx(const Mx4Args& p, hipStream_t stream) {
  const int64_t cus = cu_count(), mt = (p.R + 127) / 128, nt = (p.N + 255) / 256;
  if constexpr (AT == A_F32) {
    return launch_gemm_cfg<AT, W_BF16, OT, false, 32, 64, 1, 2, 64, 3>(p, (p.R + 31) / 32, stream);
  } else {
    if ((mt + 1) / 2 * nt >= 2 * cus)
      return launch_gemm_cfg<AT, W_BF16, OT, false, 256, 256, 4, 2, 64, 2>(p, (mt + 1) / 2, stream);
    if (mt * nt >= cus) return launch_gemm_cfg<AT, W_BF16, OT, false, 128, 256, 2, 4, 64, 3>(p, mt, stream);
    if (mt * ((p.N + 127) / 128) * 2 > cus)
      return launch_gemm_cfg<AT, W_BF16, OT, false, 128, 128, 4, 2, 64, 4>(p, mt, stream);
    return launch_gemm_cfg<AT, W_BF16, OT, false, 64, 64, 2, 2, 64, 4>(p, (p.R + 63) / 64, stream);
  }
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
  const bool vec = K % MX4_BLOCK == 0 && aligned(y, 16), bf16 = dtype == SMAUL_DTYPE_BF16;
  constexpr int64_t per = 256 * MX4_U;
  const int64_t blocks = (rows * mx4_blocks(K) * 4 + per - 1) / per;
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "mx4_dequantize: too many values");
  const dim3 grid((unsigned)blocks), block(256);
  const bool nt = rows * K * (bf16 ? 2 : 4) >= MX4_NT_BYTES;
#define SMAUL_D(B, V, N)                                                                                       \
  hipLaunchKernelGGL((mx4_dequantize_kernel<B, V, N>), grid, block, 0, stream, (const uint32_t*)codes, scales, \
                     y, rows, K)
  if (bf16 && vec && nt) SMAUL_D(true, true, true);
  else if (bf16 && vec) SMAUL_D(true, true, false);
  else if (bf16) SMAUL_D(true, false, false);
  else if (vec && nt) SMAUL_D(false, true, true);
  else if (vec) SMAUL_D(false, true, false);
  else SMAUL_D(false, false, false);
#undef SMAUL_D
  return check_launch("mx4_dequantize_kernel");
}

int64_t smaul_mx4_linear_workspace_size(int64_t rows, int64_t in_f, int64_t out_f, int dtype, int act) {
  if (rows < 0 || in_f <= 0 || out_f <= 0 || !dtype_ok(dtype)) return -1;
  return linear_parts(rows, in_f, out_f, dtype, act).total;
}

int smaul_mx4_linear(const void* x, int dtype, const uint8_t* w, const uint8_t* s, void* y, int64_t rows,
                     int64_t in_f, int64_t out_f, int act, void* workspace, int64_t workspace_bytes,
                     hipStream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || in_f <= 0 || out_f <= 0 || (act != SMAUL_ACT_KEEP && act != SMAUL_ACT_MX4))
    return fail(SMAUL_ERR_INVALID, "mx4_linear: bad sizes, dtype or act");
  if (rows == 0) return SMAUL_OK;
  if (!x || !w || !s || !y) return fail(SMAUL_ERR_INVALID, "mx4_linear: null pointer");
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(y, 16))
    return fail(SMAUL_ERR_INVALID, "mx4_linear: x, y and the codes must be 16-byte aligned");
  const LinearParts q = linear_parts(rows, in_f, out_f, dtype, act);
  if (workspace_bytes < q.total || (q.total > 0 && (!workspace || !aligned(workspace, 256))))
    return fail(SMAUL_ERR_INVALID, "mx4_linear: workspace %lld < %lld bytes, or unaligned", (long long)workspace_bytes,
                (long long)q.total);
  const bool bf16 = dtype == SMAUL_DTYPE_BF16, mx4 = act == SMAUL_ACT_MX4, pad = in_f % MX4_STAGE != 0;
  const int at = mx4 ? A_MX4 : bf16 ? A_BF16 : A_F32;
  char* ws = (char*)workspace;
  Mx4Args p{};
  p.x = mx4 || (q.gemm && (pad || !bf16)) ? ws + q.x : x;
  p.xs = (uint8_t*)ws + q.xs;
  p.w = w;
  p.s = s;
  p.y = y;
  p.R = rows;
  p.K = in_f;
  p.N = out_f;
  p.E = 1;
  p.xvec = in_f % (bf16 ? 8 : 4) == 0;
  int rc = SMAUL_OK;
  if (q.gemm) {
    const int64_t ng = mx4_groups(in_f);
    Mx4Prep f{};
    f.m[0] = Mx4Weight{w, s, (uint32_t*)(ws + q.st), pad ? (uint4*)(ws + q.wp) : nullptr, out_f, in_f, 0};
    f.x = x;
    f.xo = ws + q.x;
    f.xst = (uint32_t*)(ws + q.xs);
    f.T = rows;
    f.K = in_f;
    f.xmode = mx4 ? P_ROUND : pad || !bf16 ? P_PAD : P_NONE;
    rc = launch_prep(f, dtype, 1, stream);
    p.s = (uint8_t*)ws + q.st;
    if (pad) p.w = (uint8_t*)ws + q.wp;
    p.K = ng * MX4_GROUP;
    p.ldx = mx4 ? ng * 4 : bf16 ? p.K : 3 * p.K;
    p.ldw = ng * 4;
    p.ldy = out_f;
    p.xrows = rows;
  } else if (mx4) {
    rc = launch_quantize(x, dtype, (uint8_t*)ws + q.x, (uint8_t*)ws + q.xs, rows, in_f, stream);
  }
  if (rc) return rc;
  const Mx4Slots few{};
  const Mx4Shape shape[] = {{rows, in_f, out_f, false}};
  p.tile = pick_tile(at, shape, 0);
  const int64_t bm = tile_bm(at, p.tile);
  return launch_linear(p, at, bf16 ? O_BF16 : O_F32, q.gemm ? nullptr : &few, (rows + bm - 1) / bm, stream);
}

int64_t smaul_mx4_backward_input_workspace_size(int64_t rows, int64_t in_f, int64_t out_f, int dtype) {
  if (rows < 0 || in_f <= 0 || out_f <= 0 || !dtype_ok(dtype)) return -1;
  return dx_parts(rows, in_f, out_f, dtype).total;
}

int smaul_mx4_backward_input(const void* g, int dtype, const uint8_t* w, const uint8_t* s, void* dx, int64_t rows,
                             int64_t in_f, int64_t out_f, void* workspace, int64_t workspace_bytes,
                             hipStream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || in_f <= 0 || out_f <= 0)
    return fail(SMAUL_ERR_INVALID, "mx4_backward_input: bad sizes or dtype");
  if (rows == 0) return SMAUL_OK;
  if (!g || !w || !s || !dx) return fail(SMAUL_ERR_INVALID, "mx4_backward_input: null pointer");
  if (!aligned(w, 16)) return fail(SMAUL_ERR_INVALID, "mx4_backward_input: codes must be 16-byte aligned");
  if (!aligned(g, 16) || !aligned(dx, 16))
    return fail(SMAUL_ERR_INVALID, "mx4_backward_input: g and dx must be 16-byte aligned");
  const DxParts q = dx_parts(rows, in_f, out_f, dtype);
  if (workspace_bytes < q.total || (q.total > 0 && (!workspace || !aligned(workspace, 256))))
    return fail(SMAUL_ERR_INVALID, "mx4_backward_input: workspace %lld < %lld bytes, or unaligned",
                (long long)workspace_bytes, (long long)q.total);
  const bool bf16 = dtype == SMAUL_DTYPE_BF16;
  if (!q.gemm) {
    const int64_t blocks = mx4_blocks(in_f);
    if (!grid_fits(blocks, 512)) return fail(SMAUL_ERR_UNSUPPORTED, "mx4_backward_input: too wide a weight");
    const bool vec = out_f % 8 == 0;
    auto* kernel = bf16  ? (vec ? &mx4_dx_stream_kernel<A_BF16, true, 8> : &mx4_dx_stream_kernel<A_BF16, false, 8>)
                   : vec ? &mx4_dx_stream_kernel<A_F32, true, 8>
                         : &mx4_dx_stream_kernel<A_F32, false, 8>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(512), 0, stream, g, w, s, dx, rows, in_f, out_f);
    return check_launch("mx4_dx_stream_kernel");
  }
  char* ws = (char*)workspace;
  Mx4Prep f{};
  f.x = g;
  f.xo = ws + q.g;
  f.T = rows;
  f.K = out_f;
  f.xmode = q.lay ? P_PAD : P_NONE;
  prep_rows(f, dtype);
  const int64_t blocks = f.xblocks + q.ldo / 64 * ((in_f + 63) / 64);
  if (!grid_fits(blocks, 256))
    return fail(SMAUL_ERR_UNSUPPORTED, "mx4_backward_input: too large a weight or gradient");
  auto* kernel = bf16 ? &mx4_turn_kernel<true> : &mx4_turn_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, f, w, s, (uint16_t*)(ws + q.wt), out_f, in_f,
                     q.ldo);
  int rc = check_launch("mx4_turn_kernel");
  if (rc) return rc;
  Mx4Args p{};
  p.x = q.lay ? ws + q.g : g;
  p.w = (uint8_t*)ws + q.wt;
  p.y = dx;
  p.R = rows;
  p.K = q.lay ? q.ldo : out_f;
  p.N = in_f;
  p.ldx = bf16 ? p.K : 3 * p.K;
  p.ldw = q.ldo;
  p.ldy = in_f;
  p.E = 1;
  return bf16 ? launch_dx<A_BF16, O_BF16>(p, stream) : launch_dx<A_F32, O_F32>(p, stream);
}

// The experts' workspace: the dispatch's tables and scratch, x as the products read
// it, the hidden rows, the weights' scales (and padded codes), the slots' outputs.
struct Mx4MoeParts {
  bool gemm;
  int64_t seg_off, tile_off, perm_row, perm_w, inv, scratch, scratch_bytes, xc, xs, hc, hs, st[3], wp[3], y, total;
};
static Mx4MoeParts mx4_moe_parts(int64_t T, int64_t d, int64_t h, int64_t E, int64_t k, int dtype, int act) {
  Mx4MoeParts q{};
  Parts w;
  const int64_t R = T * k, gd = mx4_groups(d), gh = mx4_groups(h);
  const bool mx4 = act == SMAUL_ACT_MX4, f32 = dtype == SMAUL_DTYPE_F32;
  const int64_t size = f32 ? 4 : 2, wide = f32 ? 6 : 2;  // bytes of a value, and of one that the GEMM reads
  q.gemm = T > ST_ROWS;
  if (q.gemm) {
    q.seg_off = w.take((E + 1) * 4);
    q.tile_off = w.take((E + 1) * 4);
    q.perm_row = w.take(R * 4);
    q.perm_w = w.take(R * 4);
    q.inv = w.take(R * 4);
    q.scratch_bytes = smaul_moe_dispatch_workspace_size(T, E);
    q.scratch = w.take(q.scratch_bytes);
    const bool pd = d % MX4_STAGE != 0, ph = h % MX4_STAGE != 0;
    q.xc = w.take(mx4 ? T * gd * 64 : pd || f32 ? T * gd * MX4_GROUP * wide : 0);
    q.xs = w.take(mx4 ? T * gd * 4 : 0);
    q.hc = w.take(mx4 ? R * gh * 64 : R * gh * MX4_GROUP * wide);
    q.hs = w.take(mx4 ? R * gh * 4 : 0);
    for (int j = 0; j < 3; ++j) {
      q.st[j] = w.take(E * (j < 2 ? h * gd : d * gh) * 4);
      q.wp[j] = w.take(j < 2 ? (pd ? E * h * gd * 64 : 0) : (ph ? E * d * gh * 64 : 0));
    }
  } else {
    q.xc = w.take(mx4 ? T * mx4_blocks(d) * 16 : 0);
    q.xs = w.take(mx4 ? T * mx4_blocks(d) : 0);
    q.hc = w.take(mx4 ? R * mx4_blocks(h) * 16 : R * h * size);
    q.hs = w.take(mx4 ? R * mx4_blocks(h) : 0);
  }
  q.y = w.take(R * d * (mx4 ? 2 : 4));
  q.total = w.at;
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
  if (!aligned(x, 16) || !aligned(gate_w, 16) || !aligned(up_w, 16) || !aligned(down_w, 16) || !aligned(out, 16))
    return fail(SMAUL_ERR_INVALID, "mx4_moe: x, out and the codes must be 16-byte aligned");
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
  const int at = mx4 ? A_MX4 : bf16 ? A_BF16 : A_F32;
  const int64_t R = T * k, gd = mx4_groups(d), gh = mx4_groups(h);
  const bool pd = d % MX4_STAGE != 0, ph = h % MX4_STAGE != 0;
  const Mx4Shape shapes[] = {{R, d, h, true}, {R, h, d, false}};
  const int tile = pick_tile(at, shapes, E);
  const int64_t bm = tile_bm(at, tile), m_tiles = (R + bm - 1) / bm + E;
  if (q.gemm && !(mx4 || T * (pd || !bf16 ? gd * MX4_GROUP : d) * (bf16 ? 2 : 6) < (1LL << 32)))
    return fail(SMAUL_ERR_UNSUPPORTED, "mx4_moe: more than 4 GiB of x");
  if (mx4 && T * gd * 64 >= (1LL << 32)) return fail(SMAUL_ERR_UNSUPPORTED, "mx4_moe: more than 4 GiB of codes of x");
  int rc = SMAUL_OK;
  if (q.gemm) {
    rc = smaul_moe_dispatch(topi, topw, counts, seg_off, tile_off, perm_row, (float*)(ws + q.perm_w), inv, T, E, k, bm,
                            ws + q.scratch, q.scratch_bytes, stream);
    if (rc) return rc;
  }
  Mx4Args p{};
  p.x = mx4 || (q.gemm && (pd || !bf16)) ? ws + q.xc : x;
  p.xs = (uint8_t*)ws + q.xs;
  p.row_idx = perm_row;
  p.w = gate_w;
  p.s = gate_s;
  p.w2 = up_w;
  p.s2 = up_s;
  p.y = ws + q.hc;
  p.ys = (uint8_t*)ws + q.hs;
  p.K = d;
  p.N = h;
  p.seg_off = seg_off;
  p.tile_off = tile_off;
  p.E = (int)E;
  p.tile = tile;
  p.xvec = d % 8 == 0;
  Mx4Args dn = p;
  dn.x = p.y;
  dn.xs = p.ys;
  dn.row_idx = nullptr;
  dn.w = down_w;
  dn.s = down_s;
  dn.y = ws + q.y;
  dn.K = h;
  dn.N = d;
  dn.xvec = h % (bf16 ? 8 : 4) == 0;
  if (q.gemm) {
    const uint8_t* w[3] = {gate_w, up_w, down_w};
    const uint8_t* s[3] = {gate_s, up_s, down_s};
    const uint8_t* at_w[3];
    const uint8_t* at_s[3];
    Mx4Prep f{};
    for (int j = 0; j < 3; ++j) {
      const bool pad = j < 2 ? pd : ph;
      f.m[j] = Mx4Weight{w[j], s[j], (uint32_t*)(ws + q.st[j]), pad ? (uint4*)(ws + q.wp[j]) : nullptr,
                         j < 2 ? h : d, j < 2 ? d : h, 0};
      at_w[j] = pad ? (uint8_t*)ws + q.wp[j] : w[j];
      at_s[j] = (uint8_t*)ws + q.st[j];
    }
    f.x = x;
    f.xo = ws + q.xc;
    f.xst = (uint32_t*)(ws + q.xs);
    f.T = T;
    f.K = d;
    f.xmode = mx4 ? P_ROUND : pd || !bf16 ? P_PAD : P_NONE;
    rc = launch_prep(f, dtype, E, stream);
    p.w = at_w[0];
    p.s = at_s[0];
    p.w2 = at_w[1];
    p.s2 = at_s[1];
    p.K = gd * MX4_GROUP;
    p.ldx = mx4 ? gd * 4 : bf16 ? p.K : 3 * p.K;
    p.ldw = gd * 4;
    p.ldy = mx4 ? gh * 4 : gh * MX4_GROUP * (bf16 ? 1 : 3);
    p.xrows = T;
    p.yrows = R;
    dn.w = at_w[2];
    dn.s = at_s[2];
    dn.K = gh * MX4_GROUP;
    dn.ldx = p.ldy;
    dn.ldw = gh * 4;
    dn.ldy = d;
    dn.xrows = R;
  } else if (mx4) {
    rc = launch_quantize(x, dtype, (uint8_t*)ws + q.xc, (uint8_t*)ws + q.xs, T, d, stream);
  }
  if (rc) return rc;
  // up to ST_ROWS tokens the products find their rows by themselves
  // The hidden rows as they are go on in x's type, as a SwiFFN's.  Of bf16 that is an error
  // as large as the result's own rounding (2.4e-3 against 64 bits; 1.7e-3 of hidden rows in
  // two bf16 terms, which take 27.8 us for 25.1 at 64 tokens to 2 of 8 experts, 1024 by
  // 2560, and 720 for 547 at 16384).
  Mx4Slots up{topi, topw, counts, (int)T, (int)k, 1}, down{topi, topw, nullptr, (int)T, (int)k, 0};
  const Mx4Slots* few = q.gemm ? nullptr : &up;
  rc = mx4 ? launch_product<A_MX4, O_MX4, true>(p, few, m_tiles, stream)
           : bf16 ? launch_product<A_BF16, O_BF16, true>(p, few, m_tiles, stream)
                  : launch_product<A_F32, O_F32, true>(p, few, m_tiles, stream);
  if (rc) return rc;
  rc = launch_linear(dn, at, mx4 ? O_BF16 : O_F32, q.gemm ? nullptr : &down, m_tiles, stream);
  if (rc) return rc;
  const int32_t* at_row = q.gemm ? inv : nullptr;
  return mx4 ? launch_combine<false, true>(ws + q.y, topi, topw, at_row, out, T, d, k, E, stream)
             : bf16 ? launch_combine<true, true>(ws + q.y, topi, topw, at_row, out, T, d, k, E, stream)
                    : launch_combine<true, false>(ws + q.y, topi, topw, at_row, out, T, d, k, E, stream);
}

}  // extern "C"
