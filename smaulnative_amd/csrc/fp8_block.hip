// fp8_block.hip -- rows in blocks of 128 E4M3 codes on MI355X (gfx950): quantisation,
// the product of such rows with such a weight, its input gradient, and the gated
// feed-forward block with its gradients.
//
//   y[r, n]  = sum_k x[r, k] W[n, k]
//   dx[r, k] = sum_n g[r, n] W[n, k]
//   block:   h = Q(silu(x Wg^T) * (x Wu^T)),  y = h Wd^T
//   its gradients, straight through the roundings: dh = dy Wd, dg = dh u silu'(g),
//   du = dh silu(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
#include <algorithm>
#include <utility>

#include "fp8_block.h"
#include "lds_dma.h"

using smaul::check_launch;
using smaul::cu_count;
using smaul::fail;
using smaul::grid_fits;

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------
// quantisation: 16 lanes a block, 8 values a lane.  Memory bounds it both ways: 32768 x 2048
// bf16 to codes 34 us, 5.9 TB/s, of fp32 55, 6.1; codes read back to bf16 31 us, 6.4 TB/s (the
// codes from the last cache).  8192 x 1024 bf16 5.8 us, 4.4 TB/s: a launch and two rounds of
// the workgroups that run at once, one chain of loads each.
// ---------------------------------------------------------------------------
// chunk i of rows of n: its row and place in it (a 64-bit division takes as long as the loads)
__device__ __forceinline__ void fb_place(int64_t i, int64_t n, int64_t rows, int64_t& row, int64_t& c) {
  row = rows * n < 1LL << 32 ? (int64_t)((uint32_t)i / (uint32_t)n) : i / n;
  c = i - row * n;
}

template <bool BF16>
__global__ void __launch_bounds__(256)
fb_quantize_kernel(const void* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t rows,
                   int64_t K) {
  const int64_t nb = fb_blocks(K), i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t row, c;
  fb_place(i, nb * 16, rows, row, c);
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
  int64_t row, c;
  fb_place(i, nb * 16, rows, row, c);
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
// Both sides' rows: codes with their scales, or bf16 (a row's bytes a multiple of 128).
enum { F_CODES = 0, F_BF16 = 1 };
// What a tile's sums become: bf16 or fp32 rows, the gated block's hidden rows as codes, or
// (sums dh) its dg and du by the factors that the forward pass kept, or a part of them
// (fp32, one of several slices of K).
enum { O_BF16 = 0, O_F32 = 1, O_GATED = 2, O_DGATED = 3, O_PART = 4, O_GATED_EXACT = 5 };  // the last: as O_GATED

struct FbArgs {
  const uint8_t* x;   // R rows of ldx bytes
  const uint8_t* xs;  // F_CODES: their scales, `words` dwords a row
  const uint8_t* w;   // N rows
  const uint8_t* s;
  const uint8_t* w2;  // O_GATED: up's (w, s are gate's)
  const uint8_t* s2;
  void* y;            // [R][N] (O_GATED: codes [R][fb_width(N)], O_DGATED: bf16 [R][2][ldh])
  uint8_t* ys;        // O_GATED: scales
  uint8_t* kept;      // O_GATED: what the gradients take, or null; O_DGATED: that
  int64_t R, N, ldx;  // ldx: of x and w, a multiple of 128
  int64_t ldh;        // O_DGATED: N to whole stages, zeros from N on
  int splits, per;    // slices of K, each of `per` stages and a y of its own (0: one)
  int words;
};

// The kept factors a = u silu'(g) and b = silu(g), 24 bits each (bf16 alone would add its
// rounding twice to the gradients').  Both passes have them in tiles of 32 rows by 32
// columns, 16 consecutive columns of row i in lane i or i + 32, so that is how they lie: a
// tile is 6 pieces of 16 bytes a lane (a's high halves, b's, a's third bytes, b's), each
// piece a whole KB of the 64 lanes.
constexpr int FB_KEPT = 6 * 1024;
__host__ __device__ __forceinline__ int64_t fb_kept_size(int64_t T, int64_t h) {
  return (T + 31) / 32 * (fb_width(h) / 32) * FB_KEPT;
}
// piece 0 of row `row`, columns n to n + 15, of h hidden columns
__device__ __forceinline__ int64_t fb_kept_at(int64_t row, int64_t n, int64_t h) {
  return (row / 32 * (fb_width(h) / 32) + n / 32) * FB_KEPT + (row % 32 + n / 16 % 2 * 32) * 16;
}

// a float's bits, its third byte to nearest (halves up); an infinity's sum keeps its other bytes
__device__ __forceinline__ uint32_t fb_bits24(float v) { return v == v ? __float_as_uint(v) + 0x80u : 0x7fc00000u; }
// 4 or 16 values: high halves and third bytes
__device__ __forceinline__ void fb_pack24(const float (&v)[4], uint2& hi, uint32_t& lo) {
  const uint32_t u[4] = {fb_bits24(v[0]), fb_bits24(v[1]), fb_bits24(v[2]), fb_bits24(v[3])};
  hi = make_uint2(__builtin_amdgcn_perm(u[1], u[0], 0x07060302u), __builtin_amdgcn_perm(u[3], u[2], 0x07060302u));
  lo = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0501u), __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0501u),
                             0x05040100u);
}
__device__ __forceinline__ void fb_pack24(const float (&v)[16], uint4 (&hi)[2], uint4& lo) {
  uint2 h[4];
  uint32_t l[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float f[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
    fb_pack24(f, h[q], l[q]);
  }
  hi[0] = make_uint4(h[0].x, h[0].y, h[1].x, h[1].y);
  hi[1] = make_uint4(h[2].x, h[2].y, h[3].x, h[3].y);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ void fb_unpack24(const uint4 (&hi)[2], const uint4& lo, float (&v)[16]) {
  const uint32_t h[8] = {hi[0].x, hi[0].y, hi[0].z, hi[0].w, hi[1].x, hi[1].y, hi[1].z, hi[1].w};
  const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
  for (int r = 0; r < 16; ++r)
    v[r] = __uint_as_float(__builtin_amdgcn_perm(h[r / 2], l[r / 4], (r & 1 ? 0x0706000cu : 0x0504000cu) | (r & 3) << 8));
}

// silu(g) u, u silu'(g) and silu(g)
__device__ __forceinline__ float fb_gated(float g, float u, float& a, float& b) {
  const float sig = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-g * 1.4426950408889634f));
  b = g * sig;
  a = u * (sig * fmaf(g, 1.0f - sig, 1.0f));
  return b * u;
}

// f(0), ..., f(N - 1), each with its number as a constant
template <class F, int... I>
__device__ __forceinline__ void fb_each(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void fb_each(F&& f) {
  fb_each(f, std::make_integer_sequence<int, N>{});
}

// K in stages of 128 (a block, 128-byte rows), codes brought to LDS by DMA, NS stages;
// scales in chunks of 16 stages, as many.  Roles: the weight's rows are the matrix instruction's
// rows and x's its columns, and row i of a 32 x 32 tile is given weight row 16 ((i / 4) %
// 2) + 4 (i / 8) + i % 4, so that the 16 sums of a lane are 16 consecutive outputs of one
// row of x.
template <int FMT, int BM, int BN, int WM, int WN, int NS>
struct FbCfg {
  static constexpr int NW = WM * WN, XB = BM * 128, WB = BN * 128, STAGE = XB + WB;
  static constexpr int X_INS = XB / (1024 * NW), W_INS = WB / (1024 * NW), S_INS = (BM + BN) / (16 * NW);
  static constexpr int SC = FMT == F_CODES ? (BM + BN) * 16 : 0;  // a chunk of scales: 4 dwords a row
  static constexpr int TT = BM / WM / 32, WT = BN / WN / 32;
  static constexpr int LDS = NS * (STAGE + SC);
  static_assert(XB % (1024 * NW) == 0 && WB % (1024 * NW) == 0 && (BM + BN) % (16 * NW) == 0 && BN % 16 == 0,
                "whole DMA instructions");
};

// ... and its kernel: a wave's part of LDS for the rows that leave (2 KB where two workgroups
// share a CU for it), the hidden rows' maxima.  PAIRED: two workgroups a CU.
template <int FMT, int OT, int BM, int BN, int WM, int WN, int NS>
struct FbProduct : FbCfg<FMT, BM, BN, WM, WN, NS> {
  using C = FbCfg<FMT, BM, BN, WM, WN, NS>;
  static constexpr bool GATED = OT == O_GATED || OT == O_GATED_EXACT, EXACT = OT == O_F32 || OT == O_GATED_EXACT;
  static constexpr bool SMALL = NS == 2 && BM * BN <= 128 * 128;
  static constexpr int OWN = GATED ? 0 : OT == O_BF16 && SMALL ? 2048 : 4096, AMAX = GATED ? BM * WN * 4 : 0;
  static constexpr int SMEM = C::LDS + C::NW * OWN + AMAX;
  static constexpr bool PAIRED = SMALL && 2 * SMEM <= 160 * 1024;
};

__device__ __forceinline__ int fb_perm(int i) { return ((i >> 2) & 1) * 16 + (i >> 3) * 4 + (i & 3); }

typedef int i32x8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8_t fb_operand(uint4 a, uint4 b) {
  i32x8_t r;
  r[0] = (int)a.x; r[1] = (int)a.y; r[2] = (int)a.z; r[3] = (int)a.w;
  r[4] = (int)b.x; r[5] = (int)b.y; r[6] = (int)b.z; r[7] = (int)b.w;
  return r;
}

// 8 codes -> 8 bf16 (exact), times s
__device__ __forceinline__ bf16x8_t fb_decode8(int lo, int hi, float s) {
  uint4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, s, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, s, true));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, s, false));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, s, true));
  return __builtin_bit_cast(bf16x8_t, r);
}

// sums stay in AGPRs up to here: moved out early they would not fit the other registers
__device__ __forceinline__ void fb_pin(f32x16_t& v) { asm volatile("" : "+a"(v)); }

// half q of an operand's 32 bytes, as bf16
__device__ __forceinline__ bf16x8_t fb_half(const i32x8_t& v, int q) {
  return __builtin_bit_cast(bf16x8_t, make_uint4((uint32_t)v[4 * q], (uint32_t)v[4 * q + 1], (uint32_t)v[4 * q + 2],
                                                 (uint32_t)v[4 * q + 3]));
}

// tile `lin` of m_tiles by n_tiles, in groups of 8 row tiles by all column tiles
__device__ __forceinline__ void fb_tile_at(int lin, int m_tiles, int n_tiles, int& mt, int& nt) {
  constexpr int GM = 8;
  const int g = lin / (GM * n_tiles), within = lin - g * GM * n_tiles, gm = min(GM, m_tiles - g * GM);
  mt = g * GM + within % gm;
  nt = within / gm;
}

// v_mfma_scale_f32_32x32x64_f8f6f4: lane i + 32 g has 32 values of row i and one scale
// byte for them.  It sums 32 bits wide, but 8 neighbouring products are first aligned to
// the largest of them and lose what is below 2^-13 of it: 1.5e-5 of a sum of normal values
// in the mean, a hundredth of bf16's own rounding.  fp32 results are not formed so, nor
// hidden rows as long as they are few, of which a value or a block's scale that is rounded
// to its other neighbour is seen in the block's output: their codes are decoded (exactly)
// and multiplied as bf16, at half the rate (16384 x 2048 -> 5120 to fp32 275 us, 1.25 PFLOP/s).
//
// The operands of a step (64 values) are read while the step before is multiplied, the first
// of a stage during the last of the stage before; by then every wave has the rest of its
// stage in registers, so that one barrier frees the buffer for the loads of the stage after
// the next.  A workgroup walks a band of tiles as one sequence of stages.
// Several products of one K (G of them) share the launch, one after the other in the band.
//
// 16384 x 2048 -> 5120 codes to bf16: 134 us, 2.6 PFLOP/s (many in a row 160: power).  Of a 256 x
// 256 tile's 29 us the 16 stages are 24.5, 2.8 PFLOP/s, where the instruction alone reaches 4.0 on
// such values (and 4.9 on zeros): one wave a SIMD, to which a stage's two barriers and waits are
// exposed; the epilogue is the rest.  bf16, 8192 x 5120 -> 1024: 73 us, 1.2 PFLOP/s of 1.95, in a
// training step, warm, 86.
template <int G>
struct FbBatch {
  FbArgs p[G];
};
template <int FMT, int OT, int BM, int BN, int WM, int WN, int NS, int G>
__global__ void __launch_bounds__(WM * WN * 64, (FbProduct<FMT, OT, BM, BN, WM, WN, NS>::PAIRED ? 2 : 1))
fb_product_kernel(FbBatch<G> batch) {
  using C = FbProduct<FMT, OT, BM, BN, WM, WN, NS>;
  constexpr bool GATED = C::GATED, EXACT = C::EXACT;
  constexpr int TT = C::TT, WT = C::WT, BNO = GATED ? BN / 2 : BN, NW = C::NW, OWN = C::OWN;
  static_assert(!GATED || BNO == FB_BLOCK, "a tile of hidden rows is a block");
  __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, g = lane >> 5, l32 = lane & 31;
  const uint32_t lds0 = lds_offset(&smem[0]);
  // slices of K: only where every workgroup has one tile
  constexpr bool SPLITS = NS == 4 && G == 1 && (OT == O_F32 || OT == O_PART);
  const bool split = SPLITS && batch.p[0].per > 0;
  int nk = (int)(batch.p[0].ldx / 128), k0 = 0;
  int64_t part = 0;
  auto tiles = [&](int q) __attribute__((always_inline)) -> int {
    return (int)((batch.p[q].R + BM - 1) / BM * ((batch.p[q].N + BNO - 1) / BNO));
  };
  // tile `at` of all: its product, and its place there
  auto locate = [&](int at, int& mt, int& nt) __attribute__((always_inline)) -> int {
    int q = 0;
    if (split) at %= tiles(0);
#pragma unroll
    for (int j = 0; j + 1 < G; ++j)
      if (q == j && at >= tiles(j)) {
        at -= tiles(j);
        q = j + 1;
      }
    fb_tile_at(at, (int)((batch.p[q].R + BM - 1) / BM), (int)((batch.p[q].N + BNO - 1) / BNO), mt, nt);
    return q;
  };

  // XCD x (workgroup b runs on XCD b % 8) takes a contiguous band of the tiles, as long as
  // its share of the workgroups
  int total = 0;
#pragma unroll
  for (int j = 0; j < G; ++j) total += tiles(j);
  if (split) total *= batch.p[0].splits;
  const int wgs = gridDim.x, xcd = (int)blockIdx.x % 8, step = (wgs - xcd + 7) / 8;
  const int before = xcd * (wgs / 8) + min(xcd, wgs % 8);  // workgroups of the XCDs before
  const int last = (int)((int64_t)total * (before + step) / wgs);
  int lin = (int)((int64_t)total * before / wgs) + (int)blockIdx.x / 8;
  if (split && lin < last) {
    const int t = tiles(0), slice = lin / t;
    k0 = slice * batch.p[0].per;
    nk = min(nk - k0, batch.p[0].per);
    part = slice * batch.p[0].R * batch.p[0].N;
  }
  if (lin >= last) return;

  // where a lane's loads of a tile read: 32-bit offsets from its first rows; rows past the
  // end read the last one, their sums are not stored
  const uint8_t *X, *W, *XS, *WS;  // gate's; up's stand as far from them as the matrices from each other
  const int64_t to_w2 = GATED ? batch.p[0].w2 - batch.p[0].w : 0, to_s2 = GATED ? batch.p[0].s2 - batch.p[0].s : 0;
  uint32_t x_off[C::X_INS], w_off[C::W_INS], s_off[C::S_INS];
  // staged weight row r, from the tile's first: tiles of 32 (gate's, then up's), permuted
  auto w_row = [&](int r, int left) __attribute__((always_inline)) -> int {
    int t = r >> 5;
    if (GATED) t = t >= BN / 64 ? t - BN / 64 : t;
    return min(t * 32 + fb_perm(r & 31), left);
  };
  const uint32_t ld = (uint32_t)batch.p[0].ldx, sl = (uint32_t)batch.p[0].words * 4;
  bool offsets = true;  // are to be computed
  auto source = [&](int at) __attribute__((always_inline)) {
    int mt, nt;
    const FbArgs& p = batch.p[locate(at, mt, nt)];
    const int64_t row0 = (int64_t)mt * BM, n0 = (int64_t)nt * BNO;
    const int xleft = (int)min<int64_t>(p.R - 1 - row0, BM - 1), wleft = (int)min<int64_t>(p.N - 1 - n0, BNO - 1);
    X = p.x + row0 * ld + (int64_t)k0 * 128;
    if (FMT == F_CODES) XS = p.xs + row0 * sl + k0;
    W = p.w + n0 * ld + (int64_t)k0 * 128;
    if (FMT == F_CODES) WS = p.s + n0 * sl + k0;
    const bool ragged = xleft < BM - 1 || wleft < BNO - 1;
    if (!ragged && !offsets) return;  // a whole tile's offsets are there from the one before
    offsets = ragged;
    int me = lane;  // nothing of this is kept in registers from tile to tile
    asm volatile("" : "+v"(me));
#pragma unroll
    for (int a = 0; a < C::X_INS; ++a) {
      const int r = (wave * C::X_INS + a) * 8 + me / 8;
      x_off[a] = (uint32_t)min(r, xleft) * ld + (uint32_t)((me % 8 ^ swz_a(r)) * 16);
    }
#pragma unroll
    for (int b = 0; b < C::W_INS; ++b) {
      const int r = (wave * C::W_INS + b) * 8 + me / 8;
      w_off[b] = (uint32_t)w_row(r, wleft) * ld + (uint32_t)((me % 8 ^ swz_a(r)) * 16);
    }
#pragma unroll
    for (int i = 0; i < C::S_INS; ++i) {
      const int r = (wave * C::S_INS + i) * 16 + me / 4;
      s_off[i] = (uint32_t)(r < BN ? w_row(r, wleft) : min(r - BN, xleft)) * sl;
    }
  };
  // the sequence's next stage to load, of this tile or one after (behind the last tile its
  // stages again, into buffers that nobody reads): its scales where a chunk begins, its
  // codes one DMA instruction at a time
  constexpr int INS = C::X_INS + C::W_INS;
  int load_at = lin, load_k = nk, load_chunk = 0;
  auto load_begin = [&]() __attribute__((always_inline)) {
    if (load_k == nk) {
      if (load_at < last) source(load_at);
      load_at += step;
      load_k = 0;
    }
    if (FMT == F_CODES && load_k % 16 == 0) {
      const int word = min(load_k / 4 + lane % 4, batch.p[0].words - 1 - k0 / 4) * 4;
#pragma unroll
      for (int i = 0; i < C::S_INS; ++i) {
        const int r = (wave * C::S_INS + i) * 16;
        const uint8_t* from = WS + (GATED && r >= BN / 2 ? to_s2 : 0);
        if (r >= BN) from = XS;
        dma4(from, s_off[i] + word, lds0 + NS * C::STAGE + load_chunk * C::SC + (wave * C::S_INS + i) * 256);
      }
      load_chunk = load_chunk + 1 == NS ? 0 : load_chunk + 1;
    }
  };
  auto load_one = [&](int buf, int q) __attribute__((always_inline)) {
    const uint32_t l = lds0 + (uint32_t)(buf * C::STAGE);
    const int64_t at = (int64_t)load_k * 128;
    if (q < C::X_INS) {
      dma16(X + at, x_off[q < C::X_INS ? q : 0], l + (wave * C::X_INS + q) * 1024);
    } else {
      const int b = q - C::X_INS, r = (wave * C::W_INS + b) * 8;
      dma16(W + at + (GATED && r >= BN / 2 ? to_w2 : 0), w_off[b < 0 ? 0 : b], l + C::XB + (wave * C::W_INS + b) * 1024);
    }
  };
#pragma unroll
  for (int b = 0; b < NS; ++b) {
    load_begin();
#pragma unroll
    for (int q = 0; q < INS; ++q) load_one(b, q);
    ++load_k;
  }
  // (a chunk of scales stands before its stage's codes)
  wait_vm<INS * (NS - 1)>();
  __syncthreads();

  // staged row of weight tile j of this wave: its gate tiles, then its up tiles
  auto w_tile = [&](int j) __attribute__((always_inline)) -> int {
    if constexpr (GATED)
      return j < WT / 2 ? wn * (BN / WN / 2) + j * 32 : BN / 2 + wn * (BN / WN / 2) + (j - WT / 2) * 32;
    else return wn * (BN / WN) + j * 32;
  };
  i32x8_t wf[2][WT], xf[2][TT];
  uint32_t sw[WT], sx[TT], nw[WT], nx_[TT];
  // this lane's 16 bytes of a stage's first step; the others are an XOR away.  Tiles are 32
  // rows apart, which the swizzle does not see.
  const uint32_t first = (uint32_t)(l32 * 128 + (2 * g ^ swz_a(l32)) * 16);
  constexpr int READS = 2 * (TT + WT), S = TT * WT;
  auto read_one = [&](int buf, int u, int q) __attribute__((always_inline)) {  // half q % 2 of operand q / 2 of step u
    const char* at = smem + buf * C::STAGE + (first ^ (uint32_t)(u * 64 + q % 2 * 16));
    const int o = q / 2, j = o - TT;
    const uint4 v = o < TT ? *(const uint4*)(at + (wm * (BM / WM) + o * 32) * 128)
                           : *(const uint4*)(at + C::XB + w_tile(j) * 128);
    i32x8_t& r = o < TT ? xf[u][o < TT ? o : 0] : wf[u][j < 0 ? 0 : j];
    r[q % 2 * 4] = (int)v.x; r[q % 2 * 4 + 1] = (int)v.y; r[q % 2 * 4 + 2] = (int)v.z; r[q % 2 * 4 + 3] = (int)v.w;
  };
  // four stages' scales of this lane's rows, from the chunk
  auto read_scales = [&](int chunk, int word) __attribute__((always_inline)) {
    const char* at = smem + NS * C::STAGE + chunk * C::SC + l32 * 16 + word * 4;
#pragma unroll
    for (int j = 0; j < WT; ++j) nw[j] = *(const uint32_t*)(at + w_tile(j) * 16);
#pragma unroll
    for (int i = 0; i < TT; ++i) nx_[i] = *(const uint32_t*)(at + (BN + wm * (BM / WM) + i * 32) * 16);
  };
  f32x16_t acc[WT][TT];
  // product s of step u
  auto multiply = [&](int u, int s, bool fresh) __attribute__((always_inline)) {
    const f32x16_t zero = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    const int j = s / TT, i = s % TT;
    const f32x16_t c = fresh && u == 0 ? zero : acc[j][i];
    if constexpr (FMT == F_BF16) {
      acc[j][i] = c;
#pragma unroll
      for (int q = 0; q < 2; ++q)
        acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb_half(wf[u][j], q), fb_half(xf[u][i], q), acc[j][i], 0, 0, 0);
    } else if constexpr (EXACT) {
      acc[j][i] = c;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bf16x8_t x = fb_decode8(xf[u][i][2 * q], xf[u][i][2 * q + 1], fb_scale(sx[i] & 255u));
        const bf16x8_t w = fb_decode8(wf[u][j][2 * q], wf[u][j][2 * q + 1], fb_scale(sw[j] & 255u));
        acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, x, acc[j][i], 0, 0, 0);
      }
    } else {
      acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[u][j], xf[u][i], c, 0, 0, 0, (int)sw[j], 0,
                                                                 (int)sx[i]);
    }
  };
  auto pin = [&](int n) __attribute__((always_inline)) {  // the first n products stay on their side of a branch or barrier
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (s < n) fb_pin(acc[s / TT][s % TT]);
  };
  int buf = 0, chunk = 0;
  // One stage: 2 S products, the rest issued in their shadow.  The second step's operands
  // are read first; from product B1 on no wave reads this buffer any more, and the loads of
  // the stage that takes its place follow, spread out so that they do not queue; from product
  // B2 on the next stage's first operands are read, behind a wait that leaves the loads of
  // later stages (of this stage's DONE by then) in flight.
  constexpr int B1 = S * 5 / 8, B2 = S + S * 5 / 16, SPAN = 2 * S - 2 - B1;
  constexpr int STORED = GATED ? TT * WT / 2 : TT * WT * (OT == O_BF16 ? 2 : 4);  // instructions of a whole tile
  int stored = 0;
  constexpr int DONE = ((B2 - 1 - B1) * INS + SPAN - 1) / SPAN;  // of products B1 to B2 - 2
  constexpr int FLIGHT = DONE + (NS - 2) * INS;  // loads behind those of the next stage
  static_assert(FLIGHT < 64, "vmcnt range");
  auto stage = [&](int kt, bool fresh) __attribute__((always_inline)) {
    const int sh = kt % 4 * 8, next = kt + 1 == nk ? 0 : kt + 1;
#pragma unroll
    for (int j = 0; j < WT && FMT == F_CODES; ++j) sw[j] = nw[j] >> sh;
#pragma unroll
    for (int i = 0; i < TT && FMT == F_CODES; ++i) sx[i] = nx_[i] >> sh;
    if (next % 16 == 0) chunk = chunk + 1 == NS ? 0 : chunk + 1;
    const int after = buf + 1 == NS ? 0 : buf + 1;
    fb_each<2 * S>([&](auto number) __attribute__((always_inline)) {
      constexpr int s = number;
      if constexpr (s == B1) {
        pin(fresh ? B1 : S);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        load_begin();
        __builtin_amdgcn_sched_barrier(0);
      }
      multiply(s / S, s % S, fresh);
      if constexpr (s == B2 - 1) {
        __builtin_amdgcn_sched_barrier(0);
        // memory operations are done in order: behind a tile's stores, of which `stored` at
        // least were issued, the loads before them are waited for alone
        if (fresh && stored) wait_vm<(FLIGHT + STORED < 63 ? FLIGHT + STORED : 63)>();
        else wait_vm<FLIGHT>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (FMT == F_CODES) read_scales(chunk, next / 4 % 4);
      }
      fb_each<READS>([&](auto part) __attribute__((always_inline)) {
        constexpr int q = part;
        if constexpr (q * (S / 2) / READS == s) read_one(buf, 1, q);
        if constexpr (B2 + q * (2 * S - B2) / READS == s) read_one(after, 0, q);  // behind the last tile: unused
      });
      fb_each<INS>([&](auto part) __attribute__((always_inline)) {
        constexpr int q = part;
        if constexpr (B1 + q * SPAN / INS == s) load_one(buf, q);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    ++load_k;
    buf = after;
  };

#pragma unroll
  for (int q = 0; q < READS; ++q) read_one(0, 0, q);
  if constexpr (FMT == F_CODES) read_scales(0, 0);
  for (; lin < last; lin += step) {
    stage(0, true);
    for (int kt = 1; kt < nk; ++kt) stage(kt, false);
    pin(S);
    int mt, nt;
    const FbArgs& p = batch.p[locate(lin, mt, nt)];
    const int64_t row0 = (int64_t)mt * BM, n0 = (int64_t)nt * BNO;
    const int rows = (int)min<int64_t>(BM, p.R - row0);
    int el = lane;  // the stores' addresses are not kept in registers across the loop
    asm volatile("" : "+v"(el));
    const int eg = el >> 5, e32 = el & 31;
    if constexpr (GATED) {
      constexpr int HT = WT / 2;
      float* sh = (float*)(smem + C::LDS);
      const int64_t nb = fb_blocks(p.N);
      float top[TT];
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const int lr = wm * (BM / WM) + i * 32 + e32;
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < HT; ++j) {
          const int64_t n = n0 + wn * (BNO / WN) + j * 32 + eg * 16;
          const int left = (int)min<int64_t>(p.N - n, 16);
          fb_pin(acc[j][i]);
          fb_pin(acc[j + HT][i]);
          float v[16], a[16], b[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) v[r] = fb_gated(acc[j][i][r], acc[j + HT][i][r], a[r], b[r]);
          if (n0 + BNO > p.N) {  // past N: copies of the last row's
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] = r < left ? v[r] : 0.0f;
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            acc[j][i][r] = v[r];
            m = __builtin_elementwise_maximum(m, __builtin_fabsf(v[r]));  // NaN stays NaN
          }
          fb_pin(acc[j][i]);
          if (p.kept && lr < rows) {  // 8192 tokens, 1024 by 2560: 91 us with down for 74 without
            uint4 hi[2], lo;
            uint4* to = (uint4*)(p.kept + fb_kept_at(row0 + lr, n, p.N));  // pieces are 64 of these apart
            fb_pack24(a, hi, lo);
            to[0] = hi[0];
            to[64] = hi[1];
            to[256] = lo;
            fb_pack24(b, hi, lo);
            to[128] = hi[0];
            to[192] = hi[1];
            to[320] = lo;
          }
        }
        m = __builtin_elementwise_maximum(m, __shfl_xor(m, 32, 64));
        top[i] = m;
        if (WN > 1 && eg == 0) sh[lr * WN + wn] = m;
      }
      if constexpr (WN > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int q = 0; q < WN; ++q)
            top[i] = __builtin_elementwise_maximum(top[i], sh[(wm * (BM / WM) + i * 32 + e32) * WN + q]);
      }
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const int lr = wm * (BM / WM) + i * 32 + e32;
        const uint32_t byte = fb_scale_byte(__float_as_uint(top[i]) & 0x7fffffffu);
        if (lr < rows) {
#pragma unroll
          for (int j = 0; j < HT; ++j) {
            fb_pin(acc[j][i]);
            float v[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] = acc[j][i][r];
            const uint2 lo = fb_encode8(v, byte), hi = fb_encode8(v + 8, byte);
            *(uint4*)((uint8_t*)p.y + (row0 + lr) * nb * FB_BLOCK + n0 + wn * (BNO / WN) + j * 32 + eg * 16) =
                make_uint4(lo.x, lo.y, hi.x, hi.y);
          }
          if (wn == 0 && eg == 0) {
            uint8_t* s = p.ys + (row0 + lr) * ((nb + 3) / 4 * 4);
            s[nt] = (uint8_t)byte;
            if (nt + 1 == nb)
              for (int64_t q = nb; q < (nb + 3) / 4 * 4; ++q) s[q] = 0;
          }
        }
      }
      if constexpr (WN > 1) __syncthreads();  // the maxima's LDS is free for the next tile
      stored = rows == BM ? STORED : 0;
    } else if constexpr (OT == O_DGATED) {
      // 64-byte pieces of dg and of du, each through 2 KB of LDS of the wave's own; the factors
      // of the next AHEAD units of 16 values are on their way while these are multiplied (8192
      // tokens, 1024 by 2560: 82 us, one unit ahead 100; the product alone 35, the bytes 45)
      constexpr int AHEAD = TT * WT > 8 ? 2 : 3, UNITS = TT * WT;
      char* own = smem + C::LDS + wave * OWN;
      auto place = [&](int m, int r, int c) __attribute__((always_inline)) -> char* {
        return own + m * 2048 + r * 64 + (c ^ (r / 2 & 3)) * 16;
      };
      const int left = rows - wm * (BM / WM);
      const int64_t w0 = n0 + wn * (BN / WN), r0 = row0 + wm * (BM / WM);
      const int64_t last_row = (p.R - 1) / 32 * 32, last_col = fb_width(p.N) - 32;  // tiles there are
      uint4 rec[AHEAD + 1][6];
      auto factors = [&](int u, uint4 (&to)[6]) __attribute__((always_inline)) {
        const uint4* at = (const uint4*)(p.kept + fb_kept_at(min(r0 + u / WT * 32, last_row), min(w0 + u % WT * 32, last_col),
                                                             p.N)) + el;
        to[0] = at[0]; to[1] = at[64]; to[2] = at[128]; to[3] = at[192]; to[4] = at[256]; to[5] = at[320];
      };
      if (left > 0) {
        fb_each<(AHEAD < UNITS ? AHEAD : UNITS)>([&](auto unit) __attribute__((always_inline)) {
          factors(unit, rec[unit]);
        });
        fb_each<UNITS>([&](auto unit) __attribute__((always_inline)) {
          constexpr int u = unit, i = u / WT, j = u % WT, at = u % (AHEAD + 1);
          if constexpr (u + AHEAD < UNITS) factors(u + AHEAD, rec[(u + AHEAD) % (AHEAD + 1)]);
          const uint4 ah[2] = {rec[at][0], rec[at][1]}, bh[2] = {rec[at][2], rec[at][3]}, al = rec[at][4], bl = rec[at][5];
          float a[16], b[16];
          fb_unpack24(ah, al, a);
          fb_unpack24(bh, bl, b);
          fb_pin(acc[j][i]);
          const f32x16_t v = acc[j][i];
          const int in = (int)min<int64_t>(p.N - (w0 + j * 32 + eg * 16), 16);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            a[r] = r < in ? v[r] * a[r] : 0.0f;
            b[r] = r < in ? v[r] * b[r] : 0.0f;
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int k = 8 * q;
            *(uint4*)place(0, e32, 2 * eg + q) = make_uint4(pack_bf16(a[k], a[k + 1]), pack_bf16(a[k + 2], a[k + 3]),
                                                            pack_bf16(a[k + 4], a[k + 5]), pack_bf16(a[k + 6], a[k + 7]));
            *(uint4*)place(1, e32, 2 * eg + q) = make_uint4(pack_bf16(b[k], b[k + 1]), pack_bf16(b[k + 2], b[k + 3]),
                                                            pack_bf16(b[k + 4], b[k + 5]), pack_bf16(b[k + 6], b[k + 7]));
          }
          __builtin_amdgcn_wave_barrier();
          const int64_t n = w0 + j * 32 + el % 4 * 8;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int tr = h * 16 + el / 4;
            const uint4 g = *(const uint4*)place(0, tr, el % 4), t = *(const uint4*)place(1, tr, el % 4);
            if (i * 32 + tr < left && n < p.ldh) {
              uint16_t* at = (uint16_t*)p.y + (r0 + i * 32 + tr) * 2 * p.ldh + n;
              *(uint4*)at = g;
              *(uint4*)(at + p.ldh) = t;
            }
          }
          __builtin_amdgcn_wave_barrier();
        });
      }
      stored = 0;
    } else {
      // rows leave 32 at a time, as whole lines (halves from 2 KB), through LDS of the wave's
      // own, 16-byte chunks changing places by the row; its LDS accesses are done in order
      char* own = smem + C::LDS + wave * OWN;
      constexpr int ES = OT == O_BF16 ? 2 : 4, RB = OWN / 32, CH = RB / 16, UJ = RB / 32 / ES, UNITS = TT * WT / UJ;
      auto place = [&](int r, int c) __attribute__((always_inline)) -> char* {
        return own + r * RB + (c ^ (CH == 8 ? r & 7 : r / 2 & 3)) * 16;
      };
      // of the whole workgroup: its offsets are 32 bits, up to 31 rows and a piece of one
      const int64_t row_bytes = p.N * ES;
      const bool whole = n0 + BN <= p.N && p.N % (16 / ES) == 0 && row_bytes < 1LL << 27;
      const uint32_t ldy = (uint32_t)row_bytes;
      const int left = rows - wm * (BM / WM);  // rows of this wave's
      char* out = (char*)p.y + (part + (row0 + wm * (BM / WM)) * p.N + n0 + wn * (BN / WN)) * ES;
      uint4 d0, d1, d2, d3;
      auto to_lds = [&](int i, int j) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < UJ; ++h) {
          fb_pin(acc[j + h][i]);
          const f32x16_t v = acc[j + h][i];
#pragma unroll
          for (int q = 0; q < ES; ++q) {
            const int c = h * 4 + ES * eg + q, r = q * (16 / ES);
            uint4 u;
            if constexpr (OT == O_BF16)
              u = make_uint4(pack_bf16(v[r], v[r + 1]), pack_bf16(v[r + 2], v[r + 3]), pack_bf16(v[r + 4], v[r + 5]),
                             pack_bf16(v[r + 6], v[r + 7]));
            else
              u = make_uint4(__float_as_uint(v[r]), __float_as_uint(v[r + 1]), __float_as_uint(v[r + 2]),
                             __float_as_uint(v[r + 3]));
            *(uint4*)place(e32, c) = u;
          }
        }
        __builtin_amdgcn_wave_barrier();
      };
      if (whole) {
        auto store = [&](int u) __attribute__((always_inline)) {
          const int r = u / (WT / UJ) * 32 + el / CH;
          char* at = out + (int64_t)(u / (WT / UJ) * 32) * ldy + u % (WT / UJ) * RB;
          const uint32_t o = (uint32_t)(el / CH) * ldy + el % CH * 16;
          if (r < left) *(uint4*)(at + o) = d0;
          if (r + 64 / CH < left) *(uint4*)(at + o + 64 / CH * ldy) = d1;
          if constexpr (CH == 8) {
            if (r + 16 < left) *(uint4*)(at + o + 16 * ldy) = d2;
            if (r + 24 < left) *(uint4*)(at + o + 24 * ldy) = d3;
          }
        };
        fb_each<UNITS + 1>([&](auto unit) __attribute__((always_inline)) {  // stored while the next is read
          constexpr int u = unit;
          if constexpr (u < UNITS) to_lds(u / (WT / UJ), u % (WT / UJ) * UJ);
          if constexpr (u > 0) store(u - 1);
          if constexpr (u < UNITS) {
            const char* at = place(el / CH, el % CH);  // 8 rows and more apart, which the places do not see
            d0 = *(const uint4*)at;
            d1 = *(const uint4*)(at + 1024);
            if constexpr (CH == 8) {
              d2 = *(const uint4*)(at + 2048);
              d3 = *(const uint4*)(at + 3 * 1024);
            }
            __builtin_amdgcn_wave_barrier();
          }
        });
      } else {  // rows of any alignment and width, the last columns one by one
        fb_each<UNITS>([&](auto unit) __attribute__((always_inline)) {
          constexpr int u = unit, c0 = u % (WT / UJ) * (RB / ES);
          to_lds(u / (WT / UJ), u % (WT / UJ) * UJ);
          const int n = (int)min<int64_t>(p.N - n0 - wn * (BN / WN) - c0, RB / ES) - el % CH * (16 / ES);
#pragma nounroll
          for (int h = 0; h < CH / 2; ++h) {
            const int tr = h * (64 / CH) + el / CH, r = u / (WT / UJ) * 32 + tr;
            const char* v = place(tr, el % CH);
            char* at = out + r * row_bytes + (c0 + el % CH * (16 / ES)) * ES;
            if (r >= left) continue;
            if (n >= 16 / ES) {
              const uint4 w = *(const uint4*)v;
              if constexpr (OT == O_BF16) *(fb_u32x4_at2*)at = (fb_u32x4_at2){w.x, w.y, w.z, w.w};
              else *(fb_u32x4_at4*)at = (fb_u32x4_at4){w.x, w.y, w.z, w.w};
            } else {
#pragma nounroll
              for (int e = 0; e < n; ++e) {
                if constexpr (OT == O_BF16) ((uint16_t*)at)[e] = ((const uint16_t*)v)[e];
                else ((float*)at)[e] = ((const float*)v)[e];
              }
            }
          }
          __builtin_amdgcn_wave_barrier();
        });
      }
      stored = whole && rows == BM ? STORED : 0;
    }
  }
  wait_vm<0>();
}

template <int FMT, int OT, int BM, int BN, int WM, int WN, int NS, int G>
int launch_product_cfg(const FbBatch<G>& b, hipStream_t stream) {
  constexpr int BNO = OT == O_GATED || OT == O_GATED_EXACT ? BN / 2 : BN;
  int64_t tiles = 0;
  for (const FbArgs& p : b.p) {
    const int64_t mt = (p.R + BM - 1) / BM, nt = (p.N + BNO - 1) / BNO;
    if (mt > 2147483647LL || nt > 2147483647LL || mt * nt > 2147483647LL)
      return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block product: too many tiles");
    tiles += mt * nt * (p.per ? p.splits : 1);
  }
  if ((BM > BN ? BM : BN) * b.p[0].ldx >= 1LL << 32)
    return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block product: rows too wide");
  if (tiles > 2147483647LL) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block product: too many tiles");
  const int64_t wgs = cu_count() * (FbProduct<FMT, OT, BM, BN, WM, WN, NS>::PAIRED ? 2 : 1);
  hipLaunchKernelGGL((fb_product_kernel<FMT, OT, BM, BN, WM, WN, NS, G>), dim3((unsigned)(tiles < wgs ? tiles : wgs)),
                     dim3(WM * WN * 64), 0, stream, b);
  return check_launch("fb_product_kernel");
}

// Tiles that fill the chip, by the rounds they take: what a stage of a round of the CUs
// takes and what the rest of its tiles does (10 ns), times the rounds.  The 128 x 128 tile
// mostly runs two a CU, in rounds of twice the CUs, a last round of no more than one a CU in
// `one`; a last round that leaves CUs idle has a higher clock, up to 1.7 times.
struct FbTile {
  int bm, bn, one, two, rest;  // two: 0 where a CU takes them one by one
};
constexpr FbTile ROW_TILES[] = {{256, 256, 153, 0, 490}, {128, 256, 85, 0, 300}, {128, 128, 52, 105, 160}, {64, 128, 37, 0, 150}};
// decoded codes (fp32 results): 128 values a stage at the bf16 rate, and scales and fp32 rows
// together leave LDS for one workgroup only
constexpr FbTile EXACT_TILES[] = {{256, 256, 275, 0, 650}, {128, 256, 160, 0, 300}, {128, 128, 101, 0, 200}, {64, 128, 70, 0, 100}};
constexpr FbTile DGATED_TILES[] = {{256, 256, 153, 0, 1400}, {128, 256, 85, 0, 800}, {128, 128, 52, 105, 500}, {64, 128, 37, 0, 300}};
constexpr FbTile GATED_TILES[] = {{256, 256, 153, 0, 900}, {128, 256, 85, 0, 500}, {64, 256, 60, 0, 300}};

template <int N, int G>
int pick_tile(const FbTile (&tiles)[N], const FbBatch<G>& batch, bool gated) {
  const int64_t cus = cu_count(), nk = batch.p[0].ldx / 128;
  int best = 0;
  double least = 0.0;
  for (int i = 0; i < N; ++i) {
    const FbTile& t = tiles[i];
    const int64_t bn = gated ? t.bn / 2 : t.bn;
    int64_t n = 0;
    for (const FbArgs& p : batch.p) n += (p.R + t.bm - 1) / t.bm * ((p.N + bn - 1) / bn);
    const int64_t round = t.two ? 2 * cus : cus, full = n / round, left = n % round;
    const double whole = (double)(nk * (t.two ? t.two : t.one) + t.rest);
    double last = whole * (0.6 + 0.4 * (double)left / (double)round);
    if (t.two && left <= cus) last = (double)(nk * t.one + t.rest);
    const double cost = (double)full * whole + (left ? last : 0.0);
    if (i == 0 || cost < least) {
      best = i;
      least = cost;
    }
  }
  return best;
}

template <int FMT, int OT, int G>
int launch_products(const FbBatch<G>& b, hipStream_t stream) {
  if constexpr (OT == O_GATED_EXACT) {
    return launch_product_cfg<FMT, OT, 64, 256, 1, 4, 3>(b, stream);
  } else if constexpr (OT == O_GATED) {
    switch (pick_tile(GATED_TILES, b, true)) {
      case 0: return launch_product_cfg<FMT, OT, 256, 256, 2, 2, 2>(b, stream);
      case 1: return launch_product_cfg<FMT, OT, 128, 256, 2, 2, 2>(b, stream);
      default: return launch_product_cfg<FMT, OT, 64, 256, 1, 4, 3>(b, stream);
    }
  } else {
    constexpr auto& tiles = OT == O_DGATED ? DGATED_TILES : FMT == F_CODES && OT == O_F32 ? EXACT_TILES : ROW_TILES;
    static_assert(FbProduct<FMT, OT, 128, 128, 2, 2, 2>::PAIRED == (tiles[2].two > 0), "rounds as the CUs take them");
    switch (pick_tile(tiles, b, false)) {
      case 0: return launch_product_cfg<FMT, OT, 256, 256, 2, 2, 2>(b, stream);
      case 1: return launch_product_cfg<FMT, OT, 128, 256, 2, 2, 2>(b, stream);
      case 2: return launch_product_cfg<FMT, OT, 128, 128, 2, 2, 2>(b, stream);
      default: return launch_product_cfg<FMT, OT, 64, 128, 2, 2, 4>(b, stream);
    }
  }
}
// y = the slices' parts, in their order
template <bool BF16>
__global__ void __launch_bounds__(256) fb_join_kernel(const float* __restrict__ part, void* __restrict__ y, int splits,
                                                      int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < splits; ++s) {
    const float* at = part + s * n + i;
    if (i + 4 <= n) {
      const fb_u32x4_at4 u = *(const fb_u32x4_at4*)at;
      v[0] += __uint_as_float(u.x);
      v[1] += __uint_as_float(u.y);
      v[2] += __uint_as_float(u.z);
      v[3] += __uint_as_float(u.w);
    } else {
      for (int j = 0; i + j < n; ++j) v[j] += at[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (i + j < n) {
      if constexpr (BF16) ((__bf16*)y)[i + j] = (__bf16)v[j];
      else ((float*)y)[i + j] = v[j];
    }
}

// Few tiles of a long K leave most CUs idle: K in slices, as many as CUs have a tile each,
// of 8 stages and more, and another launch that joins them (3 us): 65 x 2560 -> 1024 fp32 52
// to 20 us, 509 x 2560 -> 500 18 to 9.
struct Slices {
  int splits, per;  // 0: not worth it
  int64_t bytes;
};
Slices slices(int64_t R, int64_t N, int64_t nk) {
  const int64_t tiles = (R + 63) / 64 * ((N + 127) / 128);
  Slices q{};
  int64_t most = cu_count() / std::max<int64_t>(tiles, 1);
  most = std::min(most, nk / 8);
  if (most < 2) return q;
  const int64_t per = ((nk + most - 1) / most + 3) / 4 * 4;  // whole words of scales
  q.splits = (int)((nk + per - 1) / per);
  q.per = (int)per;
  // what is saved, a stage 0.37 us, is to be more than the join
  if (q.splits < 2 || (nk - per) * 37 < 400) return Slices{};
  q.bytes = q.splits * R * N * 4;
  return q;
}
int64_t slices_bytes(int64_t R, int64_t N, int64_t nk) { return slices(R, N, nk).bytes; }

// room: slices_bytes of workspace (256-byte aligned), or null where there are none
template <int FMT, int OT>
int launch_product(const FbArgs& p, void* room, hipStream_t stream) {
  if constexpr (OT == O_BF16 || OT == O_F32) {
    const Slices q = slices(p.R, p.N, p.ldx / 128);
    if (q.splits) {
      FbArgs a = p;
      a.splits = q.splits;
      a.per = q.per;
      a.y = room;
      constexpr int PART = FMT == F_CODES && OT == O_BF16 ? O_PART : O_F32;
      if (int rc = launch_product_cfg<FMT, PART, 64, 128, 2, 2, 4>(FbBatch<1>{{a}}, stream)) return rc;
      const int64_t n = p.R * p.N;
      hipLaunchKernelGGL((fb_join_kernel<OT == O_BF16>), dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, stream,
                         (const float*)room, p.y, q.splits, n);
      return check_launch("fb_join_kernel");
    }
  }
  return launch_products<FMT, OT>(FbBatch<1>{{p}}, stream);
}

FbArgs codes_args(const void* x, const uint8_t* xs, const uint8_t* w, const uint8_t* s, void* y, int64_t R, int64_t K,
                  int64_t N) {
  FbArgs p{};
  p.x = (const uint8_t*)x;
  p.xs = xs;
  p.w = w;
  p.s = s;
  p.y = y;
  p.R = R;
  p.N = N;
  p.ldx = fb_width(K);
  p.words = (int)fb_words(K);
  return p;
}

// ---------------------------------------------------------------------------
// few rows (up to FB_FEW)
// ---------------------------------------------------------------------------
// Launches, latency and the weight's bytes are all there is: every load of a wave leaves
// at once, straight to registers, and rows that are not codes yet are rounded on the way.
constexpr int FB_FEW = 64;
enum { X_F32 = 0, X_BF16 = 1, X_CODES = 2 };  // as the C types

// 64 values of one block of a row (32 of each of its two steps, from c0 and c0 + 64) ->
// their codes, the row's other 64 in lane + 32
template <int XT>
__device__ __forceinline__ void fb_round64(const void* x, int64_t row, int64_t K, int64_t c0, i32x8_t (&op)[2],
                                           uint32_t& byte) {
  float v[8][8];
  uint32_t top = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    fb_load8<XT == X_BF16>(x, row, K, c0 + q / 4 * 64 + q % 4 * 8, v[q]);
    top = max(top, fb_amax8(v[q]));
  }
  byte = fb_scale_byte(max(top, (uint32_t)__shfl_xor((int)top, 32, 64)));
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const uint2 c = fb_encode8(v[q], byte);
    op[q / 4][q % 4 * 2] = (int)c.x;
    op[q / 4][q % 4 * 2 + 1] = (int)c.y;
  }
}

// A workgroup has 32 rows of the weight (of the gated block 16 of gate's and 16 of up's),
// its 8 waves a slice of K each; the waves' sums meet in LDS and are added in the order of
// the waves.  A lane's codes of the weight lie in a row of their own; x's, which every
// workgroup reads, do too up to 32 rows, past them they come through LDS in whole lines,
// 16-byte chunks changing places by the row (us, direct and by LDS: 1 x 1024 -> 2560 4.1 and
// 5.2, 64 x 2560 -> 1024 10.3 and 8.7).  RT: tiles of 32 rows of x.  Hidden values leave in fp32 (O_GATED): a block of their
// codes would take 256 rows of weights a workgroup, whose bytes one CU waits for longer than
// another launch takes (1 token, 1024 by 2560: 11 us for 4.5 and 2).
// Codes are decoded and multiplied as bf16 (exact) but for bf16 results of 33 to 64 rows, where the
// 8-bit instruction gains what it loses bits for: 64 x 8192 -> 8192 23.1 us for 25.3, 64 x 1024 -> 2560
// 7.4 for 7.7; of fewer rows it gains nothing (16 x 2560 -> 1024 6.3 both, 1 x 4096 -> 4096 8.6 for 8.3)
// to 4 % (1 x 8192 -> 28672 48.4 for 49.4, one row of bf16, 1024 -> 2560, 7.7 for 8.0).
template <int XT, int OT, int RT>
__global__ void __launch_bounds__(512) fb_stream_kernel(FbArgs p, int64_t K) {
  constexpr int NW = 8, U = 2;  // blocks read at once
  constexpr bool GATED = OT == O_GATED, XL = XT == X_CODES && RT > 1;
  constexpr int OWN = XL ? U * RT * 32 * FB_BLOCK : RT * 4096;  // a wave's x, and its sums
  __shared__ __attribute__((aligned(1024))) char smem[NW * OWN];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * (GATED ? 16 : 32), nb = p.ldx / FB_BLOCK, ns = (int64_t)p.words * 4;
  const int tr = fb_perm(l32);  // row of the tile: the first 16 are lane group 0's sums
  const int64_t wrow = min<int64_t>(n0 + (GATED ? tr & 15 : tr), p.N - 1);
  const uint8_t* w = (GATED && tr >= 16 ? p.w2 : p.w) + wrow * p.ldx + g * 32;
  const uint8_t* ws = (GATED && tr >= 16 ? p.s2 : p.s) + wrow * ns;
  const int rows = (int)p.R, per = (int)((nb + NW - 1) / NW);
  const int lo = (int)min<int64_t>((int64_t)wave * per, nb), hi = (int)min<int64_t>(lo + per, nb);
  f32x16_t acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] = 0.0f;
  char* own = smem + wave * OWN;
  for (int b0 = lo; b0 < hi; b0 += U) {
    i32x8_t wf[U][2], xf[U][RT][2];
    uint32_t sw[U], sx[U][RT];
    if constexpr (XL) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last pieces are read
#pragma unroll
      for (int a = 0; a < U * RT * 4; ++a) {  // 8 rows of a block
        const int u = a / (RT * 4), r0 = a % (RT * 4) * 8, r = r0 + lane / 8;
        if (r0 >= rows) continue;  // uniform; rows that nobody needs hold anything
        dma16(p.x + (int64_t)min(b0 + u, hi - 1) * FB_BLOCK,
              (uint32_t)(min(r, rows - 1) * (int)p.ldx + (lane % 8 ^ (r & 7)) * 16), lds_offset(own + a * 1024));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = min(b0 + u, hi - 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4* at = (const uint4*)(w + (int64_t)b * FB_BLOCK + h * 64);
        wf[u][h] = fb_operand(at[0], at[1]);
      }
      sw[u] = ws[b];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int64_t row = min(t * 32 + l32, rows - 1);
        if constexpr (XT == X_CODES) {
          sx[u][t] = p.xs[row * ns + b];
#pragma unroll
          for (int h = 0; h < 2 && !XL; ++h) {
            const uint4* at = (const uint4*)(p.x + row * p.ldx + (int64_t)b * FB_BLOCK + h * 64 + g * 32);
            xf[u][t][h] = fb_operand(at[0], at[1]);
          }
        } else fb_round64<XT>(p.x, row, K, (int64_t)b * FB_BLOCK + g * 32, xf[u][t], sx[u][t]);
      }
    }
    if constexpr (XL) {
      wait_vm<0>();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const char* at = own + ((u * RT + t) * 32 + l32) * FB_BLOCK;
            const int c = h * 4 + g * 2;
            xf[u][t][h] = fb_operand(*(const uint4*)(at + (c ^ (l32 & 7)) * 16), *(const uint4*)(at + (c + 1 ^ (l32 & 7)) * 16));
          }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b0 + u >= hi) break;  // uniform
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if constexpr (OT == O_F32 || GATED || RT == 1) {  // exact
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  fb_decode8(wf[u][h][2 * q], wf[u][h][2 * q + 1], fb_scale(sw[u])),
                  fb_decode8(xf[u][t][h][2 * q], xf[u][t][h][2 * q + 1], fb_scale(sx[u][t])), acc[t], 0, 0, 0);
          } else {
            acc[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[u][h], xf[u][t][h], acc[t], 0, 0, 0, (int)sw[u],
                                                                    0, (int)sx[u][t]);
          }
        }
    }
  }
  __syncthreads();
  float4* red = (float4*)smem;
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      red[((wave * RT + t) * 4 + i) * 64 + lane] =
          make_float4(acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]);
  __syncthreads();
  auto sum = [&](int t, int i, int l, float (&f)[4]) {  // of the waves: four columns of a row
    float4 v = red[(t * 4 + i) * 64 + l];
#pragma unroll
    for (int q = 1; q < NW; ++q) {
      const float4 a = red[((q * RT + t) * 4 + i) * 64 + l];
      v.x += a.x;
      v.y += a.y;
      v.z += a.z;
      v.w += a.w;
    }
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  };
  if constexpr (GATED) {
    if (tid >= RT * 128) return;
    const int l = tid & 31, i = tid >> 5 & 3, t = tid >> 7;
    float f[4], v[4], a[4], b[4];
    sum(t, i, l, f);
    sum(t, i, l + 32, v);
    const int64_t row = t * 32 + l, n = n0 + i * 4;
    if (row >= rows) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[q] = fb_gated(f[q], v[q], a[q], b[q]);
      if (n + q < p.N) ((float*)p.y)[row * p.N + n + q] = v[q];
    }
    if (p.kept) {
      uint8_t* to = p.kept + fb_kept_at(row, n0, p.N);
      uint2 hi2;
      uint32_t lo2;
      fb_pack24(a, hi2, lo2);
      *(uint2*)(to + i / 2 * 1024 + i % 2 * 8) = hi2;
      *(uint32_t*)(to + 4096 + i * 4) = lo2;
      fb_pack24(b, hi2, lo2);
      *(uint2*)(to + 2048 + i / 2 * 1024 + i % 2 * 8) = hi2;
      *(uint32_t*)(to + 5120 + i * 4) = lo2;
    }
  } else {
    for (int e = tid; e < RT * 256; e += 512) {
      const int l = e & 63, i = e >> 6 & 3, t = e >> 8;
      float f[4];
      sum(t, i, l, f);
      const int64_t row = t * 32 + (l & 31), n = n0 + (l >> 5) * 16 + i * 4;
      if (row < rows) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < p.N) {
            if constexpr (OT == O_BF16) ((__bf16*)p.y)[row * p.N + n + q] = (__bf16)f[q];
            else ((float*)p.y)[row * p.N + n + q] = f[q];
          }
      }
    }
  }
}

// v = a + b + c, each the next 8 significant bits: exact in bf16 (their upper halves), and all
// 24 of fp32.  An infinity or NaN is a alone.
__device__ __forceinline__ void fb_thirds(float v, uint32_t (&t)[3]) {
  const float x = __builtin_canonicalizef(v);
  t[0] = __float_as_uint(x) & 0xffff0000u;
  const float rest = x - __uint_as_float(t[0]), y = rest == rest ? rest : 0.0f;
  t[1] = __float_as_uint(y) & 0xffff0000u;
  t[2] = __float_as_uint(y - __uint_as_float(t[1]));
}
__device__ __forceinline__ void fb_split3(const float (&v)[8], bf16x8_t (&t)[3]) {
  uint32_t w[3][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t a[3], b[3];
    fb_thirds(v[2 * q], a);
    fb_thirds(v[2 * q + 1], b);
#pragma unroll
    for (int k = 0; k < 3; ++k) w[k][q] = __builtin_amdgcn_perm(b[k], a[k], 0x07060302u);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) t[k] = __builtin_bit_cast(bf16x8_t, make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]));
}

// The input gradient of few rows, in one launch: a workgroup has 32 CT columns of up to 64 rows,
// its 8 waves a slice of the weight's rows each.  A lane reads 32 codes of one row, and the
// wave turns 64 such rows round through LDS of its own, decoded to bf16.  The groups of rows
// and the four workgroups that share a line of codes are neighbours in one XCD's band.  (1 row
// 2560 -> 1024: 9 us, 21 by way of the turned weight.)
template <bool BF16, int RT, int CT>
__global__ void __launch_bounds__(512)
fb_dx_stream_kernel(const void* __restrict__ grad, const uint8_t* __restrict__ w, const uint8_t* __restrict__ s,
                    void* __restrict__ dx, int64_t rows, int64_t I, int64_t O) {
  constexpr int NW = 8, LD = 72, OWN = RT * 4096 > 32 * LD * 2 ? CT * RT * 4096 : CT * 32 * LD * 2, NT = BF16 ? 1 : 3;
  __shared__ __attribute__((aligned(16))) char smem[NW * OWN];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t b0 = blockIdx.x;
  {
    const int64_t full = (int64_t)gridDim.x / 8 * 8;
    if (b0 < full) b0 = b0 % 8 * (full / 8) + b0 / 8;
  }
  const int64_t groups = (rows + RT * 32 - 1) / (RT * 32), row0 = b0 % groups * (RT * 32);
  const int64_t k0 = b0 / groups * (CT * 32), nb = fb_blocks(I), ns = (nb + 3) / 4 * 4;
  const int R = (int)min<int64_t>(rows - row0, RT * 32);
  const int64_t steps = (O + 63) / 64, per = (steps + NW - 1) / NW;
  const int64_t lo = min((int64_t)wave * per, steps), hi = min(lo + per, steps);
  uint16_t* own = (uint16_t*)(smem + wave * OWN);
  f32x16_t acc[CT][RT];
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[c][t][r] = 0.0f;
  uint4 c0[CT], c1[CT];
  float sc;
  auto codes = [&](int64_t step) {  // rows past the last: zeros
    const int64_t o = step * 64 + lane;
#pragma unroll
    for (int c = 0; c < CT; ++c) c0[c] = c1[c] = make_uint4(0, 0, 0, 0);
    sc = 1.0f;
    if (o < O) {
      const uint4* at = (const uint4*)(w + o * nb * FB_BLOCK + k0);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        c0[c] = at[2 * c];
        c1[c] = at[2 * c + 1];
      }
      sc = fb_scale(s[o * ns + k0 / FB_BLOCK]);
    }
  };
  if (lo < hi) codes(lo);
  for (int64_t step = lo; step < hi; ++step) {
    float v[RT][4][8];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) fb_load8<BF16>(grad, row0 + min(t * 32 + l32, R - 1), O, step * 64 + q * 16 + g * 8, v[t][q]);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const uint32_t w8[8] = {c0[c].x, c0[c].y, c0[c].z, c0[c].w, c1[c].x, c1[c].y, c1[c].z, c1[c].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float f[4];
        fb_decode4(w8[j], sc, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) own[(c * 32 + 4 * j + e) * LD + lane] = (uint16_t)(__float_as_uint(f[e]) >> 16);
      }
    }
    if (step + 1 < hi) codes(step + 1);
    __builtin_amdgcn_wave_barrier();  // a wave's LDS accesses are done in order
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      bf16x8_t a[CT];
#pragma unroll
      for (int c = 0; c < CT; ++c) a[c] = *(const bf16x8_t*)&own[(c * 32 + fb_perm(l32)) * LD + q * 16 + g * 8];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        bf16x8_t x[3];
        if constexpr (BF16) {
          const float* f = v[t][q];
          x[0] = __builtin_bit_cast(bf16x8_t, make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]),
                                                         pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])));
        } else {
          fb_split3(v[t][q], x);
        }
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int c = 0; c < CT; ++c) acc[c][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[c], x[k], acc[c][t], 0, 0, 0);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  float4* red = (float4*)smem;
#pragma unroll
  for (int t = 0; t < CT * RT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x16_t& v = acc[t / RT][t % RT];
      red[((wave * CT * RT + t) * 4 + i) * 64 + lane] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
  __syncthreads();
  for (int e = tid; e < CT * RT * 256; e += 512) {
    const int l = e & 63, i = e >> 6 & 3, ct = e >> 8, t = ct % RT;
    float4 a = red[(ct * 4 + i) * 64 + l];
#pragma unroll
    for (int q = 1; q < NW; ++q) {
      const float4 b = red[((q * CT * RT + ct) * 4 + i) * 64 + l];
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    const int row = t * 32 + (l & 31);
    const int64_t n = k0 + ct / RT * 32 + (l >> 5) * 16 + i * 4;
    const float f[4] = {a.x, a.y, a.z, a.w};
    if (row < R) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (n + q < I) {
          if constexpr (BF16) ((__bf16*)dx)[(row0 + row) * I + n + q] = (__bf16)f[q];
          else ((float*)dx)[(row0 + row) * I + n + q] = f[q];
        }
    }
  }
}

template <int XT, int OT>
int launch_stream_of(const FbArgs& p, int64_t K, hipStream_t stream) {
  const int64_t blocks = OT == O_GATED ? (p.N + 15) / 16 : (p.N + 31) / 32;
  if (!grid_fits(blocks, 512)) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block product: too many columns");
  if (FB_FEW * p.ldx >= 1LL << 31) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block product: rows too wide");
  auto* kernel = p.R <= 32 ? &fb_stream_kernel<XT, OT, 1> : &fb_stream_kernel<XT, OT, 2>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(512), 0, stream, p, K);
  return check_launch("fb_stream_kernel");
}
// Whether fb_stream_kernel rounds rows itself: as long as a wave has one block of few of
// them, whose rounding is then less than a launch (1 x 1024 -> 2560: 7.8 us on the device for
// 4.1 and 2, but 9.7 for 12 as a call by itself; 16 x 2560 -> 1024: 11.8 for 6.3 and 2).
bool rounds_itself(int64_t rows, int64_t K) { return rows <= 16 && fb_blocks(K) <= 8; }

template <int OT>
int launch_stream(const FbArgs& p, int x_dtype, int64_t K, hipStream_t stream) {
  if (x_dtype == SMAUL_DTYPE_FP8_BLOCK) return launch_stream_of<X_CODES, OT>(p, K, stream);
  if (x_dtype == SMAUL_DTYPE_BF16) return launch_stream_of<X_BF16, OT>(p, K, stream);
  if constexpr (OT != O_GATED) return launch_stream_of<X_F32, OT>(p, K, stream);
  return fail(SMAUL_ERR_INVALID, "fp8_block_ffn: bad dtype");
}

// ---------------------------------------------------------------------------
// operands of the gradients' products: bf16 rows of whole stages (64 values)
// ---------------------------------------------------------------------------
// Several matrices a launch, each R rows of C values: bf16 rows, fp32 rows or codes
// (decoded: exact in bf16), turned round (dst [C][ld]) or as they lie (dst [R][ld]), zeros
// up to whole stages.  fp32 rows are three bf16 planes, each the next 8 bits (exact), 64
// values of each in turn; the other side's rows are then there three times.
enum { S_BF16 = 0, S_F32 = 1, S_CODES = 2 };
struct FbTurn {
  const void* src;
  const uint8_t* scales;
  uint16_t* dst;
  int64_t R, C, lds, ld;  // lds: the source's row, in values
  int64_t blocks;
  int fmt, turned, copies;
};
constexpr int FB_TURNS = 6;
struct FbTurns {
  FbTurn t[FB_TURNS];
};
__host__ __device__ __forceinline__ int64_t fb_stages(int64_t K) { return (K + 63) / 64; }

// a workgroup: 64 by 64 values, 16 of a row a thread, through LDS where they are turned.
// Memory bounds it: the gradients' of 8192 tokens, 1024 by 2560, 51 us, 290 MB
template <int FMT, bool TURNED>
__device__ __forceinline__ void fb_turn(const FbTurn& t, int64_t b, uint16_t* sh) {
  constexpr int LD = 72, PLANES = FMT == S_F32 ? 3 : 1;  // 16-byte rows off the banks' period
  const uint32_t across = (uint32_t)fb_stages(t.C), rb = (uint32_t)b / across;  // both from one 32-bit grid
  const int64_t r0 = (int64_t)rb * 64, c0 = (b - (int64_t)rb * across) * 64;
  const int tid = threadIdx.x, lr = tid >> 2, lc = (tid & 3) * 16;
  const int64_t r = r0 + lr, c = c0 + lc;
  float v[16];
#pragma unroll
  for (int q = 0; q < 16; ++q) v[q] = 0.0f;
  if (r < t.R && c < t.C) {
    if constexpr (FMT == S_CODES) {  // rows end with zero codes
      const uint4 w = *(const uint4*)((const uint8_t*)t.src + r * t.lds + c);
      const float s = fb_scale(t.scales[r * ((t.lds / FB_BLOCK + 3) / 4 * 4) + c / FB_BLOCK]);
      fb_decode4(w.x, s, v);
      fb_decode4(w.y, s, v + 4);
      fb_decode4(w.z, s, v + 8);
      fb_decode4(w.w, s, v + 12);
    } else {
      float lo[8], hi[8];
      fb_load8<FMT == S_BF16>(t.src, r, t.C, c, lo);
      fb_load8<FMT == S_BF16>(t.src, r, t.C, c + 8, hi);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        v[q] = lo[q];
        v[q + 8] = hi[q];
      }
    }
  }
  uint32_t w[PLANES][8];
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    uint32_t x[3] = {__float_as_uint(v[2 * q])}, y[3] = {__float_as_uint(v[2 * q + 1])};  // exact in bf16
    if constexpr (FMT == S_F32) {
      fb_thirds(v[2 * q], x);
      fb_thirds(v[2 * q + 1], y);
    }
#pragma unroll
    for (int p = 0; p < PLANES; ++p) w[p][q] = __builtin_amdgcn_perm(y[p], x[p], 0x07060302u);
  }
#pragma unroll
  for (int p = 0; p < PLANES; ++p) {
    if constexpr (TURNED) {
#pragma unroll
      for (int q = 0; q < 16; ++q) sh[(lc + q) * LD + lr] = (uint16_t)(w[p][q / 2] >> (16 * (q & 1)));
    } else if (r < t.R) {
      uint4* o = (uint4*)(t.dst + r * t.ld + c0 * PLANES + p * 64 + lc);
      o[0] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
      o[1] = make_uint4(w[p][4], w[p][5], w[p][6], w[p][7]);
    }
  }
  if constexpr (TURNED) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int at = tid + q * 256, i = at >> 3, j = (at & 7) * 8;
      if (c0 + i < t.C) {
        const uint4 d = *(const uint4*)&sh[i * LD + j];
        uint16_t* o = t.dst + (c0 + i) * t.ld + r0 * t.copies + j;
        for (int e = 0; e < t.copies; ++e) *(uint4*)(o + e * 64) = d;
      }
    }
  }
}

__global__ void __launch_bounds__(256) fb_turn_kernel(FbTurns a) {
  __shared__ __attribute__((aligned(16))) uint16_t sh[64 * 72];
  int64_t b = blockIdx.x;
  int k = 0;
#pragma unroll
  for (int j = 0; j + 1 < FB_TURNS; ++j)
    if (k == j && b >= a.t[j].blocks) {
      b -= a.t[j].blocks;
      k = j + 1;
    }
  const FbTurn& t = a.t[k];
  if (t.fmt == S_CODES) fb_turn<S_CODES, true>(t, b, sh);
  else if (t.fmt == S_F32) fb_turn<S_F32, false>(t, b, sh);
  else if (t.turned) fb_turn<S_BF16, true>(t, b, sh);
  else fb_turn<S_BF16, false>(t, b, sh);
}

__global__ void __launch_bounds__(256) fb_clear_kernel(uint16_t* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

int launch_turns(FbTurns& a, int n, hipStream_t stream) {
  int64_t blocks = 0;
  for (int i = 0; i < n; ++i) {
    a.t[i].blocks = fb_stages(a.t[i].R) * fb_stages(a.t[i].C);
    blocks += a.t[i].blocks;
  }
  if (!grid_fits(blocks, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block gradient: too many values");
  if (n == 0 || blocks == 0) return SMAUL_OK;
  hipLaunchKernelGGL(fb_turn_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return check_launch("fb_turn_kernel");
}

FbTurn turn_codes(const void* codes, const uint8_t* scales, int64_t R, int64_t C, uint16_t* dst, int64_t ld,
                  int copies = 1) {
  return FbTurn{codes, scales, dst, R, C, fb_width(C), ld, 0, S_CODES, 1, copies};
}
FbTurn turn_rows(const void* rows, int fmt, int64_t R, int64_t C, uint16_t* dst, int64_t ld, int turned) {
  return FbTurn{rows, nullptr, dst, R, C, C, ld, 0, fmt, turned, 1};
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

struct LinearParts {
  int64_t xc, xs, room, total;
};
LinearParts linear_parts(int64_t rows, int64_t in_f, int64_t out_f, int x_dtype) {
  LinearParts q{};
  Parts w;
  const bool round = x_dtype != SMAUL_DTYPE_FP8_BLOCK && !rounds_itself(rows, in_f);
  q.xc = w.take(round ? rows * fb_width(in_f) : 0);
  q.xs = w.take(round ? rows * fb_words(in_f) * 4 : 0);
  q.room = w.take(rows > FB_FEW ? slices_bytes(rows, out_f, fb_blocks(in_f)) : 0);
  q.total = w.at;
  return q;
}

struct FfnParts {
  int64_t xc, xs, hc, hs, hf, room, total;
};
// what the caller keeps for the gradients stands in `saved` (save), the rest in the workspace
FfnParts ffn_parts(int64_t T, int64_t d, int64_t h, int x_dtype, bool save) {
  FfnParts q{};
  Parts w;
  const bool rows = x_dtype != SMAUL_DTYPE_FP8_BLOCK && !save && !rounds_itself(T, d);
  q.xc = w.take(rows ? T * fb_width(d) : 0);
  q.xs = w.take(rows ? T * fb_words(d) * 4 : 0);
  q.hc = w.take(save ? 0 : T * fb_width(h));
  q.hs = w.take(save ? 0 : T * fb_words(h) * 4);
  q.hf = w.take(T <= FB_FEW ? T * h * 4 : 0);
  q.room = w.take(T > FB_FEW ? slices_bytes(T, d, fb_blocks(h)) : 0);
  q.total = w.at;
  return q;
}

struct FfnBackParts {
  int64_t dy, wd, wgu, dgu, dgut, xt, dyt, ht, room, total;
  int64_t lt, ld, lh;  // T, d and h to whole stages
};
FfnBackParts ffn_back_parts(int64_t T, int64_t d, int64_t h, bool dx, bool dw) {
  FfnBackParts q{};
  Parts w;
  q.lt = fb_stages(T) * 64;
  q.ld = fb_stages(d) * 64;
  q.lh = fb_stages(h) * 64;
  q.dy = w.take(d % 64 ? T * q.ld * 2 : 0);
  q.wd = w.take(h * q.ld * 2);
  q.wgu = w.take(dx ? d * q.lh * 4 : 0);
  q.dgu = w.take(T * q.lh * 4);
  q.dgut = w.take(dw ? q.lh * q.lt * 4 : 0);
  q.xt = w.take(dw ? d * q.lt * 2 : 0);
  q.dyt = w.take(dw ? d * q.lt * 2 : 0);
  q.ht = w.take(dw ? h * q.lt * 2 : 0);
  q.room = w.take(dx ? slices_bytes(T, d, q.lh / 32) : 0);
  q.total = w.at;
  return q;
}

// Whether fb_dx_stream_kernel has the call: of few rows, and of as many as one round of the
// CUs takes in two steps a wave.  There the two launches (or three, in slices) wait for one
// another longer than the weight's being turned by each group of rows takes (us, by way of
// the turned weight and so: 512 x 777 -> 1000 fp32 22.5 and 13.5, 2048 x 256 -> 256 13.1 and
// 8.8, 128 x 1024 -> 2560 bf16 13.4 and 9.5; past it 500 x 1024 -> 2560 bf16 14 and 25, in two rounds
// 3816 x 383 -> 159 bf16 11.3 and 19.7, 1078 x 205 -> 1019 fp32 15.3 and 22.8).  fp32 rows, whose
// thirds take longer than the weight, have 64 columns a workgroup where 32 take two rounds
// (2934 x 318 -> 293 17.4 by way of the turned weight, so 13.1, of 32 columns 17.4; 653 x 470 -> 1135
// 21.4, 14.0 and 18.2; at the edge, 256 workgroups, 1001 x 777 -> 1000 26.3, 18.6 and 24.2; past it
// 2804 x 315 -> 379 18.1 and 21.1; of as few outputs as 64, 205 x 64 -> 2738, 9.3 and 10.3), but 32
// where these are one round (512 rows 13.5 for 15.7).
int64_t dx_groups(int64_t rows, int64_t in_f, int columns) { return (in_f + columns - 1) / columns * ((rows + 63) / 64); }
bool dx_fits(int64_t rows, int64_t in_f, int64_t out_f, int columns) {
  return dx_groups(rows, in_f, columns) <= cu_count() && ((out_f + 63) / 64 + 7) / 8 <= 2;
}
bool dx_wide(int64_t rows, int64_t in_f, int64_t out_f, bool f32) {
  return f32 && rows > FB_FEW && !dx_fits(rows, in_f, out_f, 32) && dx_fits(rows, in_f, out_f, 64);
}
bool dx_streams(int64_t rows, int64_t in_f, int64_t out_f, bool f32) {
  return rows <= FB_FEW || dx_fits(rows, in_f, out_f, 32) || dx_wide(rows, in_f, out_f, f32);
}

struct DxParts {
  int64_t g, wt, room, total, ld;
  int copies;
};
DxParts dx_parts(int64_t rows, int64_t in_f, int64_t out_f, int dtype) {
  DxParts q{};
  Parts w;
  const bool f32 = dtype == SMAUL_DTYPE_F32;
  if (dx_streams(rows, in_f, out_f, f32)) return q;
  q.copies = f32 ? 3 : 1;
  q.ld = fb_stages(out_f) * 64 * q.copies;
  q.g = w.take(f32 || out_f % 64 ? rows * q.ld * 2 : 0);
  q.wt = w.take(in_f * q.ld * 2);
  q.room = w.take(slices_bytes(rows, in_f, q.ld / 64));
  q.total = w.at;
  return q;
}

// x [R][ld] . w [N][ld]^T, bf16 rows of whole stages
FbArgs rows_args(const void* x, const void* w, void* y, int64_t R, int64_t ld, int64_t N) {
  FbArgs p{};
  p.x = (const uint8_t*)x;
  p.w = (const uint8_t*)w;
  p.y = y;
  p.R = R;
  p.N = N;
  p.ldx = ld * 2;
  return p;
}

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
  return linear_parts(rows, in_f, out_f, x_dtype).total;
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
  const LinearParts q = linear_parts(rows, in_f, out_f, x_dtype);
  const int64_t need = q.total;
  if (workspace_bytes < need || (need > 0 && (!workspace || !fb_aligned(workspace, 256))))
    return fail(SMAUL_ERR_INVALID, "fp8_block_linear: workspace %lld < %lld bytes, or unaligned",
                (long long)workspace_bytes, (long long)need);
  if (!given && !rounds_itself(rows, in_f)) {
    uint8_t* c = (uint8_t*)workspace + q.xc;
    uint8_t* cs = (uint8_t*)workspace + q.xs;
    if (int rc = launch_quantize(x, x_dtype, c, cs, rows, in_f, stream)) return rc;
    x = c;
    xs = cs;
    x_dtype = SMAUL_DTYPE_FP8_BLOCK;
  }
  const FbArgs p = codes_args(x, xs, w, s, y, rows, in_f, out_f);
  if (rows <= FB_FEW)
    return y_dtype == SMAUL_DTYPE_BF16 ? launch_stream<O_BF16>(p, x_dtype, in_f, stream)
                                       : launch_stream<O_F32>(p, x_dtype, in_f, stream);
  void* room = (char*)workspace + q.room;
  return y_dtype == SMAUL_DTYPE_BF16 ? launch_product<F_CODES, O_BF16>(p, room, stream)
                                     : launch_product<F_CODES, O_F32>(p, room, stream);
}

int64_t smaul_fp8_block_backward_input_workspace_size(int64_t rows, int64_t in_f, int64_t out_f, int dtype) {
  if (rows < 0 || in_f <= 0 || out_f <= 0 || !fb_dtype_ok(dtype)) return -1;
  return dx_parts(rows, in_f, out_f, dtype).total;
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
  const DxParts q = dx_parts(rows, in_f, out_f, dtype);
  char* ws = (char*)workspace;
  const bool bf16 = dtype == SMAUL_DTYPE_BF16;
  if (dx_streams(rows, in_f, out_f, !bf16)) {
    const bool wide = dx_wide(rows, in_f, out_f, !bf16);
    const int64_t blocks = dx_groups(rows, in_f, wide ? 64 : 32);
    if (!grid_fits(blocks, 512)) return fail(SMAUL_ERR_UNSUPPORTED, "fp8_block_backward_input: too wide a weight");
    auto* kernel = wide   ? &fb_dx_stream_kernel<false, 2, 2>
                   : bf16 ? (rows <= 32 ? &fb_dx_stream_kernel<true, 1, 1> : &fb_dx_stream_kernel<true, 2, 1>)
                          : (rows <= 32 ? &fb_dx_stream_kernel<false, 1, 1> : &fb_dx_stream_kernel<false, 2, 1>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(512), 0, stream, g, w, s, dx, rows, in_f, out_f);
    return check_launch("fb_dx_stream_kernel");
  }
  uint16_t* wt = (uint16_t*)(ws + q.wt);
  FbTurns a{};
  int n = 0;
  a.t[n++] = turn_codes(w, s, out_f, in_f, wt, q.ld, q.copies);
  if (!bf16 || out_f % 64) {
    a.t[n++] = turn_rows(g, bf16 ? S_BF16 : S_F32, rows, out_f, (uint16_t*)(ws + q.g), q.ld, 0);
    g = ws + q.g;
  }
  if (int rc = launch_turns(a, n, stream)) return rc;
  const FbArgs p = rows_args(g, wt, dx, rows, q.ld, in_f);
  void* room = ws + q.room;
  return bf16 ? launch_product<F_BF16, O_BF16>(p, room, stream) : launch_product<F_BF16, O_F32>(p, room, stream);
}

int64_t smaul_fp8_block_ffn_saved_size(int64_t T, int64_t h) {
  if (T < 0 || h <= 0) return -1;
  return fb_kept_size(T, h);
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
  const bool few = T <= FB_FEW;
  int xt = x_dtype;
  if (!given && (save || !rounds_itself(T, d))) {
    xt = SMAUL_DTYPE_FP8_BLOCK;
    uint8_t* xc = save ? x_codes : ws + q.xc;
    uint8_t* xcs = save ? x_scales : ws + q.xs;
    if (int rc = launch_quantize(x, x_dtype, xc, xcs, T, d, stream)) return rc;
    x = xc;
    xs = xcs;
  }
  uint8_t* hc = save ? h_codes : ws + q.hc;
  uint8_t* hs = save ? h_scales : ws + q.hs;
  FbArgs p = codes_args(x, xs, gate_w, gate_s, hc, T, d, h);
  p.w2 = up_w;
  p.s2 = up_s;
  p.ys = hs;
  p.kept = (uint8_t*)saved;
  const FbArgs down = codes_args(hc, hs, down_w, down_s, y, T, h, d);
  if (!few) {
    // Exact products while a CU has no more than one of their tiles: there the error of one
    // block is a part of the output's that can be seen (92 x 196 -> 2107, against 64 bits:
    // 0.0030 for 0.0016, 0.0016 of them the output's own rounding), and the time is
    // mostly not the matrix instructions' (us: 65 x 1024 -> 2560 23.9 for 20.5, 512 26.2 for
    // 22.6, 256 x 4096 -> 8192 63 for 48).  Of more tiles the output has 0.0023, and they
    // would take half as long again (16384 x 2048 -> 5120: 689 for 445).
    const bool exact = (T + 63) / 64 * fb_blocks(h) <= cu_count();
    if (int rc = exact ? launch_product<F_CODES, O_GATED_EXACT>(p, nullptr, stream)
                       : launch_product<F_CODES, O_GATED>(p, nullptr, stream))
      return rc;
    return launch_product<F_CODES, O_BF16>(down, ws + q.room, stream);
  }
  p.y = ws + q.hf;
  if (int rc = launch_stream<O_GATED>(p, xt, d, stream)) return rc;
  if (int rc = launch_quantize(ws + q.hf, SMAUL_DTYPE_F32, hc, hs, T, h, stream)) return rc;
  return launch_stream<O_BF16>(down, SMAUL_DTYPE_FP8_BLOCK, h, stream);
}

int64_t smaul_fp8_block_ffn_backward_workspace_size(int64_t T, int64_t d, int64_t h) {
  if (T < 0 || d <= 0 || h <= 0) return -1;
  return ffn_back_parts(T, d, h, true, true).total;
}

int64_t smaul_fp8_block_ffn_backward_part_workspace_size(int64_t T, int64_t d, int64_t h, int dx, int dw) {
  if (T < 0 || d <= 0 || h <= 0) return -1;
  return ffn_back_parts(T, d, h, dx != 0, dw != 0).total;
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
  const FfnBackParts q = ffn_back_parts(T, d, h, dx != nullptr, weights);
  if (workspace_bytes < q.total || (q.total > 0 && (!workspace || !fb_aligned(workspace, 256))))
    return fail(SMAUL_ERR_INVALID, "fp8_block_ffn_backward: workspace %lld < %lld bytes, or unaligned",
                (long long)workspace_bytes, (long long)q.total);
  char* ws = (char*)workspace;
  if (T == 0) {
    const int64_t n = d * h * 2;  // bytes, cleared by a kernel: a captured call may not record a fill of memory
    for (void* p : {dgate, dup, ddown}) {
      hipLaunchKernelGGL(fb_clear_kernel, dim3((unsigned)std::min<int64_t>((n / 2 + 255) / 256, 4096)), dim3(256), 0,
                         stream, (uint16_t*)p, n / 2);
      if (int rc = check_launch("fb_clear_kernel")) return rc;
    }
    return SMAUL_OK;
  }
  uint16_t *wd = (uint16_t*)(ws + q.wd), *wgu = (uint16_t*)(ws + q.wgu), *dgu = (uint16_t*)(ws + q.dgu);
  uint16_t *dgut = (uint16_t*)(ws + q.dgut), *xt = (uint16_t*)(ws + q.xt), *dyt = (uint16_t*)(ws + q.dyt);
  uint16_t* ht = (uint16_t*)(ws + q.ht);
  FbTurns a{};
  int n = 0;
  const void* rows = dy;
  a.t[n++] = turn_codes(down_w, down_s, d, h, wd, q.ld);
  if (d % 64) {
    a.t[n++] = turn_rows(dy, S_BF16, T, d, (uint16_t*)(ws + q.dy), q.ld, 0);
    rows = ws + q.dy;
  }
  if (dx) {
    a.t[n++] = turn_codes(gate_w, gate_s, h, d, wgu, 2 * q.lh);
    a.t[n++] = turn_codes(up_w, up_s, h, d, wgu + q.lh, 2 * q.lh);
  }
  if (int rc = launch_turns(a, n, stream)) return rc;
  FbArgs p = rows_args(rows, wd, dgu, T, q.ld, h);
  p.kept = (uint8_t*)saved;
  p.ldh = q.lh;
  if (int rc = launch_product<F_BF16, O_DGATED>(p, nullptr, stream)) return rc;
  if (dx)
    if (int rc = launch_product<F_BF16, O_BF16>(rows_args(dgu, wgu, dx, T, 2 * q.lh, d), ws + q.room, stream)) return rc;
  if (!weights) return SMAUL_OK;
  FbTurns b{};
  b.t[0] = turn_rows(dgu, S_BF16, T, 2 * q.lh, dgut, q.lt, 1);
  b.t[1] = turn_codes(x_codes, x_scales, T, d, xt, q.lt);
  b.t[2] = turn_rows(dy, S_BF16, T, d, dyt, q.lt, 1);
  b.t[3] = turn_codes(h_codes, h_scales, T, h, ht, q.lt);
  if (int rc = launch_turns(b, 4, stream)) return rc;
  const FbBatch<3> grads{{rows_args(dgut, xt, dgate, h, q.lt, d),
                          rows_args(dgut + q.lh * q.lt, xt, dup, h, q.lt, d), rows_args(dyt, ht, ddown, d, q.lt, h)}};
  return launch_products<F_BF16, O_BF16>(grads, stream);
}

}  // extern "C"
