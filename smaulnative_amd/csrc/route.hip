// route.hip -- routing to experts on MI355X (gfx950), from the router's logits.
//
//   s = softmax(z) or sigmoid(z) over the E experts of a token
//   c = s + bias                       what the choice goes by (s alone without one)
//   a group's score is the sum of its group_best (1 or 2) highest c; the
//   top_groups groups with the highest are in; of their experts the k with the
//   highest c, descending, ties (of groups too) to the lowest index
//   w = s of the chosen (without the bias), over their sum (renorm; 1 / n where
//   the sum is below 1e-6), times scale
//
// An expert whose c is -inf or NaN is never chosen, nor one whose logit is -inf;
// a slot that no expert fills is -1 with weight 0 (the dispatch drops it).
// Without a bias the order is that of the logits, which no rounding of a score
// can change.
#include "smaul_common.h"

using smaul::check_launch;
using smaul::fail;

namespace {

constexpr int ROUTE_MAX_E = 512, ROUTE_MAX_K = 16, ROUTE_MAX_G = 64;
constexpr float ROUTE_MIN_SUM = 1e-6f;  // as the softmax router's guard

__device__ __forceinline__ float route_load(const void* z, int64_t i, int bf16) {
  return bf16 ? __uint_as_float((uint32_t)((const uint16_t*)z)[i] << 16) : ((const float*)z)[i];
}

struct RouteArgs {
  const void* z;
  const float* bias;
  float* prob;  // null: not wanted
  int64_t* topi;
  float* topw;
  int64_t T;
  int E, k, bf16, sigmoid, groups, top_groups, group_best, renorm;
  float scale;
};

template <class T>
__device__ __forceinline__ T wave_max_f(T v) {
  for (int o = 32; o >= 1; o >>= 1) {
    const T u = __shfl_xor(v, o, 64);
    v = u > v || v != v ? u : v;
  }
  return v;
}
template <class T>
__device__ __forceinline__ T wave_sum_f(T v) {
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// what this wave's lanes wrote to LDS is read by its other lanes after this
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// One token by one wave, the scores and every comparison in 64 bits: two experts
// next to each other are told apart whatever a rounding in 32 bits would say.
// sh: E doubles of this wave.
__device__ __forceinline__ void route_row64(const RouteArgs& p, int64_t t, int lane, double* sh) {
  constexpr int NV = ROUTE_MAX_E / 64;
  const double inf = __builtin_huge_val();
  double s[NV], key[NV];
  double m = -inf;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int e = lane + 64 * v;
    key[v] = e < p.E ? (double)route_load(p.z, t * p.E + e, p.bf16) : -inf;
    m = key[v] > m ? key[v] : m;
  }
  if (p.sigmoid) {
#pragma unroll
    for (int v = 0; v < NV; ++v) s[v] = 1.0 / (1.0 + exp(-key[v]));
  } else {
    m = wave_max_f(m);
    double sum = 0.0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      s[v] = lane + 64 * v < p.E ? exp(key[v] - m) : 0.0;
      sum += s[v];
    }
    sum = wave_sum_f(sum);
#pragma unroll
    for (int v = 0; v < NV; ++v) s[v] = s[v] / sum;
  }
  if (p.prob) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (lane + 64 * v < p.E) p.prob[t * p.E + lane + 64 * v] = (float)s[v];
  }
  // the choice's c in LDS for the groups; key: what the experts are ordered by
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int e = lane + 64 * v;
    if (e < p.E) {
      const double c = p.bias ? s[v] + (double)p.bias[e] : s[v];
      const bool live = key[v] > -inf && c > -inf;
      sh[e] = live ? c : -inf;
      key[v] = live ? (p.bias ? c : key[v]) : -inf;
    }
  }
  uint64_t in = ~0ull;
  const int per = p.E / p.groups;
  if (p.top_groups < p.groups) {
    wave_sync();
    double score = -inf;
    if (lane < p.groups) {
      double b1 = -inf, b2 = -inf;
      for (int j = 0; j < per; ++j) {
        const double c = sh[lane * per + j];
        b2 = c > b1 ? b1 : (c > b2 ? c : b2);
        b1 = c > b1 ? c : b1;
      }
      score = p.group_best == 2 && b2 > -inf ? b1 + b2 : b1;
    }
    int ahead = 0;
    for (int g = 0; g < p.groups; ++g) {
      const double o = __shfl(score, g, 64);
      ahead += o > score || (o == score && g < lane);
    }
    in = __ballot(lane < p.groups && ahead < p.top_groups);
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int e = lane + 64 * v;
    if (e < p.E && !((in >> (e / per)) & 1ull)) key[v] = -inf;
  }
  // the highest left, k times over; lane j keeps slot j
  int mine = -1, n = 0;
  double mys = 0.0, total = 0.0;
  for (int j = 0; j < p.k; ++j) {
    double bk = -inf, bs = 0.0;
    int be = 0x7fffffff;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (key[v] > bk) {
        bk = key[v];
        bs = s[v];
        be = lane + 64 * v;
      }
    for (int o = 32; o >= 1; o >>= 1) {
      const double k2 = __shfl_xor(bk, o, 64), s2 = __shfl_xor(bs, o, 64);
      const int e2 = __shfl_xor(be, o, 64);
      if (k2 > bk || (k2 == bk && e2 < be)) {
        bk = k2;
        bs = s2;
        be = e2;
      }
    }
    if (!(bk > -inf)) break;  // uniform: nobody is left
    if (lane == j) {
      mine = be;
      mys = bs;
    }
    ++n;
    total += bs;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (lane + 64 * v == be) key[v] = -inf;
  }
  if (lane < p.k) {
    double w = mys;
    if (p.renorm && mine >= 0) w = total < (double)ROUTE_MIN_SUM ? 1.0 / n : mys / total;
    p.topi[t * p.k + lane] = mine;
    p.topw[t * p.k + lane] = (float)(w * p.scale);
  }
  wave_sync();
}

constexpr int ROUTE_WAVES = 4;

__global__ void __launch_bounds__(ROUTE_WAVES * 64) route_kernel(RouteArgs p) {
  __shared__ double sh[ROUTE_WAVES][ROUTE_MAX_E];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * ROUTE_WAVES + wave;
  if (t < p.T) route_row64(p, t, lane, sh[wave]);
}

// ---------------------------------------------------------------------------
// backward: 16 lanes a token, V consecutive experts a lane
// ---------------------------------------------------------------------------
struct RouteGradArgs {
  const float* dtopw;
  const void* z;
  const int64_t* topi;
  const float* dprob;  // null: none
  void* dz;            // of z's type
  int64_t T;
  int E, k, bf16, sigmoid, renorm;
  float scale;
};

__device__ __forceinline__ float sum16(float v) {
  for (int o = 8; o >= 1; o >>= 1) v += __shfl_xor(v, o, 16);
  return v;
}

template <int V>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteGradArgs p) {
  const int l = threadIdx.x & 15;
  const int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  if (t >= p.T) return;  // whole groups of 16 lanes
  const int e0 = l * V;
  float s[V], ns[V], ds[V];
  float m = -__builtin_huge_valf();
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s[v] = e0 + v < p.E ? route_load(p.z, t * p.E + e0 + v, p.bf16) : -__builtin_huge_valf();
    m = fmaxf(m, s[v]);
    ds[v] = p.dprob && e0 + v < p.E ? p.dprob[t * p.E + e0 + v] : 0.0f;
  }
  for (int o = 8; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 16));
  float sum = 1.0f;
  if (p.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      ns[v] = 1.0f / (1.0f + expf(s[v]));
      s[v] = 1.0f / (1.0f + expf(-s[v]));
    }
  } else {
    sum = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = e0 + v < p.E ? expf(s[v] - m) : 0.0f;
      sum += s[v];
    }
    sum = sum16(sum);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = s[v] / sum;
  }
  // lane j has slot j: its score again, from its logit
  int64_t e = -1;
  float g = 0.0f, w = 0.0f;
  if (l < p.k) {
    e = p.topi[t * p.k + l];
    if (e >= 0 && e < p.E) {
      const float z = route_load(p.z, t * p.E + e, p.bf16);
      w = p.sigmoid ? 1.0f / (1.0f + expf(-z)) : expf(z - m) / sum;
      g = p.dtopw[t * p.k + l] * p.scale;
    } else {
      e = -1;
    }
  }
  if (p.renorm) {
    // w / W: dw = (g - sum g w / W) / W; the equal weights of a sum too small to
    // divide by do not depend on the scores
    const float total = sum16(w), mean = sum16(g * w) / total;
    g = total >= ROUTE_MIN_SUM ? (e >= 0 ? (g - mean) / total : 0.0f) : 0.0f;
  }
  const int ei = (int)e;
  for (int j = 0; j < p.k; ++j) {
    const int ej = __shfl(ei, j, 16);
    const float gj = __shfl(g, j, 16);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e0 + v == ej) ds[v] += gj;
  }
  float dot = 0.0f;
  if (!p.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) dot += s[v] * ds[v];
    dot = sum16(dot);
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (e0 + v < p.E) {
      const float d = p.sigmoid ? ds[v] * s[v] * ns[v] : s[v] * (ds[v] - dot);
      const int64_t i = t * p.E + e0 + v;
      if (p.bf16) ((__bf16*)p.dz)[i] = (__bf16)d;
      else ((float*)p.dz)[i] = d;
    }
}

int check_route(const char* what, int dtype, int64_t T, int64_t E, int64_t k, int score) {
  if (dtype != SMAUL_DTYPE_F32 && dtype != SMAUL_DTYPE_BF16) return fail(SMAUL_ERR_INVALID, "%s: bad dtype", what);
  if (T < 0 || E < 1 || k < 1 || k > E) return fail(SMAUL_ERR_INVALID, "%s: need T >= 0 and 1 <= k <= E", what);
  if (E > ROUTE_MAX_E || k > ROUTE_MAX_K)
    return fail(SMAUL_ERR_UNSUPPORTED, "%s: more than %d experts or top %d", what, ROUTE_MAX_E, ROUTE_MAX_K);
  if (score != SMAUL_SCORE_SOFTMAX && score != SMAUL_SCORE_SIGMOID)
    return fail(SMAUL_ERR_INVALID, "%s: bad score", what);
  if (T > (1LL << 31)) return fail(SMAUL_ERR_UNSUPPORTED, "%s: more than 2^31 tokens", what);
  return SMAUL_OK;
}

}  // namespace

extern "C" {

int smaul_moe_route(const void* logits, int dtype, const float* bias, float* prob, int64_t* topi, float* topw,
                    int64_t T, int64_t E, int64_t k, int score, int64_t groups, int64_t top_groups, int group_best,
                    int renorm, float scale, hipStream_t stream) {
  int rc = check_route("route", dtype, T, E, k, score);
  if (rc) return rc;
  if (groups < 1 || E % groups != 0 || top_groups < 1 || top_groups > groups || top_groups * (E / groups) < k)
    return fail(SMAUL_ERR_INVALID, "route: groups must divide E, and top_groups of them hold k experts");
  if (groups > ROUTE_MAX_G) return fail(SMAUL_ERR_UNSUPPORTED, "route: more than %d groups", ROUTE_MAX_G);
  if (group_best != 1 && group_best != 2) return fail(SMAUL_ERR_INVALID, "route: group_best must be 1 or 2");
  if (T == 0) return SMAUL_OK;
  if (!logits || !topi || !topw) return fail(SMAUL_ERR_INVALID, "route: null pointer");
  const RouteArgs p{logits, bias, prob, topi, topw, T, (int)E, (int)k, dtype == SMAUL_DTYPE_BF16,
                    score == SMAUL_SCORE_SIGMOID, (int)groups, (int)top_groups, group_best, renorm != 0, scale};
  hipLaunchKernelGGL(route_kernel, dim3((unsigned)((T + ROUTE_WAVES - 1) / ROUTE_WAVES)), dim3(ROUTE_WAVES * 64), 0,
                     stream, p);
  return check_launch("route_kernel");
}

int smaul_moe_route_backward(const float* dtopw, const void* logits, int dtype, const int64_t* topi,
                             const float* dprob, void* dlogits, int64_t T, int64_t E, int64_t k, int score,
                             int renorm, float scale, hipStream_t stream) {
  int rc = check_route("route_backward", dtype, T, E, k, score);
  if (rc) return rc;
  if (T == 0) return SMAUL_OK;
  if (!dtopw || !logits || !topi || !dlogits) return fail(SMAUL_ERR_INVALID, "route_backward: null pointer");
  const RouteGradArgs p{dtopw, logits, topi, dprob, dlogits, T, (int)E, (int)k, dtype == SMAUL_DTYPE_BF16,
                        score == SMAUL_SCORE_SIGMOID, renorm != 0, scale};
  const dim3 grid((unsigned)((T + 15) / 16)), block(256);
#define SMAUL_RB(V) hipLaunchKernelGGL((route_backward_kernel<V>), grid, block, 0, stream, p)
  if (E <= 16) SMAUL_RB(1);
  else if (E <= 64) SMAUL_RB(4);
  else if (E <= 128) SMAUL_RB(8);
  else if (E <= 256) SMAUL_RB(16);
  else SMAUL_RB(32);
#undef SMAUL_RB
  return check_launch("route_backward_kernel");
}

}  // extern "C"
