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
#include "e4m3.h"

using smaul::check_launch;
using smaul::fail;
using smaul::grid_fits;

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
// NV: ceil(E / 64) or more; sh: E doubles of this wave.
template <int NV>
__device__ __forceinline__ void route_row64(const RouteArgs& p, int64_t t, int lane, double* sh) {
  const double inf = __builtin_huge_val();
  double s[NV], key[NV];
  double m = -inf, sum = 1.0;
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
    sum = 0.0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      s[v] = lane + 64 * v < p.E ? exp(key[v] - m) : 0.0;
      sum += s[v];
    }
    sum = wave_sum_f(sum);
#pragma unroll
    for (int v = 0; v < NV; ++v) s[v] = s[v] / sum;
  }
  // the choice's c in LDS for the groups; key: what the experts are ordered by
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int e = lane + 64 * v;
    if (e < p.E) {
      if (p.prob) p.prob[t * p.E + e] = (float)s[v];
      const double c = p.bias ? s[v] + (double)p.bias[e] : s[v];
      const bool live = key[v] > -inf && c > -inf;
      sh[e] = live ? c : -inf;
      key[v] = live ? (p.bias ? c : key[v]) : -inf;
    }
  }
  if (p.top_groups < p.groups) {
    wave_sync();
    const int per = p.E / p.groups;
    double score = -inf;
    if (lane < p.groups) {
      double b1 = -inf, b2 = -inf;
#pragma unroll 8
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
    const uint64_t in = __ballot(lane < p.groups && ahead < p.top_groups);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int e = lane + 64 * v;
      if (e < p.E && !((in >> (e / per)) & 1ull)) key[v] = -inf;
    }
  }
  // the highest left, k times over; lane j keeps slot j
  int mine = -1, n = 0;
  for (int j = 0; j < p.k; ++j) {
    double bk = -inf;
    int be = 0x7fffffff;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (key[v] > bk) {
        bk = key[v];
        be = lane + 64 * v;
      }
    for (int o = 32; o >= 1; o >>= 1) {
      const double k2 = __shfl_xor(bk, o, 64);
      const int e2 = __shfl_xor(be, o, 64);
      if (k2 > bk || (k2 == bk && e2 < be)) {
        bk = k2;
        be = e2;
      }
    }
    if (!(bk > -inf)) break;  // uniform: nobody is left
    if (lane == j) mine = be;
    ++n;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (lane + 64 * v == be) key[v] = -inf;
  }
  double w = 0.0;
  if (mine >= 0) {
    const double z = (double)route_load(p.z, t * p.E + mine, p.bf16);
    w = p.sigmoid ? 1.0 / (1.0 + exp(-z)) : exp(z - m) / sum;
  }
  const double total = wave_sum_f(w);
  if (lane < p.k) {
    if (p.renorm && mine >= 0) w = total < (double)ROUTE_MIN_SUM ? 1.0 / n : w / total;
    p.topi[t * p.k + lane] = mine;
    p.topw[t * p.k + lane] = (float)(w * p.scale);
  }
  wave_sync();
}

// ---------------------------------------------------------------------------
// forward: 16 lanes a token, expert 16 v + lane in register v
// ---------------------------------------------------------------------------
// The scores are fp32.  An expert's key is one word: its c (or logit) as an ordered
// integer, the lowest bits replaced by V - 1 - v.  The highest key left is a maximum
// over the heads of a lane's lists and four lane exchanges; its low bits say which v, the
// lowest lane that has it which expert: equal values come out in the order of their index.
//
// What the rounding of the scores or those lost bits could change is not decided in 32
// bits: experts closer than the error bound are ordered by their c in 64 bits among
// the few found, and where two groups (the last one in, the first one out) or the
// scores of a softmax with a bias are that close, the token is done again by
// route_row64.  What bounds it is the vector instructions, about 1300 for four tokens of
// 256 experts: 65536 tokens take 47 us (their bytes 30), 225 in 64 bits throughout, one
// wave a token.
constexpr int ROUTE_WAVES = 4, ROUTE_TOK = ROUTE_WAVES * 4;

template <int CTRL>
__device__ __forceinline__ uint32_t row_ror(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// over the 16 lanes of a token, in every lane (rotations by 8, 4, 2, 1)
#define SMAUL_ROW_REDUCE(v, op)      \
  do {                               \
    v = op(v, row_ror<0x128>(v));    \
    v = op(v, row_ror<0x124>(v));    \
    v = op(v, row_ror<0x122>(v));    \
    v = op(v, row_ror<0x121>(v));    \
  } while (0)
__device__ __forceinline__ uint32_t op_umax(uint32_t a, uint32_t b) { return max(a, b); }
__device__ __forceinline__ uint32_t op_fmax(uint32_t a, uint32_t b) {
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
__device__ __forceinline__ uint32_t op_fadd(uint32_t a, uint32_t b) {
  return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}
__device__ __forceinline__ float row_max(float v) {
  uint32_t u = __float_as_uint(v);
  SMAUL_ROW_REDUCE(u, op_fmax);
  return __uint_as_float(u);
}
__device__ __forceinline__ float row_sum(float v) {
  uint32_t u = __float_as_uint(v);
  SMAUL_ROW_REDUCE(u, op_fadd);
  return __uint_as_float(u);
}

// exp, to |x| 2^-24 of its value and two units
__device__ __forceinline__ float route_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float route_score(float z, int sigmoid, float m, float inv) {
  return sigmoid ? __builtin_amdgcn_rcpf(1.0f + route_exp(-z)) : route_exp(z - m) * inv;
}

// floats as integers of the same order
__device__ __forceinline__ uint32_t route_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float route_unkey(uint32_t k) {
  return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k);
}

template <int V>
__global__ void __launch_bounds__(ROUTE_WAVES * 64) route_kernel(RouteArgs p) {
  constexpr uint32_t LOW = V - 1;
  constexpr float INF = __builtin_huge_valf();
  // route_row64's doubles, or the c of the wave's four tokens
  constexpr int SH = 4 * (V * 16 + 8) / 2 > ROUTE_MAX_E ? 4 * (V * 16 + 8) / 2 : ROUTE_MAX_E;
  __shared__ double sh64[ROUTE_WAVES][SH];
  __shared__ uint32_t shg[ROUTE_TOK][ROUTE_MAX_G];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, tq = lane >> 4;
  const int64_t t = (int64_t)blockIdx.x * ROUTE_TOK + threadIdx.x / 16;
  const bool on = t < p.T;
  const int64_t row = (on ? t : p.T - 1) * p.E;  // lanes past the end follow along, and store nothing
  float z[V], s[V], b[V];
  // whole sixteens, known to all lanes, need no comparison in each
  auto each = [&](auto f, auto past) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if ((v + 1) * 16 <= p.E || v * 16 + l < p.E) f(v);
      else past(v);
    }
  };
  if (p.bf16) {
    const uint16_t* at = (const uint16_t*)p.z + row + l;
    each([&](int v) { z[v] = bf2f(at[v * 16]); }, [&](int v) { z[v] = -INF; });
  } else {
    const float* at = (const float*)p.z + row + l;
    each([&](int v) { z[v] = at[v * 16]; }, [&](int v) { z[v] = -INF; });
  }
  if (p.bias) each([&](int v) { b[v] = p.bias[l + v * 16]; }, [&](int v) { b[v] = 0.0f; });
  float m = -INF, inv = 1.0f;
  if (!p.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) m = fmaxf(m, z[v]);
    m = row_max(m);
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = v * 16 + l < p.E ? route_exp(z[v] - m) : 0.0f;
      sum += s[v];
    }
    inv = 1.0f / row_sum(sum);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = s[v] * inv;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = route_score(z[v], 1, 0.0f, 0.0f);
  }
  if (p.prob && on) {
    float* at = p.prob + row + l;
    each([&](int v) { at[v * 16] = s[v]; }, [](int) {});
  }
  // Error of a c: the sum's V + 4 roundings and the exponential's, on scores of at
  // most s_top (the row's highest), and the rounding of c itself.
  const float s_err = (p.sigmoid ? 1.0f : inv) * (V + 16) * 0x1p-24f;
  uint32_t key[V];
  auto set_key = [&](int v, float c, float by) {  // by: what the choice goes by
    const bool live = z[v] > -INF && c > -INF;
    s[v] = live ? c : -INF;  // from here on: c
    key[v] = live ? (route_key(by) & ~LOW) | (LOW - v) : 0u;
  };
  if constexpr (V > 16) {  // the registers of both loops would cost more waves than they save
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float c = p.bias ? s[v] + b[v] : s[v];
      set_key(v, c, p.bias ? c : z[v] + 0.0f);
    }
  } else if (p.bias) {
#pragma unroll
    for (int v = 0; v < V; ++v) set_key(v, s[v] + b[v], s[v] + b[v]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) set_key(v, s[v], z[v] + 0.0f);  // -0 is 0: a tie
  }
  bool tied = false;  // groups in and out too near
  if (p.top_groups < p.groups) {
    // c to LDS, a group to a lane; the groups' scores to LDS, and each lane counts
    // the groups ahead of its own
    float* sc = (float*)sh64[wave] + tq * (V * 16 + 8);  // 8: the tokens' rows in other banks
#pragma unroll
    for (int v = 0; v < V; ++v) sc[v * 16 + l] = s[v];
    wave_sync();
    const int per = p.E / p.groups;
    uint32_t* sg = shg[wave * 4 + tq];  // the groups' scores, ordered as integers
    float top = 0.0f;
    for (int g = l; g < p.groups; g += 16) {
      float b1 = -INF, b2 = -INF;
      auto take = [&](float c) {
        b2 = __builtin_amdgcn_fmed3f(b1, b2, c);
        asm("v_max_f32 %0, %1, %2" : "=v"(b1) : "v"(b1), "v"(c));  // fmaxf makes its operands canonical first
      };
      // each lane from another place on: other banks
      if (per % 4 == 0) {
        int i = 4 * l % per;
        for (int j = 0; j < per; j += 4) {
          const float4 c = *(const float4*)(sc + g * per + i);
          i = i + 4 == per ? 0 : i + 4;
          take(c.x);
          take(c.y);
          take(c.z);
          take(c.w);
        }
      } else {
        int i = l % per;
        for (int j = 0; j < per; ++j) {
          take(sc[g * per + i]);
          i = i + 1 == per ? 0 : i + 1;
        }
      }
      const float score = p.group_best == 2 && b2 > -INF ? b1 + b2 : b1;
      sg[g] = route_key(score + 0.0f);
      if (b1 > -INF) top = fmaxf(top, fmaxf(fabsf(b1), fabsf(score)));
    }
    wave_sync();
    uint64_t in = 0;
    float lowest = INF, highest = -INF;  // of the groups in and out
    for (int g0 = 0; g0 < p.groups; g0 += 16) {
      const int g = g0 + l;
      bool chosen = false;
      if (g < p.groups) {
        const uint32_t own = sg[g];
        const float mine = route_unkey(own);
        int ahead = 0;
        for (int o = 0; o < p.groups; ++o) ahead += sg[o] + (o < g ? 1u : 0u) > own;  // ties: the first
        chosen = ahead < p.top_groups;
        if (chosen) lowest = fminf(lowest, mine);
        else highest = fmaxf(highest, mine);
      }
      in |= (__ballot(chosen) >> (tq * 16) & 0xffffull) << g0;
    }
    lowest = -row_max(-lowest);
    highest = row_max(highest);
    top = row_max(top);
    // groups without a live expert may change places
    tied = highest > -INF && lowest - highest <= 4.0f * s_err + 8.0f * 0x1p-24f * top;
    const uint32_t in0 = (uint32_t)in, in1 = (uint32_t)(in >> 32);
    auto keep = [&](int v, uint32_t g) {
      const uint32_t word = p.groups > 32 && g >= 32 ? in1 : in0;
      key[v] &= (uint32_t)__builtin_amdgcn_sbfe((int)word, g & 31, 1);
    };
    const uint32_t magic = ((1u << 20) + per - 1) / per;  // e / per for e, per <= 512
    if (per % 16 == 0) {  // a sixteen is of one group
#pragma unroll
      for (int v = 0; v < V; ++v) keep(v, v * 16u * magic >> 20);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) keep(v, (v * 16 + l) * magic >> 20);
    }
  }
  // Lane j gets the j-th highest, and its key.  A lane's keys are lists of four in order,
  // so that a round looks at their heads alone, and a list whose head is gone moves up.
  constexpr int L = V < 4 ? V : 4;
  auto order = [&](int a, int b) {
    const uint32_t high = max(key[a], key[b]), low = min(key[a], key[b]);
    key[a] = high;
    key[b] = low;
  };
#pragma unroll
  for (int v = 0; v < V; v += L) {
    if constexpr (L == 2) order(v, v + 1);
    if constexpr (L == 4) {
      order(v, v + 1);
      order(v + 2, v + 3);
      order(v, v + 2);
      order(v + 1, v + 3);
      order(v + 1, v + 2);
    }
  }
  int mine = -1;
  uint32_t val = 0u, best = 0u;
  auto highest = [&]() {  // the lane's; best: the token's
    uint32_t own = key[0];
#pragma unroll
    for (int v = L; v < V; v += L) own = max(own, key[v]);
    best = own;
    SMAUL_ROW_REDUCE(best, op_umax);
    return own;
  };
  auto take = [&](uint32_t own, bool store) {
    // the lowest lane that has it
    const uint32_t has = (uint32_t)(__ballot(own == best) >> (tq * 16)) & 0xffffu;
    const int owner = __builtin_ctz(has);
    if (store) {
      val = best;
      mine = (int)(LOW - (best & LOW)) * 16 + owner;
    }
    const uint32_t gone = l == owner ? best : 1u;  // 1: no key (a live one is over 2^22)
#pragma unroll
    for (int v = 0; v < V; v += L) {
      const bool up = key[v] == gone;
#pragma unroll
      for (int j = 0; j < L; ++j) key[v + j] = up ? (j + 1 < L ? key[v + j + 1] : 0u) : key[v + j];
    }
  };
  for (int j = 0; j < p.k; ++j) {
    const uint32_t own = highest();
    take(own, l == j);
  }
  if (val == 0u) mine = -1;
  int n = __popc((uint32_t)(__ballot(val != 0u) >> (tq * 16)) & 0xffffu);
  // is b, which is not above a, too near to be told apart?
  auto too_near = [&](uint32_t a, uint32_t b) {
    const uint32_t ua = a & ~LOW, ub = b & ~LOW;
    if (b == 0u) return false;
    if (!p.bias) return !p.bf16 && ua == ub;  // logits that the low bits may tell apart
    const float fa = route_unkey(ua), fb = route_unkey(ub);
    // each c is off by s_err and half a unit, the second may gain V units by its low bits
    return !(fa - fb > 2.0f * s_err + (V + 2) * 0x1p-23f * fmaxf(fabsf(fa), fabsf(fb)));
  };
  // lane j: the j-th and the one before; lane 0: the last and the next that is left out
  uint32_t own = highest();
  const int from = l == 0 ? p.k - 1 : l - 1;
  const uint32_t before = (uint32_t)__shfl((int)val, from, 16);
  const bool close = l < p.k && too_near(before, l == 0 ? best : val);
  bool again = tied, near = false, on_and_on = false;
  if (__ballot(close || tied)) {
    // Experts of one logit and one bias are equal in 64 bits too, and stand in the order
    // of their indices as it is: a batch's padding, whose experts are all the same, needs
    // no second look (512 rows of it took 20 us of 25).
    const float zm = mine >= 0 ? route_load(p.z, row + mine, p.bf16) : 0.0f;
    const float bm = p.bias && mine >= 0 ? p.bias[mine] : 0.0f;
    const bool differ = !(zm == __shfl(zm, from, 16) && bm == __shfl(bm, from, 16));
    auto any = [&](bool q) { return ((uint32_t)(__ballot(q) >> (tq * 16)) & 0xffffu) != 0u; };
    near = any(close && l > 0 && differ);
    // the last that is chosen, and the next
    const float zr = __shfl(zm, p.k - 1, 16), br = __shfl(bm, p.k - 1, 16);
    const bool border = any(close && l == 0);
    bool even = false;
    if (border) {  // best is no 0
      const int next = (int)(LOW - (best & LOW)) * 16 +
                       __builtin_ctz((uint32_t)(__ballot(own == best) >> (tq * 16)) & 0xffffu);
      even = route_load(p.z, row + next, p.bf16) == zr && (!p.bias || p.bias[next] == br);
    }
    // Where they are equal: is any other expert near them?  And where groups tie: is
    // any expert other than the chosen, which are all equal?
    const bool scan = even || (tied && !any(l > 0 && l < p.k && differ));
    const uint32_t ur = (uint32_t)__shfl((int)val, p.k - 1, 16) & ~LOW;
    const float fr = route_unkey(ur);
    bool other = false, uneven = false;
    for (int e = __ballot(scan) ? l : p.E; e < p.E; e += 16) {
      const float z = route_load(p.z, row + e, p.bf16) + 0.0f, be = p.bias ? p.bias[e] : 0.0f;
      if (z == zr && be == br) continue;
      uneven = true;
      const float c = p.bias ? route_score(z, p.sigmoid, m, inv) + be : z;
      // twice too_near's bound, on either side
      other |= p.bias ? !(fabsf(fr - c) > 4.0f * s_err + (2 * V + 4) * 0x1p-23f * fmaxf(fabsf(fr), fabsf(c)))
                      : (route_key(c) & ~LOW) == ur;
    }
    on_and_on = border && (!even || any(other));
    near |= on_and_on;
    again = tied && (!scan || any(uneven));
  }
  // the walk goes on past k while the next is too near to the last to be left out
  uint32_t last = best;
  for (int j = p.k; __ballot(on_and_on); ++j) {
    if (on_and_on && j == 16) {  // more of them than lanes
      again = true;
      on_and_on = false;
    }
    if (on_and_on) n = j + 1;
    last = best;
    take(own, on_and_on && l == j);
    own = highest();
    on_and_on = on_and_on && too_near(last, best);
  }
  // Neighbours too near for 32 bits: the n found are ordered by what they are in 64
  // (the sum of a softmax with a bias is left to route_row64).
  if (p.bias && !p.sigmoid) again |= near;
  if (__ballot(near && !again)) {
    double x = -__builtin_huge_val();
    if (mine >= 0) {
      x = (double)route_load(p.z, row + mine, p.bf16);
      if (p.bias) x = 1.0 / (1.0 + exp(-x)) + (double)p.bias[mine];
    }
    int ahead = 0;
    for (int i = 0; i < 16; ++i) {
      const double y = __shfl(x, i, 16);
      const int e = __shfl(mine, i, 16);
      ahead += y > x || (y == x && e < mine);
    }
    int sorted = -1;
    for (int i = 0; i < 16; ++i) {
      const int e = __shfl(mine, i, 16), at = __shfl(ahead, i, 16);
      if (e >= 0 && at == l) sorted = e;
    }
    mine = sorted;
  }
  if (l >= p.k) mine = -1;
  n = min(n, p.k);
  float w = 0.0f;
  if (mine >= 0) w = route_score(route_load(p.z, row + mine, p.bf16), p.sigmoid, m, inv);
  const float total = row_sum(w);
  if (p.renorm && mine >= 0) w = total < ROUTE_MIN_SUM ? 1.0f / n : w / total;
  // a sum next to the guard's border is the 64-bit form's to decide
  if (p.renorm) again |= fabsf(total - ROUTE_MIN_SUM) <= 64 * 0x1p-24f * ROUTE_MIN_SUM;
  if (on && l < p.k) {
    p.topi[t * p.k + l] = mine;
    p.topw[t * p.k + l] = w * p.scale;
  }
  uint64_t redo = __ballot(again && on && l == 0);
  while (redo) {  // uniform
    const int q = __builtin_ctzll(redo) >> 4;
    redo &= redo - 1;
    route_row64<(V + 3) / 4>(p, (int64_t)blockIdx.x * ROUTE_TOK + wave * 4 + q, lane, sh64[wave]);
  }
}

// ---------------------------------------------------------------------------
// Backward.  A score's gradient is dprob's, plus for a chosen expert scale dtopw, with
// renorm through w / sum w; then softmax's s (ds - sum s ds) or sigmoid's ds s (1 - s).
// A masked expert (-inf, a score of 0) has no gradient and gives none, whatever dprob holds
// there, nor does a row that has no other: its products are those where 0 times anything
// is 0 (a comparison for each score takes 8 % more time).
// One pass over z, dprob and dz, and their bytes are what it costs (65536 x 256 fp32, 201
// MB: 36 us, 5.5 TB/s).  16 lanes a token, V experts a lane.  VEC (E % 4 == 0, 16-byte aligned): four
// neighbours at a time, so that a token's lanes read 256 bytes in a row (140 us with each lane's V in a row).
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

// a b, and 0 where either is 0, whatever the other
__device__ __forceinline__ float mul_zero(float a, float b) {
  float r;
  asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

template <int V, bool VEC>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteGradArgs p) {
  constexpr float INF = __builtin_huge_valf();
  const int l = threadIdx.x & 15;
  const int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4, row = t * p.E;
  if (t >= p.T) return;  // whole groups of 16 lanes
  auto expert = [&](int v) { return VEC ? v / 4 * 64 + 4 * l + v % 4 : v * 16 + l; };
  float s[V], ns[V], ds[V];  // scores, 1 - them (sigmoid), their gradients
  if constexpr (VEC) {
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      const bool in = expert(v) < p.E;
      float4 z = make_float4(-INF, -INF, -INF, -INF), d = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (in && p.bf16) {
        const uint2 u = *(const uint2*)((const uint16_t*)p.z + row + expert(v));
        z = make_float4(bf2f(u.x & 0xffffu), bf2f(u.x >> 16), bf2f(u.y & 0xffffu), bf2f(u.y >> 16));
      } else if (in) {
        z = *(const float4*)((const float*)p.z + row + expert(v));
      }
      if (in && p.dprob) d = *(const float4*)(p.dprob + row + expert(v));
      s[v] = z.x; s[v + 1] = z.y; s[v + 2] = z.z; s[v + 3] = z.w;
      ds[v] = d.x; ds[v + 1] = d.y; ds[v + 2] = d.z; ds[v + 3] = d.w;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool in = expert(v) < p.E;
      s[v] = in ? route_load(p.z, row + expert(v), p.bf16) : -INF;
      ds[v] = in && p.dprob ? p.dprob[row + expert(v)] : 0.0f;
    }
  }
  // lane j has slot j: its score again, from its logit
  int64_t e = -1;
  float zj = 0.0f, g = 0.0f, w = 0.0f;
  if (l < p.k) {
    e = p.topi[t * p.k + l];
    if (e >= 0 && e < p.E) {
      zj = route_load(p.z, row + e, p.bf16);
      g = p.dtopw[t * p.k + l] * p.scale;
    } else {
      e = -1;
    }
  }
  float m = 0.0f, inv = 0.0f;
  if (p.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float x = route_exp(-fabsf(s[v])), r = __builtin_amdgcn_rcpf(1.0f + x), xr = x * r;
      ns[v] = s[v] < 0.0f ? r : xr;
      s[v] = s[v] < 0.0f ? xr : r;
    }
  } else {
    m = -INF;
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) m = fmaxf(m, s[v]);
    m = row_max(m);
    m = m == -INF ? 0.0f : m;  // nobody: scores of 0
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = expert(v) < p.E ? route_exp(s[v] - m) : 0.0f;
      sum += s[v];
    }
    sum = row_sum(sum);
    inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] *= inv;
  }
  if (e >= 0) w = route_score(zj, p.sigmoid, m, inv);
  if (p.renorm) {
    // w / W: dw = (g - sum g w / W) / W; the equal weights of a sum too small to
    // divide by do not depend on the scores
    const float total = row_sum(w), mean = row_sum(g * w) / total;
    g = total >= ROUTE_MIN_SUM ? (e >= 0 ? (g - mean) / total : 0.0f) : 0.0f;
  }
  const int ei = (int)e;
  for (int j = 0; j < p.k; ++j) {
    const int ej = __shfl(ei, j, 16);
    const float gj = __shfl(g, j, 16);
#pragma unroll
    for (int v = 0; v < V; ++v) ds[v] += expert(v) == ej ? gj : 0.0f;
  }
  float dot = 0.0f;
  if (!p.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) dot += mul_zero(s[v], ds[v]);
    dot = row_sum(dot);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float m0 = mul_zero(s[v], p.sigmoid ? ds[v] : ds[v] - dot);
    ds[v] = p.sigmoid ? m0 * ns[v] : m0;
  }
  if constexpr (VEC) {
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      if (expert(v) >= p.E) continue;
      if (p.bf16)
        *(uint2*)((uint16_t*)p.dz + row + expert(v)) =
            make_uint2(pack_bf16(ds[v], ds[v + 1]), pack_bf16(ds[v + 2], ds[v + 3]));
      else *(float4*)((float*)p.dz + row + expert(v)) = make_float4(ds[v], ds[v + 1], ds[v + 2], ds[v + 3]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (expert(v) >= p.E) continue;
      if (p.bf16) ((__bf16*)p.dz)[row + expert(v)] = (__bf16)ds[v];
      else ((float*)p.dz)[row + expert(v)] = ds[v];
    }
  }
}

int check_route(const char* what, int dtype, int64_t T, int64_t E, int64_t k, int score) {
  if (dtype != SMAUL_DTYPE_F32 && dtype != SMAUL_DTYPE_BF16) return fail(SMAUL_ERR_INVALID, "%s: bad dtype", what);
  if (T < 0 || E < 1 || k < 1 || k > E) return fail(SMAUL_ERR_INVALID, "%s: need T >= 0 and 1 <= k <= E", what);
  if (E > ROUTE_MAX_E || k > ROUTE_MAX_K)
    return fail(SMAUL_ERR_UNSUPPORTED, "%s: more than %d experts or top %d", what, ROUTE_MAX_E, ROUTE_MAX_K);
  if (score != SMAUL_SCORE_SOFTMAX && score != SMAUL_SCORE_SIGMOID)
    return fail(SMAUL_ERR_INVALID, "%s: bad score", what);
  if (!grid_fits((T + 15) / 16, 256)) return fail(SMAUL_ERR_UNSUPPORTED, "%s: 2^28 tokens or more", what);
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
  const dim3 grid((unsigned)((T + ROUTE_TOK - 1) / ROUTE_TOK)), block(ROUTE_WAVES * 64);
#define SMAUL_R(V) hipLaunchKernelGGL((route_kernel<V>), grid, block, 0, stream, p)
  if (E <= 16) SMAUL_R(1);
  else if (E <= 32) SMAUL_R(2);
  else if (E <= 64) SMAUL_R(4);
  else if (E <= 128) SMAUL_R(8);
  else if (E <= 256) SMAUL_R(16);
  else SMAUL_R(32);
#undef SMAUL_R
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
  const bool vec = E % 4 == 0 && (((uintptr_t)logits | (uintptr_t)dlogits | (uintptr_t)dprob) & 15) == 0;
#define SMAUL_RB(V)                                                                              \
  do {                                                                                           \
    if (vec) hipLaunchKernelGGL((route_backward_kernel<V, true>), grid, block, 0, stream, p);    \
    else hipLaunchKernelGGL((route_backward_kernel<V, false>), grid, block, 0, stream, p);       \
  } while (0)
  if (E <= 64) SMAUL_RB(4);
  else if (E <= 128) SMAUL_RB(8);
  else if (E <= 256) SMAUL_RB(16);
  else SMAUL_RB(32);
#undef SMAUL_RB
  return check_launch("route_backward_kernel");
}

}  // extern "C"
