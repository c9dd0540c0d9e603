// Routing from given logits and its backward, with their C entry points: softmax or sigmoid scores, a selection bias,
// groups, top-k, renormalised weights.
#include "hmoe_common.h"

namespace hmoe {

// Four tokens per wave: the 16 lanes of segment q take one token, lane j of it experts 16 i + j (i < EPL).
// What bounds it: the selection's instructions (an fp64 score per expert, the sorting network) and their latency; the logits
// are read once, 8 MB at 8192 x 256, 2 us at the rate of a large copy.  Sixteen lanes a token: a wave's exchanges stay inside
// rows of 16 lanes (DPP), and four tokens share every instruction.  8192 tokens, 256 experts in 8 groups, top-8, sigmoid with
// bias: 11.0 us; with the library's exp and division and the options branched on per element 15.1.  The best k of E by a
// sorting network and four merges of lists across the lanes, not by k rounds of arg-max: those cost about 110 instructions
// each, the network 38 and a merge 55 for lists of eight.
constexpr int kGateMaxE = 512, kGateMaxK = 16, kGateMaxGroups = 64;
constexpr double kGateDead = -1e300;    // an expert that cannot be chosen while another is left
constexpr double kGateNone = -1.5e308;  // no expert

struct GateArgs {
  const void* logits;
  int64_t ld;
  int dt;
  const float* bias;
  const uint8_t* live;
  int T, E, k, sigmoid, renorm, n_group, topk_group, group_top;
  uint32_t inv_eg;  // ceil(2^20 / experts per group): (e * inv_eg) >> 20 is e's group for e < 512
  float scaling;
  int32_t* ids;
  float* w;
};

__device__ __forceinline__ float gate_logit(const GateArgs& a, int64_t t, int e) {
  const int64_t i = t * a.ld + e;
  if (a.dt == HMOE_DT_F32) return static_cast<const float*>(a.logits)[i];
  const uint16_t b = static_cast<const uint16_t*>(a.logits)[i];
  return a.dt == HMOE_DT_F16 ? Elt<true>::one(b) : bf2f(b);
}
// a lane's logits: experts 16 i + j, -inf past E.  All loads first (the index is held inside the row), the type once.
template <int EPL>
__device__ __forceinline__ void gate_logits(const GateArgs& a, int64_t t, int j, float (&lg)[EPL]) {
  if (a.dt == HMOE_DT_F32) {
    const float* p = static_cast<const float*>(a.logits) + t * a.ld;
#pragma unroll
    for (int i = 0; i < EPL; ++i) lg[i] = p[min(16 * i + j, a.E - 1)];
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(a.logits) + t * a.ld;
    uint16_t w[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) w[i] = p[min(16 * i + j, a.E - 1)];
#pragma unroll
    for (int i = 0; i < EPL; ++i) lg[i] = a.dt == HMOE_DT_F16 ? Elt<true>::one(w[i]) : bf2f(w[i]);
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) lg[i] = 16 * i + j < a.E ? lg[i] : -__builtin_inff();
}

// max / min without the quieting of NaN that fmax does (no operand is a NaN)
__device__ __forceinline__ double dmax(double a, double b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ double dmin(double a, double b) {
  double r;
  asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

template <int S>
__device__ __forceinline__ double lane_xor_d(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)lane_xor_i<S>((int)(uint32_t)u), hi = (uint32_t)lane_xor_i<S>((int)(uint32_t)(u >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// sums over the 16 lanes of a segment, every lane ending with the same value
__device__ __forceinline__ float seg_sum(float v) {
  v = bfly_add<8>(v);
  v = bfly_add<4>(v);
  v = bfly_add<2>(v);
  return bfly_add<1>(v);
}
__device__ __forceinline__ float seg_max(float v) {
  v = bfly_max<8>(v);
  v = bfly_max<4>(v);
  v = bfly_max<2>(v);
  return bfly_max<1>(v);
}
__device__ __forceinline__ double seg_sum_d(double v) {
  v += lane_xor_d<8>(v);
  v += lane_xor_d<4>(v);
  v += lane_xor_d<2>(v);
  return v + lane_xor_d<1>(v);
}

// a b + c with c in scalar registers (the compiler would copy such a constant into vector registers for every element)
__device__ __forceinline__ double fma_sc(double a, double b, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}

// exp in fp64 to about 1e-14: x = n ln 2 + r (one fma: the product is exact, and ln 2 itself is off by 2e-17 n), then the
// Taylor polynomial of degree 11 on |r| <= ln 2 / 2, whose first dropped term is below 7e-15, and the scaling by 2^n.  Finer
// than the 43 bits a sort key keeps, and a third of the library function's instructions.  Inputs beyond 1e4 in absolute value
// are clamped there: the results are 0 or inf either way.
__device__ __forceinline__ double gate_exp(double x) {
  x = dmin(dmax(x, -1e4), 1e4);
  const double n = __builtin_rint(x * 1.4426950408889634074);
  const double r = __builtin_fma(n, -0.69314718055994530942, x);
  double p = 1.0 / 39916800.0;
  p = fma_sc(p, r, 1.0 / 3628800.0);
  p = fma_sc(p, r, 1.0 / 362880.0);
  p = fma_sc(p, r, 1.0 / 40320.0);
  p = fma_sc(p, r, 1.0 / 5040.0);
  p = fma_sc(p, r, 1.0 / 720.0);
  p = fma_sc(p, r, 1.0 / 120.0);
  p = fma_sc(p, r, 1.0 / 24.0);
  p = fma_sc(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_ldexp(p, (int)n);
}
// 1 / x for 1 <= x: the hardware's estimate and two Newton steps (x = inf: 0)
__device__ __forceinline__ double gate_rcp(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
  r = __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
  return x < 1e300 ? r : 0.0;
}

// Sort keys.  The selection value in fp64, its lowest nine mantissa bits replaced by the expert's index so that equal
// values order by the lower index: one v_max_f64 / v_min_f64 then compares value and index at once.  43 mantissa bits
// stay, more than an fp32 logit has (selection without bias and groups is exact) and 2^20 times finer than an fp32 score.
__device__ __forceinline__ double gate_key(double v, int e) {
  v = v > -1e299 ? (v < 1e300 ? v : 1e300) : kGateDead;
  v += 0.0;  // -0 -> +0
  uint64_t u = __builtin_bit_cast(uint64_t, v) & ~(uint64_t)511;
  u |= (uint64_t)(v < 0.0 ? e : 511 - e);
  return __builtin_bit_cast(double, u);
}
__device__ __forceinline__ int gate_key_expert(double key) {
  const int low = (int)(__builtin_bit_cast(uint64_t, key) & 511);
  return key < 0.0 ? low : 511 - low;
}

// descending bitonic networks over registers
template <int N>
__device__ __forceinline__ void bitonic_merge(double (&a)[N], int base, int n, bool desc) {
#pragma unroll
  for (int s = n / 2; s > 0; s >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i)
      if (!(i & s)) {
        const double x = a[base + i], y = a[base + i + s];
        a[base + i] = desc ? dmax(x, y) : dmin(x, y);
        a[base + i + s] = desc ? dmin(x, y) : dmax(x, y);
      }
}
template <int N>
__device__ __forceinline__ void bitonic_sort(double (&a)[N]) {
#pragma unroll
  for (int n = 2; n <= N; n <<= 1)
#pragma unroll
    for (int b = 0; b < N; b += n) bitonic_merge(a, b, n, n == N || !(b & n));
}
// the largest N of two descending lists, descending, in a
template <int N>
__device__ __forceinline__ void keep_top(double (&a)[N], const double (&b)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = dmax(a[i], b[N - 1 - i]);
  bitonic_merge(a, 0, N, true);
}
template <int S, int N>
__device__ __forceinline__ void keep_top_xor(double (&a)[N]) {
  double b[N];
#pragma unroll
  for (int i = 0; i < N; ++i) b[i] = lane_xor_d<S>(a[i]);
  keep_top(a, b);
}

__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// L: list length, the power of two at or above k.
template <int EPL, int L, bool GROUPS, bool SIG>
__global__ __launch_bounds__(256) void route_scores_kernel(GateArgs a) {
  constexpr int W = 4;
  __shared__ double s_key[GROUPS ? W * 4 : 1][GROUPS ? EPL * 16 : 1];
  __shared__ double s_grp[GROUPS ? W * 4 : 1][GROUPS ? kGateMaxGroups : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, seg = lane >> 4;
  const int64_t tw = ((int64_t)blockIdx.x * W + wave) * 4;
  if (tw >= a.T) return;
  const int64_t t = tw + seg < a.T ? tw + seg : a.T - 1;  // (the lanes past T redo the last token and store nothing)
  float lg[EPL], bias[EPL];
  gate_logits(a, t, j, lg);
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) bias[i] = a.bias[min(16 * i + j, a.E - 1)];
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) bias[i] = 0.0f;
  }
  // softmax: the row's largest logit and the sum of exp(l - m); a row without a logit above -inf has the sum 0 and scores 0
  float m = -__builtin_inff(), S = 1.0f;
  if constexpr (!SIG) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) m = fmaxf(m, lg[i]);
    m = seg_max(m);
    S = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float x = hexp(lg[i] - m);
      S += lg[i] != -__builtin_inff() ? x : 0.0f;
    }
    S = seg_sum(S);
  }
  // selection values
  double v[EPL];
  if (GROUPS || a.bias) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      if constexpr (SIG) {
        v[i] = gate_rcp(1.0 + gate_exp(-(double)lg[i]));
      } else {
        const double x = gate_exp((double)lg[i] - (double)m);
        v[i] = lg[i] > -__builtin_inff() ? x : 0.0;
        sum += v[i];
      }
    }
    const double inv = SIG ? 1.0 : 1.0 / seg_sum_d(sum);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const bool on = lg[i] > -__builtin_inff() && bias[i] > -__builtin_inff();
      const double x = v[i] * inv + (double)bias[i];
      v[i] = on ? x : -__builtin_inf();
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) v[i] = lg[i] > -__builtin_inff() ? (double)lg[i] : -__builtin_inf();
  }
  if constexpr (GROUPS) {
    double* key = s_key[wave * 4 + seg];
    double* grp = s_grp[wave * 4 + seg];
    const int eg = a.E / a.n_group;
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[16 * i + j] = v[i] == v[i] ? v[i] : -__builtin_inf();
    wave_lds_sync();
    // groups 16 q + j, or with at most eight of them lanes j and j + 8 half of group j each
    const int parts = a.n_group <= 8 ? 2 : 1, part = parts == 2 ? j >> 3 : 0;
    double mine[kGateMaxGroups / 16];
#pragma unroll
    for (int q = 0; q < kGateMaxGroups / 16; ++q) {
      mine[q] = -__builtin_inf();
      if (16 * q >= a.n_group) break;
      const int g = parts == 2 ? j & 7 : 16 * q + j;
      const bool have = g < a.n_group;
      double m1 = -__builtin_inf(), m2 = -__builtin_inf();
      const double* gk = key + (have ? g * eg : 0);
      for (int i0 = part; i0 < eg; i0 += 4 * parts) {
        double x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = gk[min(i0 + i * parts, eg - 1)];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double y = i0 + i * parts < eg ? x[i] : -__builtin_inf();
          m2 = dmax(m2, dmin(m1, y));
          m1 = dmax(m1, y);
        }
      }
      if (parts == 2) {
        const double o1 = lane_xor_d<8>(m1), o2 = lane_xor_d<8>(m2);
        m2 = dmax(dmin(m1, o1), dmax(m2, o2));
        m1 = dmax(m1, o1);
      }
      const double val = a.group_top == 2 ? m1 + m2 : m1;
      mine[q] = have && val == val ? val : -__builtin_inf();
      if (have) grp[g] = mine[q];
    }
    wave_lds_sync();
    uint64_t kept = 0;
#pragma unroll
    for (int q = 0; q < kGateMaxGroups / 16; ++q) {
      if (16 * q >= a.n_group) break;
      const int g = parts == 2 ? j & 7 : 16 * q + j;
      int before = 0;  // groups ahead of mine
      for (int o = 0; o < a.n_group; ++o) {
        const double x = grp[o];
        before += x > mine[q] || (x == mine[q] && o < g);
      }
      const uint64_t vote = __ballot(g < a.n_group && before < a.topk_group);
      kept |= (vote >> (16 * seg) & 0xffff) << (16 * q);
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const uint32_t g = ((uint32_t)(16 * i + j) * a.inv_eg) >> 20;
      v[i] = kept >> (g & 63) & 1 ? v[i] : -__builtin_inf();
    }
  }
  // top L of the lane's own, then of pairs of lanes
  double top[L];
  constexpr int CH = (EPL + L - 1) / L;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    double x[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int ii = c * L + i, e = 16 * ii + j;
      if (ii < EPL) {
        const double key = gate_key(v[ii < EPL ? ii : 0], e);
        x[i] = e < a.E ? key : kGateNone;
      } else {
        x[i] = kGateNone;
      }
    }
    bitonic_sort(x);
    if (c == 0) {
#pragma unroll
      for (int i = 0; i < L; ++i) top[i] = x[i];
    } else {
      keep_top(top, x);
    }
  }
  keep_top_xor<8>(top);
  keep_top_xor<4>(top);
  keep_top_xor<2>(top);
  keep_top_xor<1>(top);
  // lane j takes slot j
  double mykey = top[0];
#pragma unroll
  for (int i = 1; i < L; ++i) mykey = j == i ? top[i] : mykey;
  const bool slot = j < a.k;
  const int e = slot ? min(gate_key_expert(mykey), a.E - 1) : 0;
  const bool dead = mykey < -1e299;
  float s = 0.0f;
  if (slot) {
    const float l = gate_logit(a, t, e);
    if constexpr (SIG)
      s = dead ? 0.0f : 1.0f / (1.0f + hexp(-l));
    else
      s = dead || S == 0.0f ? (S == S ? 0.0f : S) : hexp(l - m) / S;
  }
  const float den = a.renorm ? seg_sum(s) + 1e-20f : 1.0f;
  float w = s / den * a.scaling;
  if (slot && tw + seg < a.T) {
    const bool on = !a.live || a.live[t];
    a.ids[t * a.k + j] = on ? e : -1;
    a.w[t * a.k + j] = on ? w : 0.0f;
  }
}

struct GateBwdArgs {
  GateArgs f;  // logits, ld, dt, T, E, k, sigmoid, renorm, scaling, ids (read), w (read)
  const float* dw;
  void* dlogits;  // (T, E) of the logits' type
};

// dlogits of the slots' weights w_j = c s_j / (sum s + 1e-20) (renorm) or c s_j: with u_j = c dw_j,
// ds_j = (u_j - (sum u s) / den) / den or u_j; sigmoid dl_e = ds s (1 - s) at the chosen experts, softmax
// dl_e = p_e (ds_e - sum_j p_j ds_j) at every expert.  A slot with an id outside [0, E) or the weight 0 (no expert was
// left for it) has no gradient, a token without any other slot zeros; an expert named by several slots gets their sum.
template <int EPL, bool SIG>
__global__ __launch_bounds__(256) void route_scores_bwd_kernel(GateBwdArgs b) {
  constexpr int W = 4;
  __shared__ float s_dp[W * 4][EPL * 16];
  const GateArgs& a = b.f;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, seg = lane >> 4;
  const int64_t tw = ((int64_t)blockIdx.x * W + wave) * 4;
  if (tw >= a.T) return;
  const bool real = tw + seg < a.T;
  const int64_t t = real ? tw + seg : a.T - 1;
  float* dp = s_dp[wave * 4 + seg];
  float lg[EPL];
  float m = -__builtin_inff(), S = 0.0f;
  if constexpr (!SIG) gate_logits(a, t, j, lg);
#pragma unroll
  for (int i = 0; i < EPL; ++i) dp[16 * i + j] = 0.0f;
  // lane j takes slot j
  int e = -1;
  float l = 0.0f, u = 0.0f;
  if (j < a.k) {
    e = a.ids[t * a.k + j];
    const float w = a.w[t * a.k + j];
    u = b.dw[t * a.k + j] * a.scaling;
    l = gate_logit(a, t, min(max(e, 0), a.E - 1));
    if (e < 0 || e >= a.E || w == 0.0f) e = -1;
  }
  if constexpr (!SIG) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) m = fmaxf(m, lg[i]);
    m = seg_max(m);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float x = hexp(lg[i] - m);
      lg[i] = lg[i] != -__builtin_inff() ? x : 0.0f;
      S += lg[i];
    }
    S = seg_sum(S);
  }
  // s, and for the sigmoid its derivative s (1 - s) = x / (1 + x)^2 with x = exp(-|l|), without the cancellation in 1 - s
  float s = 0.0f, slope = 1.0f;
  if (SIG) {
    const float x = hexp(-fabsf(l)), r = 1.0f / (1.0f + x);
    s = l >= 0.0f ? r : x * r;
    slope = x * r * r;
  } else {
    s = S == 0.0f ? 0.0f : hexp(l - m) / S;
  }
  if (e < 0) s = u = 0.0f;
  float ds = u;
  if (a.renorm) {
    const float den = seg_sum(s) + 1e-20f;
    ds = (u - seg_sum(u * s) / den) / den;
  }
  if (e < 0) ds = 0.0f;
  const float pdp = seg_sum(s * ds);
  wave_lds_sync();
  if (e >= 0) atomicAdd(&dp[e], ds * slope);
  wave_lds_sync();
  const float inv = S == 0.0f ? 0.0f : 1.0f / S;
  // (a token none of whose slots counts, as padding does, has a zero gradient whatever its logits are)
  const bool any = __ballot(e >= 0) >> (16 * seg) & 0xffff;
  float d[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    d[i] = dp[16 * i + j];
    if constexpr (!SIG) d[i] = any ? lg[i] * inv * (d[i] - pdp) : 0.0f;
  }
  if (!real) return;
  if (a.dt == HMOE_DT_F32) {
    float* p = static_cast<float*>(b.dlogits) + t * a.E;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (16 * i + j < a.E) p[16 * i + j] = d[i];
  } else {
    uint16_t* p = static_cast<uint16_t*>(b.dlogits) + t * a.E;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (16 * i + j < a.E) p[16 * i + j] = (uint16_t)(a.dt == HMOE_DT_F16 ? cvt_h2(d[i], d[i]) : cvt_bf2(d[i], d[i]));
  }
}

// calls f(EPL) for E experts
template <class F>
static void by_experts(int E, F&& f) {
  const int n = (E + 15) / 16;
  if (n <= 1) f(std::integral_constant<int, 1>());
  else if (n <= 2) f(std::integral_constant<int, 2>());
  else if (n <= 4) f(std::integral_constant<int, 4>());
  else if (n <= 8) f(std::integral_constant<int, 8>());
  else if (n <= 16) f(std::integral_constant<int, 16>());
  else f(std::integral_constant<int, 32>());
}
template <class F>
static void by_slots(int k, F&& f) {
  if (k <= 2) f(std::integral_constant<int, 2>());
  else if (k <= 4) f(std::integral_constant<int, 4>());
  else if (k <= 8) f(std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 16>());
}

static int gate_check(const void* logits, int64_t ld, int dt, int64_t T, int E, int k, int score) {
  if (T < 0 || E <= 0 || k <= 0 || (score != HMOE_SCORE_SOFTMAX && score != HMOE_SCORE_SIGMOID)) return HMOE_ERR_ARG;
  if (dt != HMOE_DT_F32 && dt != HMOE_DT_BF16 && dt != HMOE_DT_F16) return HMOE_ERR_DTYPE;
  if (E > kGateMaxE || k > kGateMaxK || k > E || T > INT32_MAX) return HMOE_ERR_SHAPE;
  if (T > 0 && (!logits || ld < E)) return HMOE_ERR_ARG;
  return HMOE_OK;
}

}  // namespace hmoe

using namespace hmoe;

extern "C" {

int hmoe_route_scores(const void* logits, int64_t ld, int dtype, const float* bias, const uint8_t* live, int64_t T,
                      int E, int k, int score, int n_group, int topk_group, int group_top, int renorm, float scaling,
                      int32_t* topk_ids, float* topk_w, hmoe_stream_t stream) {
  const int rc = gate_check(logits, ld, dtype, T, E, k, score);
  if (rc) return rc;
  if (n_group < 1 || topk_group < 1 || topk_group > n_group || E % n_group || (group_top != 1 && group_top != 2))
    return HMOE_ERR_SHAPE;
  const bool groups = topk_group < n_group;
  const int eg = E / n_group;
  if (groups && (n_group > kGateMaxGroups || eg < group_top || k > topk_group * eg)) return HMOE_ERR_SHAPE;
  if (T == 0) return HMOE_OK;
  if (!topk_ids || !topk_w) return HMOE_ERR_ARG;
  const GateArgs a = {logits, ld, dtype, bias, live, (int)T, E, k, score == HMOE_SCORE_SIGMOID, renorm, n_group,
                      topk_group, group_top, (uint32_t)(((1 << 20) + eg - 1) / eg), scaling, topk_ids, topk_w};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((T + 15) / 16));
  by_experts(E, [&](auto epl) {
    by_slots(k, [&](auto l) {
      constexpr int EPL = decltype(epl)::value, L = decltype(l)::value;
#define HMOE_GATE(G, S) hipLaunchKernelGGL((route_scores_kernel<EPL, L, G, S>), grid, dim3(256), 0, s, a)
      if (groups) {
        if (a.sigmoid) HMOE_GATE(true, true);
        else HMOE_GATE(true, false);
      } else {
        if (a.sigmoid) HMOE_GATE(false, true);
        else HMOE_GATE(false, false);
      }
#undef HMOE_GATE
    });
  });
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

int hmoe_route_scores_bwd(const float* dtopk_w, const float* topk_w, const void* logits, int64_t ld, int dtype,
                          const int32_t* topk_ids, int64_t T, int E, int k, int score, int renorm, float scaling,
                          void* dlogits, hmoe_stream_t stream) {
  const int rc = gate_check(logits, ld, dtype, T, E, k, score);
  if (rc || T == 0) return rc;
  if (!dtopk_w || !topk_w || !topk_ids || !dlogits) return HMOE_ERR_ARG;
  GateBwdArgs b = {};
  b.f.logits = logits;
  b.f.ld = ld;
  b.f.dt = dtype;
  b.f.T = (int)T;
  b.f.E = E;
  b.f.k = k;
  b.f.sigmoid = score == HMOE_SCORE_SIGMOID;
  b.f.renorm = renorm;
  b.f.scaling = scaling;
  b.f.ids = const_cast<int32_t*>(topk_ids);
  b.f.w = const_cast<float*>(topk_w);
  b.dw = dtopk_w;
  b.dlogits = dlogits;
  by_experts(E, [&](auto epl) {
    constexpr int EPL = decltype(epl)::value;
    const dim3 grid((unsigned)((T + 15) / 16));
    if (b.f.sigmoid)
      hipLaunchKernelGGL((route_scores_bwd_kernel<EPL, true>), grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), b);
    else
      hipLaunchKernelGGL((route_scores_bwd_kernel<EPL, false>), grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), b);
  });
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

}  // extern "C"
