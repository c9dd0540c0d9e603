// Routing from given logits and its backward, with their C entry points: softmax or sigmoid scores, a selection bias,
// groups, top-k, renormalised weights.
#include "hmoe_common.h"

namespace hmoe {

// Four tokens per wave: the 16 lanes of segment q take one token, lane j of it experts 16 i + j (i < EPL).
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
template <int EPL, int L, bool GROUPS>
__global__ __launch_bounds__(256) void route_scores_kernel(GateArgs a) {
  constexpr int W = 4;
  __shared__ double s_key[GROUPS ? W * 4 : 1][GROUPS ? EPL * 16 : 1];
  __shared__ double s_grp[GROUPS ? W * 4 : 1][GROUPS ? kGateMaxGroups : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, seg = lane >> 4;
  const int64_t tw = ((int64_t)blockIdx.x * W + wave) * 4;
  if (tw >= a.T) return;
  const int64_t t = tw + seg < a.T ? tw + seg : a.T - 1;  // (the lanes past T redo the last token and store nothing)
  float lg[EPL];
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = 16 * i + j;
    lg[i] = e < a.E ? gate_logit(a, t, e) : -__builtin_inff();
    m = fmaxf(m, lg[i]);
  }
  m = seg_max(m);
  // softmax: the sum of exp(l - m); a row without a finite logit has the sum 0 and scores 0
  float S = 1.0f;
  if (!a.sigmoid) {
    float p = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (16 * i + j < a.E && lg[i] != -__builtin_inff()) p += hexp(lg[i] - m);
    S = seg_sum(p);
  }
  // selection values
  double v[EPL];
  if (GROUPS || a.bias) {
    double ex[EPL], sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const bool on = lg[i] > -__builtin_inff();
      ex[i] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)lg[i])) : on ? exp((double)lg[i] - (double)m) : 0.0;
      sum += ex[i];
    }
    const double inv = a.sigmoid ? 1.0 : 1.0 / seg_sum_d(sum);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = 16 * i + j;
      const float b = a.bias && e < a.E ? a.bias[e] : 0.0f;
      const bool on = lg[i] > -__builtin_inff() && b > -__builtin_inff();
      v[i] = on ? ex[i] * inv + (double)b : -__builtin_inf();
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
    double mine[kGateMaxGroups / 16];
#pragma unroll
    for (int q = 0; q < kGateMaxGroups / 16; ++q) {
      const int g = 16 * q + j;
      mine[q] = -__builtin_inf();
      if (g < a.n_group) {
        double m1 = -__builtin_inf(), m2 = -__builtin_inf();
        for (int i = 0; i < eg; ++i) {
          const double x = key[g * eg + i];
          m2 = dmax(m2, dmin(m1, x));
          m1 = dmax(m1, x);
        }
        const double val = a.group_top == 2 ? m1 + m2 : m1;
        mine[q] = val == val ? val : -__builtin_inf();
        grp[g] = mine[q];
      }
    }
    wave_lds_sync();
    uint64_t kept = 0;
#pragma unroll
    for (int q = 0; q < kGateMaxGroups / 16; ++q) {
      if (16 * q >= a.n_group) break;
      const int g = 16 * q + j;
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
      if (!(kept >> (g & 63) & 1)) v[i] = -__builtin_inf();
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
      x[i] = ii < EPL && e < a.E ? gate_key(v[ii < EPL ? ii : 0], e) : kGateNone;
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
    if (a.sigmoid)
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
// left for it) has no gradient; an expert named by several slots gets their sum.
template <int EPL>
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
  if (!a.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = 16 * i + j;
      lg[i] = e < a.E ? gate_logit(a, t, e) : -__builtin_inff();
      m = fmaxf(m, lg[i]);
    }
    m = seg_max(m);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      lg[i] = lg[i] != -__builtin_inff() ? hexp(lg[i] - m) : 0.0f;
      S += lg[i];
    }
    S = seg_sum(S);
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) dp[16 * i + j] = 0.0f;
  int e = -1;
  float s = 0.0f, u = 0.0f;
  if (j < a.k) {
    e = a.ids[t * a.k + j];
    if (e < 0 || e >= a.E || a.w[t * a.k + j] == 0.0f) e = -1;
    if (e >= 0) {
      const float l = gate_logit(a, t, e);
      s = a.sigmoid ? 1.0f / (1.0f + hexp(-l)) : S == 0.0f ? 0.0f : hexp(l - m) / S;
      u = b.dw[t * a.k + j] * a.scaling;
    }
  }
  float ds = u;
  if (a.renorm) {
    const float den = seg_sum(s) + 1e-20f;
    ds = (u - seg_sum(u * s) / den) / den;
  }
  if (e < 0) ds = 0.0f;
  const float pdp = seg_sum(s * ds);
  wave_lds_sync();
  if (e >= 0) atomicAdd(&dp[e], a.sigmoid ? ds * s * (1.0f - s) : ds);
  wave_lds_sync();
  const float inv = S == 0.0f ? 0.0f : 1.0f / S;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int o = 16 * i + j;
    if (o >= a.E || !real) continue;
    const float d = a.sigmoid ? dp[o] : lg[i] * inv * (dp[o] - pdp);
    const int64_t at = t * a.E + o;
    if (a.dt == HMOE_DT_F32)
      static_cast<float*>(b.dlogits)[at] = d;
    else
      static_cast<uint16_t*>(b.dlogits)[at] = (uint16_t)(a.dt == HMOE_DT_F16 ? cvt_h2(d, d) : cvt_bf2(d, d));
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
  else if (n <= 12) f(std::integral_constant<int, 12>());
  else if (n <= 16) f(std::integral_constant<int, 16>());
  else if (n <= 24) f(std::integral_constant<int, 24>());
  else f(std::integral_constant<int, 32>());
}
template <class F>
static void by_slots(int k, F&& f) {
  if (k <= 1) f(std::integral_constant<int, 1>());
  else if (k <= 2) f(std::integral_constant<int, 2>());
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
      if (groups)
        hipLaunchKernelGGL((route_scores_kernel<EPL, L, true>), grid, dim3(256), 0, s, a);
      else
        hipLaunchKernelGGL((route_scores_kernel<EPL, L, false>), grid, dim3(256), 0, s, a);
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
    hipLaunchKernelGGL((route_scores_bwd_kernel<decltype(epl)::value>), dim3((unsigned)((T + 15) / 16)), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), b);
  });
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

}  // extern "C"
