// Softmax selection for up to 16 experts, one 16-lane segment per token: shared by the router's kernels (route.hip) and the
// layer for a few tokens (few.hip), which have to choose alike to the last bit.
#pragma once
#include <type_traits>

#include "hmoe_common.h"

namespace hmoe {

// wave-wide argmax of (value, index): larger value wins, equal values go to the lower index; an index of 0x7fffffff
// marks an empty candidate.  The winner is unique, so any exchange pattern gives every lane the same result.
__device__ __forceinline__ void argmax_take(float& bv, int& be, float ov, int oe) {
  const bool take = oe != 0x7fffffff && (be == 0x7fffffff || ov > bv || (ov == bv && oe < be));
  if (take) {
    bv = ov;
    be = oe;
  }
}

// one arg-max exchange step over lanes l ^ S inside 16-lane rows, carrying a payload (argmax_take's rule)
template <int S>
__device__ __forceinline__ void seg_argmax_step(float& bv, int& be, float& bp) {
  const float ov = lane_xor<S>(bv), op = lane_xor<S>(bp);
  const int oe = lane_xor_i<S>(be);
  if (oe != 0x7fffffff && (be == 0x7fffffff || ov > bv || (ov == bv && oe < be))) {
    bv = ov;
    be = oe;
    bp = op;
  }
}

// The softmax selection of route_select for E <= 16, NI groups of four tokens per wave: lane l holds, for each i < NI,
// the logit of expert l % 16 of token t0 + i + NI (l / 16) (ignored past E).  Segment (16-lane) butterflies give the
// 64-lane ones' results bit for bit (those only add exact zeros and compare with -inf from the lanes past E; the
// arg-max with ties to the lower index does not depend on the reduction tree), so ids, weights and logits equal
// route_select's.  The NI selections advance together (independent exchange chains side by side), the winner's
// probability numerator is carried through the arg-max exchanges, and lane j of a segment keeps selection j.
template <int NI>
__device__ __forceinline__ void route_select16(const float (&lg)[NI], int t0, int lane, int T, int E, int k,
                                               int renorm, float scaling, float* __restrict__ logits,
                                               int32_t* __restrict__ ids, float* __restrict__ wout) {
#pragma clang fp contract(off)
  const int e = lane & 15;
  const bool valid = e < E;
  float m[NI], num[NI], S[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) m[i] = valid ? lg[i] : -__builtin_inff();
  auto max_step = [&](auto sc) {
    constexpr int SS = decltype(sc)::value;
#pragma unroll
    for (int i = 0; i < NI; ++i) m[i] = fmaxf(m[i], lane_xor<SS>(m[i]));
  };
  max_step(std::integral_constant<int, 8>());
  max_step(std::integral_constant<int, 4>());
  max_step(std::integral_constant<int, 2>());
  max_step(std::integral_constant<int, 1>());
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    num[i] = valid ? hexp(__fsub_rn(lg[i], m[i])) : 0.0f;
    S[i] = num[i];
  }
  auto sum_step = [&](auto sc) {
    constexpr int SS = decltype(sc)::value;
#pragma unroll
    for (int i = 0; i < NI; ++i) S[i] = __fadd_rn(S[i], lane_xor<SS>(S[i]));
  };
  sum_step(std::integral_constant<int, 8>());
  sum_step(std::integral_constant<int, 4>());
  sum_step(std::integral_constant<int, 2>());
  sum_step(std::integral_constant<int, 1>());
  int64_t t[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    t[i] = (int64_t)t0 + i + NI * (lane >> 4);
    if (logits && t[i] < T && valid) logits[t[i] * E + e] = lg[i];
  }
  bool taken[NI];
  float ssum[NI], my_p[NI];
  int my_e[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    taken[i] = false;
    ssum[i] = my_p[i] = 0.0f;
    my_e[i] = 0;
  }
  for (int jj = 0; jj < k; ++jj) {
    float bv[NI], bp[NI];
    int be[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const bool cand = valid && !taken[i];
      bv[i] = cand ? lg[i] : 0.0f;
      be[i] = cand ? e : 0x7fffffff;
      bp[i] = num[i];
    }
    auto arg_step = [&](auto sc) {
      constexpr int SS = decltype(sc)::value;
#pragma unroll
      for (int i = 0; i < NI; ++i) seg_argmax_step<SS>(bv[i], be[i], bp[i]);
    };
    arg_step(std::integral_constant<int, 8>());
    arg_step(std::integral_constant<int, 4>());
    arg_step(std::integral_constant<int, 2>());
    arg_step(std::integral_constant<int, 1>());
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (be[i] == e) taken[i] = true;
      const float p = __fdiv_rn(bp[i], S[i]);
      ssum[i] = jj == 0 ? p : __fadd_rn(ssum[i], p);
      if (e == jj) {
        my_p[i] = p;
        my_e[i] = be[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if (t[i] < T && e < k) {
      const float wj = renorm ? __fmul_rn(__fdiv_rn(my_p[i], __fadd_rn(ssum[i], 1e-20f)), scaling)
                              : __fmul_rn(my_p[i], scaling);
      ids[t[i] * k + e] = my_e[i];
      wout[t[i] * k + e] = wj;
    }
  }
}

}  // namespace hmoe
