// SwiGLU whose backward reads an 8-bit checkpoint: the forward keeps g and u as e4m3 with a power-of-two scale per 32 columns
// (f8_common.h), half the bytes of [g | u] in 16 bits and none of the activation; the backward forms the gradients and the
// activation again from what was kept.
//
//   forward   act = silu(g) u;  keep Q(g), Q(u)
//   backward  with g, u the kept values and s = sigmoid(g):  da = w dh,  du = da g s,  dg = da u (s + g s (1 - s)),
//             act' = g s u,  dw = sum over the row of dh act'
//
// One pass over the data each, memory-bound (everything in fp32 between one read and one rounding): the forward moves
// 8.06 M h bytes, the backward 12.06 M h.  Blocks of 32: a scale costs 1/32 byte a value, and a block is four lanes' eight
// values, so its largest one takes two exchanges.  32768 rows of h 4096 in bf16: 186 us forward, 5.8 TB/s, 236 us backward, 6.9
// (a copy of 2 GB 5.0).  Non-temporal stores took 181 and 230 us there, but 10.4 instead of 9.3 us for 4096 rows of h 1024.
#include <algorithm>

#include "f8_common.h"

namespace hmoe {

constexpr int kPackBlock = 32;

template <bool F16>
__device__ __forceinline__ void unpack8(uint4 w, float* v) {
  using X = Elt<F16>;
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = X::lo(u[i]);
    v[2 * i + 1] = X::hi(u[i]);
  }
}
template <bool F16>
__device__ __forceinline__ uint4 pack8(const float* v) {
  using X = Elt<F16>;
  return make_uint4(X::pack2(v[0], v[1]), X::pack2(v[2], v[3]), X::pack2(v[4], v[5]), X::pack2(v[6], v[7]));
}

// eight values of a block of 32 (four lanes) -> e4m3, and the scale's byte; lanes past the row hold zeros
__device__ __forceinline__ uint2 pack_block(const float* v, uint8_t& sb) {
  float m = 0.0f;
#pragma unroll
  for (int t = 0; t < 8; ++t) m = fmaxf(m, f8_abs(v[t]));
  m = bfly_max<2>(bfly_max<1>(m));
  const int e = f8_exp(m);
  const float inv = f8_inv(e);
  sb = (uint8_t)(e + 127);
  return make_uint2(f8_pack4(v[0], v[1], v[2], v[3], inv), f8_pack4(v[4], v[5], v[6], v[7], inv));
}
__device__ __forceinline__ void unpack_block(uint2 w, uint8_t sb, float* v) {
  f8_unpack2<0>(w.x, v[0], v[1]);
  f8_unpack2<1>(w.x, v[2], v[3]);
  f8_unpack2<0>(w.y, v[4], v[5]);
  f8_unpack2<1>(w.y, v[6], v[7]);
  const float s = f8_pow((int)sb - 127);
#pragma unroll
  for (int t = 0; t < 8; ++t) v[t] *= s;
}

// TPR threads a row (a multiple of 4; a power of two), 256 / TPR rows a workgroup.
template <bool F16, int TPR>
__global__ __launch_bounds__(256) void swiglu_pack_kernel(const uint16_t* __restrict__ gu, int64_t ldgu, int64_t M, int h,
                                                          int nb, uint16_t* __restrict__ act, uint8_t* __restrict__ q,
                                                          uint8_t* __restrict__ s) {
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (row >= M) return;
  const uint16_t* pg = gu + row * ldgu;
  for (int c = threadIdx.x % TPR; c < 4 * nb; c += TPR) {  // (whole blocks of four lanes: the exchanges stay inside them)
    const int col = c * 8;
    const bool in = col < h;
    float g[8], u[8], a[8];
    if (in) {
      unpack8<F16>(*reinterpret_cast<const uint4*>(pg + col), g);
      unpack8<F16>(*reinterpret_cast<const uint4*>(pg + h + col), u);
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t) g[t] = u[t] = 0.0f;
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) a[t] = silu_f(g[t]) * u[t];
    uint8_t sg, su;
    const uint2 qg = pack_block(g, sg), qu = pack_block(u, su);
    if (in) {
      *reinterpret_cast<uint4*>(act + row * h + col) = pack8<F16>(a);
      *reinterpret_cast<uint2*>(q + row * 2 * h + col) = qg;
      *reinterpret_cast<uint2*>(q + row * 2 * h + h + col) = qu;
    }
    if ((c & 3) == 0) {
      s[row * 2 * nb + c / 4] = sg;
      s[row * 2 * nb + nb + c / 4] = su;
    }
  }
}

template <bool F16, int TPR>
__global__ __launch_bounds__(256) void swiglu_pack_bwd_kernel(const uint16_t* __restrict__ dh, const uint8_t* __restrict__ q,
                                                              const uint8_t* __restrict__ s, const void* __restrict__ w,
                                                              int w_dt, int64_t M, int h, int nb, uint16_t* __restrict__ dgu,
                                                              uint16_t* __restrict__ act, const int32_t* __restrict__ order,
                                                              float* __restrict__ dw) {
  __shared__ float part[4];
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  float sum = 0.0f;
  if (row < M) {
    float wr = 1.0f;
    if (w) {
      if (w_dt == HMOE_DT_F32) wr = static_cast<const float*>(w)[row];
      else wr = w_dt == HMOE_DT_BF16 ? Elt<false>::one(static_cast<const uint16_t*>(w)[row])
                                     : Elt<true>::one(static_cast<const uint16_t*>(w)[row]);
    }
    for (int c = threadIdx.x % TPR; c * 8 < h; c += TPR) {
      const int col = c * 8;
      float d[8], g[8], u[8], dg[8], du[8], a[8];
      unpack8<F16>(*reinterpret_cast<const uint4*>(dh + row * h + col), d);
      unpack_block(*reinterpret_cast<const uint2*>(q + row * 2 * h + col), s[row * 2 * nb + c / 4], g);
      unpack_block(*reinterpret_cast<const uint2*>(q + row * 2 * h + h + col), s[row * 2 * nb + nb + c / 4], u);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const float sg = sigmoid_f(g[t]), l = g[t] * sg, da = d[t] * wr;
        du[t] = da * l;
        dg[t] = (da * u[t]) * __builtin_fmaf(l, 1.0f - sg, sg);
        a[t] = l * u[t];
        sum = __builtin_fmaf(d[t], a[t], sum);
      }
      *reinterpret_cast<uint4*>(dgu + row * 2 * h + col) = pack8<F16>(dg);
      *reinterpret_cast<uint4*>(dgu + row * 2 * h + h + col) = pack8<F16>(du);
      if (act) *reinterpret_cast<uint4*>(act + row * h + col) = pack8<F16>(a);
    }
  }
  if (!dw) return;
  // the row's sum, always in the same order: over the lanes of a wave, then over the waves
  sum = bfly_add<4>(bfly_add<2>(bfly_add<1>(sum)));
  if constexpr (TPR >= 16) sum = bfly_add<8>(sum);
  if constexpr (TPR >= 32) sum = bfly_add<16>(sum);
  if constexpr (TPR >= 64) sum = bfly_add<32>(sum);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    constexpr int W = TPR / 64;
    const int w0 = threadIdx.x / TPR * W;
    sum = part[w0];
#pragma unroll
    for (int i = 1; i < W; ++i) sum += part[w0 + i];
  }
  if (threadIdx.x % TPR == 0 && row < M) {
    const int64_t f = order ? (int64_t)order[row] : row;
    if (f >= 0) dw[f] = sum;  // (a row past those that a dispatch counted has order -1)
  }
}

// threads per row: the least power of two from 8 on that takes a row in one step, at most a workgroup
template <class F>
static void pick_tpr(int lanes, F&& f) {
  if (lanes <= 8) f(std::integral_constant<int, 8>{});
  else if (lanes <= 16) f(std::integral_constant<int, 16>{});
  else if (lanes <= 32) f(std::integral_constant<int, 32>{});
  else if (lanes <= 64) f(std::integral_constant<int, 64>{});
  else if (lanes <= 128) f(std::integral_constant<int, 128>{});
  else f(std::integral_constant<int, 256>{});
}

static int pack_check(int64_t M, int64_t h, int dtype) {
  if (M < 0 || h <= 0) return HMOE_ERR_ARG;
  if (dtype != HMOE_DT_BF16 && dtype != HMOE_DT_F16) return HMOE_ERR_DTYPE;
  if (h % 8 || h > (1 << 28) || M > INT32_MAX) return HMOE_ERR_SHAPE;
  return HMOE_OK;
}
// a launch has fewer than 2^32 threads
static bool pack_fits(int64_t M, int nb) {
  bool ok = false;
  pick_tpr(4 * nb, [&](auto tpr) { ok = (M + 256 / decltype(tpr)::value - 1) / (256 / decltype(tpr)::value) < (1 << 24); });
  return ok;
}
static bool mis(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

}  // namespace hmoe

using namespace hmoe;

extern "C" {

int hmoe_swiglu_pack(const void* gu, int64_t ldgu, int64_t M, int64_t h, void* act, void* q, uint8_t* s, int dtype,
                     hmoe_stream_t stream) {
  const int rc = pack_check(M, h, dtype);
  if (rc || M == 0) return rc;
  if (!gu || !act || !q || !s || ldgu < 2 * h || ldgu % 8 || mis(gu, 16) || mis(act, 16) || mis(q, 8)) return HMOE_ERR_ARG;
  const int nb = (int)((h + kPackBlock - 1) / kPackBlock);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (!pack_fits(M, nb)) return HMOE_ERR_SHAPE;
  pick_tpr(4 * nb, [&](auto tpr) {
    constexpr int TPR = decltype(tpr)::value;
    const dim3 grid((unsigned)((M + 256 / TPR - 1) / (256 / TPR)));
    if (dtype == HMOE_DT_BF16)
      hipLaunchKernelGGL((swiglu_pack_kernel<false, TPR>), grid, dim3(256), 0, st, static_cast<const uint16_t*>(gu), ldgu, M,
                         (int)h, nb, static_cast<uint16_t*>(act), static_cast<uint8_t*>(q), s);
    else
      hipLaunchKernelGGL((swiglu_pack_kernel<true, TPR>), grid, dim3(256), 0, st, static_cast<const uint16_t*>(gu), ldgu, M,
                         (int)h, nb, static_cast<uint16_t*>(act), static_cast<uint8_t*>(q), s);
  });
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

int hmoe_swiglu_pack_bwd(const void* dh, const void* q, const uint8_t* s, const void* w, int w_dtype, int64_t M, int64_t h,
                         void* dgu, void* act, const int32_t* order, float* dw, int dtype, hmoe_stream_t stream) {
  const int rc = pack_check(M, h, dtype);
  if (rc) return rc;
  if (w && w_dtype != HMOE_DT_F32 && w_dtype != HMOE_DT_BF16 && w_dtype != HMOE_DT_F16) return HMOE_ERR_DTYPE;
  if (M == 0) return HMOE_OK;
  if (!dh || !q || !s || !dgu || mis(dh, 16) || mis(q, 8) || mis(dgu, 16) || mis(act, 16)) return HMOE_ERR_ARG;
  const int nb = (int)((h + kPackBlock - 1) / kPackBlock);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (!pack_fits(M, nb)) return HMOE_ERR_SHAPE;
  pick_tpr(4 * nb, [&](auto tpr) {
    constexpr int TPR = decltype(tpr)::value;
    const dim3 grid((unsigned)((M + 256 / TPR - 1) / (256 / TPR)));
    if (dtype == HMOE_DT_BF16)
      hipLaunchKernelGGL((swiglu_pack_bwd_kernel<false, TPR>), grid, dim3(256), 0, st, static_cast<const uint16_t*>(dh),
                         static_cast<const uint8_t*>(q), s, w, w_dtype, M, (int)h, nb, static_cast<uint16_t*>(dgu),
                         static_cast<uint16_t*>(act), order, dw);
    else
      hipLaunchKernelGGL((swiglu_pack_bwd_kernel<true, TPR>), grid, dim3(256), 0, st, static_cast<const uint16_t*>(dh),
                         static_cast<const uint8_t*>(q), s, w, w_dtype, M, (int)h, nb, static_cast<uint16_t*>(dgu),
                         static_cast<uint16_t*>(act), order, dw);
  });
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

}  // extern "C"
