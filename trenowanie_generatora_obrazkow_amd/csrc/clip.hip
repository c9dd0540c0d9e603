// The global norm of a list of gradients and their clipping, with their C entry points.  Both read every gradient once
// and are bound by that.
#include "hmoe_common.h"

#include <algorithm>
#include <cmath>
#include <cstdlib>

namespace hmoe {

// The tensors of a launch travel in its arguments (no device table to copy, and a captured launch keeps its list).
constexpr int kClipTensors = 128;   // per launch: 3.8 KB of the 4 KB of arguments
constexpr int kClipChunk = 16384;   // elements a workgroup takes at a time
constexpr int kClipAhead = 8;       // vectors of eight elements a thread of the scaling kernel has on their way
constexpr int kClipBlocks = 2048;   // workgroups per launch: eight per CU

struct ClipList {
  const void* p[kClipTensors];
  void* o[kClipTensors];
  int64_t n[kClipTensors];
  uint32_t first[kClipTensors + 1];  // first chunk of each tensor; first[count] = all chunks
  uint8_t dt[kClipTensors];          // type of p | type of o << 4
  int count;
};
static_assert(sizeof(ClipList) + 64 <= 4096, "kernel arguments");

__device__ __forceinline__ int clip_tensor(const ClipList& l, uint32_t chunk) {
  int lo = 0, hi = l.count;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (l.first[m] <= chunk)
      lo = m;
    else
      hi = m;
  }
  return lo;
}

// eight elements from an address aligned to an element only (views of a bucket)
struct __attribute__((packed, aligned(2))) Raw16 { uint32_t w[4]; };
struct __attribute__((packed, aligned(4))) Raw32 { float f[4]; };

template <int DT>
__device__ __forceinline__ void clip_load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (DT == HMOE_DT_F32) {
    const Raw32* q = reinterpret_cast<const Raw32*>(static_cast<const float*>(p) + i);
    const Raw32 a = q[0], b = q[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a.f[e];
      v[4 + e] = b.f[e];
    }
  } else {
    using X = Elt<DT == HMOE_DT_F16>;
    const Raw16 u = *reinterpret_cast<const Raw16*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = X::lo(u.w[e]);
      v[2 * e + 1] = X::hi(u.w[e]);
    }
  }
}
template <int DT>
__device__ __forceinline__ float clip_load1(const void* p, int64_t i) {
  if constexpr (DT == HMOE_DT_F32) return static_cast<const float*>(p)[i];
  else return Elt<DT == HMOE_DT_F16>::one(static_cast<const uint16_t*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void clip_store8(void* p, int64_t i, const float (&v)[8]) {
  if constexpr (DT == HMOE_DT_F32) {
    Raw32* q = reinterpret_cast<Raw32*>(static_cast<float*>(p) + i);
    q[0] = Raw32{{v[0], v[1], v[2], v[3]}};
    q[1] = Raw32{{v[4], v[5], v[6], v[7]}};
  } else {
    using X = Elt<DT == HMOE_DT_F16>;
    *reinterpret_cast<Raw16*>(static_cast<uint16_t*>(p) + i) =
        Raw16{{X::pack2(v[0], v[1]), X::pack2(v[2], v[3]), X::pack2(v[4], v[5]), X::pack2(v[6], v[7])}};
  }
}
template <int DT>
__device__ __forceinline__ void clip_store1(void* p, int64_t i, float v) {
  if constexpr (DT == HMOE_DT_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)Elt<DT == HMOE_DT_F16>::pack2(v, v);
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s, 64);
  return v;
}
// sum over the 256 threads of a block, for every thread
__device__ __forceinline__ double block_sum_d(double v, double* lds) {
  v = wave_sum_d(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <class F>
__device__ __forceinline__ void clip_by_type(int dt, F&& f) {
  if (dt == HMOE_DT_F32) f(std::integral_constant<int, HMOE_DT_F32>());
  else if (dt == HMOE_DT_F16) f(std::integral_constant<int, HMOE_DT_F16>());
  else f(std::integral_constant<int, HMOE_DT_BF16>());
}

// part[block] = the sum of the squares of the block's chunks, in fp64: fp32 squares would overflow from 1.8e19 on and
// vanish below 2e-23, and the fp64 fma keeps up with the loads: 302M bf16 elements in 139 us (median of 20 launches, 4.3 TB/s;
// the best 118, 5.1 TB/s, the rate of a large copy).  The chunks, and so the order of the sum, go by the list and by which of
// its tensors follow each other in memory.
__global__ __launch_bounds__(256) void clip_norm_kernel(ClipList l, double* part) {
  __shared__ double lds[4];
  double acc = 0.0;
  const uint32_t chunks = l.first[l.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int ti = clip_tensor(l, c);
    const int64_t i0 = (int64_t)(c - l.first[ti]) * kClipChunk, i1 = min(l.n[ti], i0 + kClipChunk);
    const void* p = l.p[ti];
    clip_by_type(l.dt[ti] & 15, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      int64_t i = i0 + threadIdx.x * 8;
      for (; i + 8 <= i1; i += 256 * 8) {
        float v[8];
        clip_load8<DT>(p, i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc = __builtin_fma((double)v[e], (double)v[e], acc);
      }
      for (; i < i1; ++i) {  // the thread that holds the chunk's last, partial vector
        const double v = clip_load1<DT>(p, i);
        acc = __builtin_fma(v, v, acc);
      }
    });
  }
  acc = block_sum_d(acc, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

__global__ __launch_bounds__(256) void clip_total_kernel(const double* part, int n, double* sq) {
  __shared__ double lds[4];
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) acc += part[i];
  acc = block_sum_d(acc, lds);
  if (threadIdx.x == 0) *sq = acc;
}

__device__ __forceinline__ float clip_coef(double norm, double max_norm) {
  const double c = max_norm / (norm + 1e-6);
  return c < 1.0 ? (float)c : norm == norm ? 1.0f : __builtin_nanf("");
}

// out = grad * factor, from the back of the list: what the norm read last may still lie in the 256 MB cache (98.6M fp32
// elements 137.5 us against 142).  Eight vectors a thread on their way: 302M bf16 elements into fp32 338 us (5.3 TB/s) against
// 361 with four and 369 with one.
__global__ __launch_bounds__(256) void clip_scale_kernel(ClipList l, const double* sq, double max_norm, float* norm_out) {
  const double norm = sqrt(*sq);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const float coef = clip_coef(norm, max_norm);
  const uint32_t chunks = l.first[l.count];
  for (uint32_t cc = blockIdx.x; cc < chunks; cc += gridDim.x) {
    const uint32_t c = chunks - 1 - cc;
    const int ti = clip_tensor(l, c);
    const void* p = l.p[ti];
    void* o = l.o[ti];
    if (p == o && coef == 1.0f) continue;  // nothing to change in place (one address: one type, clip_overlap)
    const int64_t i0 = (int64_t)(c - l.first[ti]) * kClipChunk, i1 = min(l.n[ti], i0 + kClipChunk);
    clip_by_type(l.dt[ti] & 15, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      auto walk = [&](auto odt) {
        constexpr int OT = decltype(odt)::value;
        int64_t i = i0 + threadIdx.x * 8;
        for (; i + (kClipAhead - 1) * 256 * 8 + 8 <= i1; i += kClipAhead * 256 * 8) {
          float v[kClipAhead][8];
#pragma unroll
          for (int k = 0; k < kClipAhead; ++k) clip_load8<DT>(p, i + k * 256 * 8, v[k]);
#pragma unroll
          for (int k = 0; k < kClipAhead; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] *= coef;
            clip_store8<OT>(o, i + k * 256 * 8, v[k]);
          }
        }
        for (; i + 8 <= i1; i += 256 * 8) {
          float v[8];
          clip_load8<DT>(p, i, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= coef;
          clip_store8<OT>(o, i, v);
        }
        for (; i < i1; ++i) clip_store1<OT>(o, i, clip_load1<DT>(p, i) * coef);
      };
      if (l.dt[ti] >> 4 == HMOE_DT_F32)
        walk(std::integral_constant<int, HMOE_DT_F32>());
      else
        walk(dt);
    });
  }
}

// Fills a list from the tensors at i on (empty ones are left out) and moves i behind them.  Tensors that follow each other in
// memory, as the views of a gradient bucket do, and whose outputs do so too are walked as one: fewer entries and launches.
static int clip_list(const void* const* grads, void* const* out, const int64_t* numel, const int* dtypes,
                     const int* out_dtypes, int n, int& i, ClipList& l) {
  l.count = 0;
  uint64_t chunks = 0;
  for (; i < n; ++i) {
    const int64_t m = numel[i];
    const int dt = dtypes[i];
    if (m < 0) return HMOE_ERR_ARG;
    if (dt != HMOE_DT_F32 && dt != HMOE_DT_F16 && dt != HMOE_DT_BF16) return HMOE_ERR_DTYPE;
    const int ot = out_dtypes ? out_dtypes[i] : dt;
    if (ot != dt && ot != HMOE_DT_F32) return HMOE_ERR_DTYPE;
    if (m == 0) continue;
    const uintptr_t al = (dt == HMOE_DT_F32 ? 3 : 1), ao = (ot == HMOE_DT_F32 ? 3 : 1);
    void* o = out ? out[i] : nullptr;
    if (!grads[i] || (reinterpret_cast<uintptr_t>(grads[i]) & al) || (out && !o) || (reinterpret_cast<uintptr_t>(o) & ao))
      return HMOE_ERR_ARG;
    const int64_t sz = dt == HMOE_DT_F32 ? 4 : 2, so = ot == HMOE_DT_F32 ? 4 : 2;
    const uint8_t kind = (uint8_t)(dt | ot << 4);
    if (m > INT64_MAX / 8) return HMOE_ERR_SHAPE;
    if (l.count) {
      const int b = l.count - 1;
      if (kind == l.dt[b] && static_cast<const char*>(l.p[b]) + l.n[b] * sz == grads[i] &&
          (!out || static_cast<char*>(l.o[b]) + l.n[b] * so == o)) {
        l.n[b] += m;
        continue;
      }
      if (l.count == kClipTensors) break;
    }
    l.p[l.count] = grads[i];
    l.o[l.count] = o;
    l.n[l.count] = m;
    l.dt[l.count++] = kind;
  }
  for (int b = 0; b < l.count; ++b) {
    l.first[b] = (uint32_t)chunks;
    chunks += ((uint64_t)l.n[b] + kClipChunk - 1) / kClipChunk;
    if (chunks > 0x7fffffffu) return HMOE_ERR_SHAPE;
  }
  l.first[l.count] = (uint32_t)chunks;
  return HMOE_OK;
}

// Whether a tensor that is written lies over any other of the call (its own gradient at the same address and of the same type
// is in place).  Workgroups walk the chunks in any order, so such a call would race.  Listed in the order of their addresses,
// as views of a bucket are, the tensors need no sorting; 300 of them take 1 us then.  -1: no host memory to look.
struct ClipSpan {
  uintptr_t first, end;
  bool written;
};
static int clip_overlap(const void* const* grads, void* const* out, const int64_t* numel, const int* dtypes,
                        const int* out_dtypes, int n) {
  ClipSpan few[1024];
  ClipSpan* s = n <= 512 ? few : static_cast<ClipSpan*>(std::malloc(2 * (size_t)n * sizeof(ClipSpan)));
  if (!s) return -1;
  int m = 0;
  bool sorted = true;
  auto put = [&](const void* p, int64_t bytes, bool written) {
    const uintptr_t first = reinterpret_cast<uintptr_t>(p);
    sorted = sorted && (m == 0 || s[m - 1].first <= first);
    s[m++] = {first, first + (uintptr_t)bytes, written};
  };
  for (int i = 0; i < n; ++i) {
    if (numel[i] == 0) continue;
    const bool own = grads[i] == out[i] && dtypes[i] == out_dtypes[i];
    if (!own) put(grads[i], numel[i] * (dtypes[i] == HMOE_DT_F32 ? 4 : 2), false);
    put(out[i], numel[i] * (out_dtypes[i] == HMOE_DT_F32 ? 4 : 2), true);
  }
  if (!sorted) std::sort(s, s + m, [](const ClipSpan& a, const ClipSpan& b) { return a.first < b.first; });
  uintptr_t any = 0, written = 0;  // ends of what came before
  int over = 0;
  for (int i = 0; i < m && !over; ++i) {
    over = s[i].first < (s[i].written ? any : written);
    any = std::max(any, s[i].end);
    if (s[i].written) written = std::max(written, s[i].end);
  }
  if (s != few) std::free(s);
  return over;
}

static unsigned clip_grid(const ClipList& l) {
  const uint32_t c = l.first[l.count];
  return c < kClipBlocks ? c : kClipBlocks;
}

static int clip_check(const void* const* grads, const int64_t* numel, const int* dtypes, int n) {
  if (n < 0 || (n > 0 && (!grads || !numel || !dtypes))) return HMOE_ERR_ARG;
  return HMOE_OK;
}

}  // namespace hmoe

using namespace hmoe;

extern "C" {

size_t hmoe_grad_sq_norm_workspace_size(int n) {
  return n < 0 ? 0 : (size_t)((n + kClipTensors - 1) / kClipTensors + 1) * kClipBlocks * sizeof(double);
}

int hmoe_grad_sq_norm(const void* const* grads, const int64_t* numel, const int* dtypes, int n, double* sq_norm,
                      void* workspace, size_t workspace_bytes, hmoe_stream_t stream) {
  int rc = clip_check(grads, numel, dtypes, n);
  if (rc) return rc;
  if (!sq_norm || (reinterpret_cast<uintptr_t>(sq_norm) & 7)) return HMOE_ERR_ARG;
  if (!workspace || workspace_bytes < hmoe_grad_sq_norm_workspace_size(n)) return HMOE_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return HMOE_ERR_ARG;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  ClipList l;
  for (int i = 0; i < n;) {  // the whole list is checked before the first launch
    rc = clip_list(grads, nullptr, numel, dtypes, nullptr, n, i, l);
    if (rc) return rc;
  }
  int parts = 0;
  for (int i = 0; i < n;) {
    clip_list(grads, nullptr, numel, dtypes, nullptr, n, i, l);
    if (l.count == 0) continue;
    const unsigned g = clip_grid(l);
    hipLaunchKernelGGL(clip_norm_kernel, dim3(g), dim3(256), 0, s, l, part + parts);
    HMOE_CHECK_LAUNCH();
    parts += (int)g;
  }
  hipLaunchKernelGGL(clip_total_kernel, dim3(1), dim3(256), 0, s, part, parts, sq_norm);
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

int hmoe_grad_clip_f64(const void* const* grads, void* const* out, const int64_t* numel, const int* dtypes,
                       const int* out_dtypes, int n, const double* sq_norm, double max_norm, float* norm,
                       hmoe_stream_t stream) {
  int rc = clip_check(grads, numel, dtypes, n);
  if (rc) return rc;
  if (!sq_norm || (n > 0 && (!out || !out_dtypes)) || !(max_norm >= 0.0)) return HMOE_ERR_ARG;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  ClipList l;
  for (int i = 0; i < n;) {
    rc = clip_list(grads, out, numel, dtypes, out_dtypes, n, i, l);
    if (rc) return rc;
  }
  if (n > 0) {
    const int over = clip_overlap(grads, out, numel, dtypes, out_dtypes, n);
    if (over) return over < 0 ? HMOE_ERR_WORKSPACE : HMOE_ERR_OVERLAP;
  }
  bool first = true;
  int i = 0;
  do {
    clip_list(grads, out, numel, dtypes, out_dtypes, n, i, l);
    if (l.count == 0 && !first) continue;
    // (an empty list still writes the norm)
    hipLaunchKernelGGL(clip_scale_kernel, dim3(l.count ? clip_grid(l) : 1), dim3(256), 0, s, l, sq_norm, max_norm,
                       first ? norm : nullptr);
    HMOE_CHECK_LAUNCH();
    first = false;
  } while (i < n);
  return HMOE_OK;
}

int hmoe_grad_clip(const void* const* grads, void* const* out, const int64_t* numel, const int* dtypes,
                   const int* out_dtypes, int n, const double* sq_norm, float max_norm, float* norm,
                   hmoe_stream_t stream) {
  return hmoe_grad_clip_f64(grads, out, numel, dtypes, out_dtypes, n, sq_norm, (double)max_norm, norm, stream);
}

}  // extern "C"
