// The norms around the routed block, with their C entry points: the RMS norm before it with weight and per-sample
// scale / shift, and the sum over the routed slots, RMS norm, gate and scaled residual after it; both with backward.
// A row is T x d work of a few operations per element, so every kernel here is bound by the rows it reads and writes.
#include "hmoe_common.h"

namespace hmoe {

// ---------------------------------------------------------------------------------------------------------------
// Eight consecutive elements as fp32, of a type known at compile time (rows) or at run time (parameters: a branch that
// is uniform over the grid).
// ---------------------------------------------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t off, float (&v)[8]) {
  if constexpr (DT == HMOE_DT_F32) {
    const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + off);
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else {
    using X = Elt<DT == HMOE_DT_F16>;
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + off);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = X::lo(w[i]);
      v[2 * i + 1] = X::hi(w[i]);
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t off, const float (&v)[8]) {
  if constexpr (DT == HMOE_DT_F32) {
    f32x4* q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + off);
    q[0] = f32x4{v[0], v[1], v[2], v[3]};
    q[1] = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    using X = Elt<DT == HMOE_DT_F16>;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + off) =
        make_uint4(X::pack2(v[0], v[1]), X::pack2(v[2], v[3]), X::pack2(v[4], v[5]), X::pack2(v[6], v[7]));
  }
}

__device__ __forceinline__ void load8_rt(const void* p, int dt, int64_t off, float (&v)[8]) {
  if (dt == HMOE_DT_F32)
    load8<HMOE_DT_F32>(p, off, v);
  else if (dt == HMOE_DT_F16)
    load8<HMOE_DT_F16>(p, off, v);
  else
    load8<HMOE_DT_BF16>(p, off, v);
}

__device__ __forceinline__ void store8_rt(void* p, int dt, int64_t off, const float (&v)[8]) {
  if (dt == HMOE_DT_F32)
    store8<HMOE_DT_F32>(p, off, v);
  else if (dt == HMOE_DT_F16)
    store8<HMOE_DT_F16>(p, off, v);
  else
    store8<HMOE_DT_BF16>(p, off, v);
}

// ---------------------------------------------------------------------------------------------------------------
// Rows -> samples.  starts (B + 1,): sample b holds rows starts[b] .. starts[b + 1] - 1, the other rows are padding;
// without starts, B runs of L rows.  The values of starts only choose among the B parameter rows and bound loops that
// stay inside the T rows, so a malformed array gives wrong results and no access out of range.
// ---------------------------------------------------------------------------------------------------------------
struct Samples {
  const int32_t* starts;
  int B, L, T;
};

// the sample of row r (-1 or B: a padding row before the first / behind the last) and the end of its run of rows
__device__ __forceinline__ int sample_of(const Samples& s, int r, int& end) {
  if (!s.starts) {
    const int b = (uint32_t)r / (uint32_t)s.L;
    end = (b + 1) * s.L;
    return b;
  }
  int lo = -1, hi = s.B + 1;  // starts[lo] <= r < starts[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (s.starts[m] <= r)
      lo = m;
    else
      hi = m;
  }
  end = hi <= s.B ? s.starts[hi] : s.T;
  end = end > r ? end : r + 1;
  return lo;
}

// ---------------------------------------------------------------------------------------------------------------
// A row is held by WPR waves, each lane VPL vectors of eight columns: vector i of lane l of the row's 64 WPR is
// l + 64 WPR i.
// ---------------------------------------------------------------------------------------------------------------
constexpr int64_t kNormMaxD = 16 * 64 * 2 * 8;  // the widest: 16 waves, 64 lanes, two vectors of eight columns

// sums of two values over a row's waves; every lane of the row ends with both
template <int WPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
  a = wave_sum_butterfly(a);
  b = wave_sum_butterfly(b);
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x >> 6, row = wave / WPR * WPR;
    __syncthreads();  // the last use of red is over
    if ((threadIdx.x & 63) == 0) {
      red[2 * wave] = a;
      red[2 * wave + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) {
      a += red[2 * (row + i)];
      b += red[2 * (row + i) + 1];
    }
  }
}

__device__ __forceinline__ float inv_rms(float sumsq, int d, float eps) { return 1.0f / sqrtf(sumsq / (float)d + eps); }

struct NormParams {
  const void *weight, *scale, *shift;  // (d,), (B, d), (B, d): NULL for none; norm_residual: scale is the gate
  int weight_dt, scale_dt, shift_dt;
};

struct NormInArgs {
  const void* x;
  int64_t ldx;
  void* h;
  NormParams p;
  Samples s;
  int d;
  float eps;
};

// h = x r w (1 + scale_b) + shift_b, r = (mean(x^2) + eps)^-1/2, 0 on padding rows.  Waves walk rows grid-strided.
template <int ST, int HT, int VPL, int WPR>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void norm_in_kernel(NormInArgs a) {
  __shared__ float red[2 * 16];
  const int nv = a.d / 8, rpb = (int)(blockDim.x >> 6) / WPR;
  const int lane = threadIdx.x % (64 * WPR);
  for (int r0 = blockIdx.x * rpb; r0 < a.s.T; r0 += gridDim.x * rpb) {
    const int r = r0 + threadIdx.x / (64 * WPR);
    const bool row = r < a.s.T;
    float x[VPL][8];
    float sq = 0.0f, unused = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
      if (row && c < nv) load8<ST>(a.x, (int64_t)r * a.ldx + 8 * c, x[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += x[i][e] * x[i][e];
    }
    row_sum2<WPR>(sq, unused, red);
    const float rms = inv_rms(sq, a.d, a.eps);
    if (!row) continue;
    int end;
    const int b = sample_of(a.s, r, end);
    const bool live = b >= 0 && b < a.s.B;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
      if (c >= nv) continue;
      float h[8], t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = live ? x[i][e] * rms : 0.0f;
      if (live) {
        if (a.p.weight) {
          load8_rt(a.p.weight, a.p.weight_dt, 8 * c, t);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] *= t[e];
        }
        if (a.p.scale) {
          load8_rt(a.p.scale, a.p.scale_dt, (int64_t)b * a.d + 8 * c, t);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] *= 1.0f + t[e];
        }
        if (a.p.shift) {
          load8_rt(a.p.shift, a.p.shift_dt, (int64_t)b * a.d + 8 * c, t);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] += t[e];
        }
      }
      store8<HT>(a.h, (int64_t)r * a.d + 8 * c, h);
    }
  }
}

struct NormOutArgs {
  const void* y;  // (T k, d)
  const int32_t* inv_pos;
  const void *add, *x;
  int64_t ldx;
  void* out;
  NormParams p;
  Samples s;
  int d, k, norm;
  float eps, alpha;
};

// the k slots of row r, columns 8 c .. 8 c + 7, summed in slot order in fp32, then the addend; a slot routed nowhere
// adds nothing (its row of y was never written)
template <int HT>
__device__ __forceinline__ void load_slots(const void* y, const int32_t* inv_pos, const void* add, int k, int d, int r,
                                           int c, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.0f;
  float t[8];
  for (int j = 0; j < k; ++j) {
    const int64_t f = (int64_t)r * k + j;
    load8<HT>(y, f * d + 8 * c, t);
    const bool on = !inv_pos || inv_pos[f] >= 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += on ? t[e] : 0.0f;
  }
  if (add) {
    load8<HT>(add, (int64_t)r * d + 8 * c, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
  }
}

// out = alpha x + gate_b w s r(s), s the sum over the row's slots; alpha x on padding rows (whose y is not used)
template <int ST, int HT, int VPL, int WPR>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void norm_out_kernel(NormOutArgs a) {
  __shared__ float red[2 * 16];
  const int nv = a.d / 8, rpb = (int)(blockDim.x >> 6) / WPR;
  const int lane = threadIdx.x % (64 * WPR);
  for (int r0 = blockIdx.x * rpb; r0 < a.s.T; r0 += gridDim.x * rpb) {
    const int r = r0 + threadIdx.x / (64 * WPR);
    const bool row = r < a.s.T;
    float y[VPL][8];
    float sq = 0.0f, unused = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[i][e] = 0.0f;
      if (row && c < nv) load_slots<HT>(a.y, a.inv_pos, a.add, a.k, a.d, r, c, y[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += y[i][e] * y[i][e];
    }
    float rms = 1.0f;
    if (a.norm) {
      row_sum2<WPR>(sq, unused, red);
      rms = inv_rms(sq, a.d, a.eps);
    }
    if (!row) continue;
    int end;
    const int b = sample_of(a.s, r, end);
    const bool live = b >= 0 && b < a.s.B;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
      if (c >= nv) continue;
      float x[8], t[8], z[8];
      load8<ST>(a.x, (int64_t)r * a.ldx + 8 * c, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = live ? y[i][e] * rms : 0.0f;
      if (live && a.p.weight) {
        load8_rt(a.p.weight, a.p.weight_dt, 8 * c, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] *= t[e];
      }
      if (live && a.p.scale) {
        load8_rt(a.p.scale, a.p.scale_dt, (int64_t)b * a.d + 8 * c, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] *= t[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = a.alpha * x[e] + z[e];
      store8<ST>(a.out, (int64_t)r * a.d + 8 * c, z);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Backward.  Block c takes the R rows from c R on, in pieces of one sample; its row groups (WPR waves each) walk a
// piece's rows and keep column sums in registers, which are added over the groups in LDS in group order.  With
// n = v r the normed row (v = x, or the slots' sum) and u the upstream row:
//   norm_in:  g = u w (1 + scale_b), dx = r (g - n mean(g n)) + c dres, A_b = sum u n, dshift_b = sum u,
//             dscale_b = w A_b, dw = sum_rows u (1 + scale_b) n
//   norm_out: g = u w gate_b,        dy = r (g - n mean(g n)),          A_b = sum u n,
//             dgate_b = w A_b,  dw = sum_rows u gate_b n
// mean(g n) = r sum(g v) / d, so both row sums (v^2 and g v) are taken in one exchange.
// A sample inside one block's rows is finished by that block; pieces of longer ones go to slot c + b of the workspace
// (c and b never fall along the rows and one of them grows from piece to piece, so slots are distinct) and
// norm_sums_kernel adds them in chunk order.
// ---------------------------------------------------------------------------------------------------------------
struct NormBwdArgs {
  const void* u;  // upstream rows (contiguous)
  const void* v;  // norm_in: x (row stride ldv); norm_out: y (T k, d)
  int64_t ldv;
  const int32_t* inv_pos;
  const void* add;
  const void* dres;
  float dres_scale;
  void* dv;
  NormParams p;
  void *dweight, *dscale, *dshift;  // of the parameters' types; NULL to skip
  float* part;    // (chunks + B) x nsum x d
  float* wpart;   // chunks x d
  Samples s;
  int d, k, norm, R;
  float eps;
};

template <bool OUT, int ST, int HT, int VPL, int WPR>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 512) void norm_bwd_kernel(NormBwdArgs a) {
  constexpr int UT = OUT ? ST : HT;  // upstream type
  __shared__ float red[2 * 16];
  extern __shared__ float colsum[];  // (row groups) x d
  const int nv = a.d / 8, ngrp = (int)(blockDim.x >> 6) / WPR;
  const int lane = threadIdx.x % (64 * WPR), grp = threadIdx.x / (64 * WPR);
  const int r_begin = blockIdx.x * a.R, r_end = min(a.s.T, r_begin + a.R);
  const bool sums = a.dscale || a.dshift;
  const int nsum = (a.dscale != nullptr) + (a.dshift != nullptr);
  float wacc[VPL][8];
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) wacc[i][e] = 0.0f;
  // adds a column sum over the row groups and hands eight columns at a time to fin(column vector, sums)
  auto over_groups = [&](const float (&acc)[VPL][8], auto&& fin) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
      if (c < nv) store8<HMOE_DT_F32>(colsum, (int64_t)grp * a.d + 8 * c, acc[i]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < nv; c += blockDim.x) {
      float t[8], q[8];
      load8<HMOE_DT_F32>(colsum, 8 * c, t);
      for (int g = 1; g < ngrp; ++g) {
        load8<HMOE_DT_F32>(colsum, (int64_t)g * a.d + 8 * c, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] += q[e];
      }
      fin(c, t);
    }
  };
  for (int r0 = r_begin; r0 < r_end;) {
    int end;
    const int b = sample_of(a.s, r0, end);
    const int piece_end = min(end, r_end);
    const bool live = b >= 0 && b < a.s.B;
    if (!live) {  // padding rows: no gradient from the norm
      for (int r = r0 + grp; r < piece_end; r += ngrp)
        for (int c = lane; c < nv; c += 64 * WPR) {
          float t[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] = 0.0f;
          if (a.dres) {
            load8<ST>(a.dres, (int64_t)r * a.d + 8 * c, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] *= a.dres_scale;
          }
          store8<OUT ? HT : ST>(a.dv, (int64_t)r * a.d + 8 * c, t);
        }
      r0 = piece_end;
      continue;
    }
    float aacc[VPL][8], sacc[VPL][8], wm[VPL][8];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        aacc[i][e] = sacc[i][e] = 0.0f;
        wm[i][e] = 1.0f;
      }
      if (c < nv) {
        float t[8];
        if (a.p.weight) load8_rt(a.p.weight, a.p.weight_dt, 8 * c, wm[i]);
        if (a.p.scale) {
          load8_rt(a.p.scale, a.p.scale_dt, (int64_t)b * a.d + 8 * c, t);
#pragma unroll
          for (int e = 0; e < 8; ++e) wm[i][e] *= OUT ? t[e] : 1.0f + t[e];
        }
      }
    }
    for (int rg = r0; rg < piece_end; rg += ngrp) {
      const int r = rg + grp;
      const bool row = r < piece_end;
      float u[VPL][8], v[VPL][8];
      float sq = 0.0f, dot = 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int c = lane + 64 * WPR * i;
#pragma unroll
        for (int e = 0; e < 8; ++e) u[i][e] = v[i][e] = 0.0f;
        if (row && c < nv) {
          load8<UT>(a.u, (int64_t)r * a.d + 8 * c, u[i]);
          if constexpr (OUT)
            load_slots<HT>(a.v, a.inv_pos, a.add, a.k, a.d, r, c, v[i]);
          else
            load8<ST>(a.v, (int64_t)r * a.ldv + 8 * c, v[i]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sq += v[i][e] * v[i][e];
          dot += u[i][e] * wm[i][e] * v[i][e];
        }
      }
      float rms = 1.0f, proj = 0.0f;  // proj = r^3 mean(g v): dv = r g - v proj
      if (a.norm) {
        row_sum2<WPR>(sq, dot, red);
        rms = inv_rms(sq, a.d, a.eps);
        proj = rms * rms * rms * (dot / (float)a.d);
      }
      if (!row) continue;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int c = lane + 64 * WPR * i;
        if (c >= nv) continue;
        float t[8], dr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float n = v[i][e] * rms;
          aacc[i][e] += u[i][e] * n;
          sacc[i][e] += u[i][e];
          t[e] = rms * (u[i][e] * wm[i][e]) - v[i][e] * proj;
        }
        if (a.dres) {
          load8<ST>(a.dres, (int64_t)r * a.d + 8 * c, dr);
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] += a.dres_scale * dr[e];
        }
        store8<OUT ? HT : ST>(a.dv, (int64_t)r * a.d + 8 * c, t);
      }
    }
    if (a.dweight) {  // the weight's sum: A_b (1 + scale_b), or A_b gate_b
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int c = lane + 64 * WPR * i;
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = OUT ? 1.0f : 0.0f;
        if (a.p.scale && c < nv) load8_rt(a.p.scale, a.p.scale_dt, (int64_t)b * a.d + 8 * c, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) wacc[i][e] += (OUT ? t[e] : 1.0f + t[e]) * aacc[i][e];
      }
    }
    if (sums) {
      // (whole: this block holds every row of the sample)
      const int first = a.s.starts ? a.s.starts[b] : b * a.s.L;
      const bool whole = first >= r_begin && end <= r_end;
      float* slot = a.part + (int64_t)(blockIdx.x + b) * nsum * a.d;
      if (a.dscale)
        over_groups(aacc, [&](int c, float (&t)[8]) {
          if (!whole) {
            store8<HMOE_DT_F32>(slot, 8 * c, t);
            return;
          }
          if (a.p.weight) {
            float q[8];
            load8_rt(a.p.weight, a.p.weight_dt, 8 * c, q);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] *= q[e];
          }
          store8_rt(a.dscale, a.p.scale_dt, (int64_t)b * a.d + 8 * c, t);
        });
      if (a.dshift)
        over_groups(sacc, [&](int c, float (&t)[8]) {
          if (whole)
            store8_rt(a.dshift, a.p.shift_dt, (int64_t)b * a.d + 8 * c, t);
          else
            store8<HMOE_DT_F32>(slot, (int64_t)(nsum - 1) * a.d + 8 * c, t);
        });
    }
    r0 = piece_end;
  }
  if (a.dweight)
    over_groups(wacc, [&](int c, float (&t)[8]) {
      store8<HMOE_DT_F32>(a.wpart, (int64_t)blockIdx.x * a.d + 8 * c, t);
    });
}

// The column sums left in the workspace: block (item, 64-column slab), item < B: sample item's sums, unless one chunk
// finished it (an empty sample gets zeros); item B: the weight's over all chunks.  16 waves take every 16th slot.
__global__ __launch_bounds__(1024) void norm_sums_kernel(NormBwdArgs a, int nchunk) {
  __shared__ float lds[2][16][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, b = blockIdx.x;
  const int col = blockIdx.y * 64 + tx;
  const int nsum = (a.dscale != nullptr) + (a.dshift != nullptr);
  const bool weight = b == a.s.B;
  int c0 = 0, c1 = nchunk - 1;
  if (!weight) {
    int s = a.s.starts ? a.s.starts[b] : b * a.s.L, e = a.s.starts ? a.s.starts[b + 1] : (b + 1) * a.s.L;
    s = max(0, min(s, a.s.T));
    e = max(0, min(e, a.s.T));
    c0 = s / a.R;
    c1 = (e - 1) / a.R;
    if (e <= s)
      c1 = c0 - 1;  // empty: zeros
    else if (c0 == c1)
      return;
  }
  float t0 = 0.0f, t1 = 0.0f;
  if (col < a.d) {
    for (int c = c0 + ty; c <= c1; c += 16) {
      if (weight) {
        t0 += a.wpart[(int64_t)c * a.d + col];
      } else {
        const float* slot = a.part + (int64_t)(c + b) * nsum * a.d + col;
        t0 += slot[0];
        if (nsum == 2) t1 += slot[a.d];
      }
    }
  }
  lds[0][ty][tx] = t0;
  lds[1][ty][tx] = t1;
  __syncthreads();
  if (ty != 0 || col >= a.d) return;
  for (int i = 1; i < 16; ++i) {
    t0 += lds[0][i][tx];
    t1 += lds[1][i][tx];
  }
  auto put = [&](void* p, int dt, int64_t off, float v) {
    if (dt == HMOE_DT_F32)
      static_cast<float*>(p)[off] = v;
    else
      static_cast<uint16_t*>(p)[off] = (uint16_t)(dt == HMOE_DT_F16 ? cvt_h2(v, v) : cvt_bf2(v, v));
  };
  if (weight) {
    put(a.dweight, a.p.weight_dt, col, t0);
    return;
  }
  const int64_t off = (int64_t)b * a.d + col;
  if (a.dscale) {
    float w = 1.0f;
    if (a.p.weight)
      w = a.p.weight_dt == HMOE_DT_F32 ? static_cast<const float*>(a.p.weight)[col]
          : a.p.weight_dt == HMOE_DT_F16 ? Elt<true>::one(static_cast<const uint16_t*>(a.p.weight)[col])
                                         : Elt<false>::one(static_cast<const uint16_t*>(a.p.weight)[col]);
    put(a.dscale, a.p.scale_dt, off, w * t0);
  }
  if (a.dshift) put(a.dshift, a.p.shift_dt, off, a.dscale ? t1 : t0);
}

// ---------------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------------
static inline bool al16(const void* p) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static inline bool float_dt(int dt) { return dt == HMOE_DT_BF16 || dt == HMOE_DT_F16 || dt == HMOE_DT_F32; }

// stream type (x, out) and block type (h, y): equal, or an fp32 stream around a 16-bit block
static int norm_types(int sdt, int hdt) {
  if (!float_dt(sdt) || !float_dt(hdt)) return HMOE_ERR_DTYPE;
  return sdt == hdt || sdt == HMOE_DT_F32 ? HMOE_OK : HMOE_ERR_DTYPE;
}

static int norm_sizes(int64_t T, int64_t d, int64_t B, const int32_t* starts) {
  if (T < 0 || d <= 0 || B < 1) return HMOE_ERR_ARG;
  if (d % 8 || d > kNormMaxD || T > INT32_MAX / 2 || B > INT32_MAX / 2 || T + B > INT32_MAX / 2) return HMOE_ERR_SHAPE;
  if (!starts && T % B) return HMOE_ERR_SHAPE;
  return HMOE_OK;
}

static int norm_params(const NormParams& p) {
  if ((p.weight && !float_dt(p.weight_dt)) || (p.scale && !float_dt(p.scale_dt)) || (p.shift && !float_dt(p.shift_dt)))
    return HMOE_ERR_DTYPE;
  return al16(p.weight) && al16(p.scale) && al16(p.shift) ? HMOE_OK : HMOE_ERR_ARG;
}

// calls f(VPL, WPR) as integral constants for width d: one wave per row up to 2048 columns, four up to 8192, else 16
template <class F>
static void by_width(int64_t d, F&& f) {
  const int64_t nv = d / 8;
#define HMOE_W(V, W) f(std::integral_constant<int, V>(), std::integral_constant<int, W>())
  if (nv <= 64) HMOE_W(1, 1);
  else if (nv <= 128) HMOE_W(2, 1);
  else if (nv <= 192) HMOE_W(3, 1);
  else if (nv <= 256) HMOE_W(4, 1);
  else if (nv <= 512) HMOE_W(2, 4);
  else if (nv <= 768) HMOE_W(3, 4);
  else if (nv <= 1024) HMOE_W(4, 4);
  else HMOE_W(2, 16);
#undef HMOE_W
}

// calls f(ST, HT) as integral constants
template <class F>
static void by_types(int sdt, int hdt, F&& f) {
#define HMOE_T(S, H) f(std::integral_constant<int, S>(), std::integral_constant<int, H>())
  if (sdt == HMOE_DT_BF16) HMOE_T(HMOE_DT_BF16, HMOE_DT_BF16);
  else if (sdt == HMOE_DT_F16) HMOE_T(HMOE_DT_F16, HMOE_DT_F16);
  else if (hdt == HMOE_DT_BF16) HMOE_T(HMOE_DT_F32, HMOE_DT_BF16);
  else if (hdt == HMOE_DT_F16) HMOE_T(HMOE_DT_F32, HMOE_DT_F16);
  else HMOE_T(HMOE_DT_F32, HMOE_DT_F32);
#undef HMOE_T
}

// blocks of a forward launch: a row per wave (or per WPR waves), at most eight blocks per CU of 256
static unsigned norm_grid(int64_t T, int rows_per_block) {
  const int64_t g = (T + rows_per_block - 1) / rows_per_block;
  return (unsigned)(g < 2048 ? g : 2048);
}

// rows per block of the backward: about 512 blocks
static int bwd_rows(int64_t T, int groups) {
  int64_t r = (T + 511) / 512;
  r = (r + groups - 1) / groups * groups;
  return (int)(r > 0 ? r : groups);
}
static int bwd_groups(int64_t d) { return d <= 2048 ? 8 : d <= 8192 ? 2 : 1; }

static size_t norm_bwd_ws(int64_t T, int64_t d, int64_t B, int nsum, bool weight) {
  if (T < 0 || d <= 0 || B < 1) return 0;
  const int64_t R = bwd_rows(T, bwd_groups(d)), nchunk = (T + R - 1) / R;
  return (size_t)((nchunk + B) * nsum + (weight ? nchunk : 0)) * (size_t)d * 4 + 16;
}

template <bool OUT>
static int norm_bwd_run(NormBwdArgs& a, int sdt, int hdt, void* workspace, size_t workspace_bytes, hipStream_t s) {
  const int nsum = (a.dscale != nullptr) + (a.dshift != nullptr);
  const int groups = bwd_groups(a.d);
  a.R = bwd_rows(a.s.T, groups);
  const int nchunk = (a.s.T + a.R - 1) / a.R;
  const bool final = nsum || a.dweight;
  if (final) {
    if (!workspace || workspace_bytes < norm_bwd_ws(a.s.T, a.d, a.s.B, nsum, a.dweight != nullptr))
      return HMOE_ERR_WORKSPACE;
    if (!al16(workspace)) return HMOE_ERR_ARG;
    a.part = static_cast<float*>(workspace);
    a.wpart = a.part + (int64_t)(nchunk + a.s.B) * nsum * a.d;
  }
  if (nchunk) {
    const size_t lds = final ? (size_t)groups * a.d * 4 : 0;
    by_types(sdt, hdt, [&](auto st, auto ht) {
      by_width(a.d, [&](auto v, auto w) {
        constexpr int W = decltype(w)::value;
        hipLaunchKernelGGL((norm_bwd_kernel<OUT, decltype(st)::value, decltype(ht)::value, decltype(v)::value, W>),
                           dim3(nchunk), dim3(W == 16 ? 1024 : 512), lds, s, a);
      });
    });
    HMOE_CHECK_LAUNCH();
  }
  if (final) {
    const int items = (nsum ? a.s.B : 0) + (a.dweight ? 1 : 0);
    // without sample sums the weight's item comes first
    NormBwdArgs f = a;
    if (!nsum) f.s.B = 0;
    hipLaunchKernelGGL(norm_sums_kernel, dim3(items, (a.d + 63) / 64), dim3(1024), 0, s, f, nchunk);
    HMOE_CHECK_LAUNCH();
  }
  return HMOE_OK;
}

}  // namespace hmoe

using namespace hmoe;

extern "C" {

int hmoe_norm_modulate(const void* x, int64_t ldx, int x_dtype, const void* weight, int weight_dtype,
                       const void* scale, const void* shift, int mod_dtype, const int32_t* starts, int64_t B, int64_t T,
                       int64_t d, float eps, void* h, int h_dtype, hmoe_stream_t stream) {
  int rc = norm_sizes(T, d, B, starts);
  if (rc == HMOE_OK) rc = norm_types(x_dtype, h_dtype);
  const NormParams p = {weight, scale, shift, weight_dtype, mod_dtype, mod_dtype};
  if (rc == HMOE_OK) rc = norm_params(p);
  if (rc || T == 0) return rc;
  if (!x || !h || ldx < d || ldx % 8 || !al16(x) || !al16(h)) return HMOE_ERR_ARG;
  const NormInArgs a = {x, ldx, h, p, {starts, (int)B, starts ? 0 : (int)(T / B), (int)T}, (int)d, eps};
  by_types(x_dtype, h_dtype, [&](auto st, auto ht) {
    by_width(d, [&](auto v, auto w) {
      constexpr int W = decltype(w)::value;
      hipLaunchKernelGGL((norm_in_kernel<decltype(st)::value, decltype(ht)::value, decltype(v)::value, W>),
                         dim3(norm_grid(T, W == 1 ? 4 : 1)), dim3(W == 16 ? 1024 : 256), 0,
                         reinterpret_cast<hipStream_t>(stream), a);
    });
  });
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

int hmoe_norm_residual(const void* y, const int32_t* inv_pos, int k, const void* add, int y_dtype, const void* x,
                       int64_t ldx, int x_dtype, const void* weight, int weight_dtype, const void* gate, int gate_dtype,
                       const int32_t* starts, int64_t B, int64_t T, int64_t d, int norm, float eps, float alpha,
                       void* out, hmoe_stream_t stream) {
  int rc = norm_sizes(T, d, B, starts);
  if (rc == HMOE_OK) rc = norm_types(x_dtype, y_dtype);
  const NormParams p = {weight, gate, nullptr, weight_dtype, gate_dtype, 0};
  if (rc == HMOE_OK) rc = norm_params(p);
  if (k < 1) return HMOE_ERR_ARG;
  if (rc || T == 0) return rc;
  if (!y || !x || !out || ldx < d || ldx % 8 || !al16(y) || !al16(x) || !al16(out) || !al16(add)) return HMOE_ERR_ARG;
  const NormOutArgs a = {y, inv_pos, add, x, ldx, out, p, {starts, (int)B, starts ? 0 : (int)(T / B), (int)T}, (int)d,
                         k, norm, eps, alpha};
  by_types(x_dtype, y_dtype, [&](auto st, auto ht) {
    by_width(d, [&](auto v, auto w) {
      constexpr int W = decltype(w)::value;
      hipLaunchKernelGGL((norm_out_kernel<decltype(st)::value, decltype(ht)::value, decltype(v)::value, W>),
                         dim3(norm_grid(T, W == 1 ? 4 : 1)), dim3(W == 16 ? 1024 : 256), 0,
                         reinterpret_cast<hipStream_t>(stream), a);
    });
  });
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

size_t hmoe_norm_modulate_bwd_workspace_size(int64_t T, int64_t d, int64_t B) { return norm_bwd_ws(T, d, B, 2, true); }

int hmoe_norm_modulate_bwd(const void* dh, int h_dtype, const void* x, int64_t ldx, int x_dtype, const void* weight,
                           int weight_dtype, const void* scale, const void* shift, int mod_dtype, const int32_t* starts,
                           int64_t B, int64_t T, int64_t d, float eps, const void* dres, float dres_scale, void* dx,
                           void* dweight, void* dscale, void* dshift, void* workspace, size_t workspace_bytes,
                           hmoe_stream_t stream) {
  int rc = norm_sizes(T, d, B, starts);
  if (rc == HMOE_OK) rc = norm_types(x_dtype, h_dtype);
  const NormParams p = {weight, scale, shift, weight_dtype, mod_dtype, mod_dtype};
  if (rc == HMOE_OK) rc = norm_params(p);
  if (rc) return rc;
  if ((dweight && !weight) || (dscale && !scale) || (dshift && !shift)) return HMOE_ERR_ARG;
  if (!al16(dweight) || !al16(dscale) || !al16(dshift)) return HMOE_ERR_ARG;
  if (T > 0 && (!dh || !x || !dx || ldx < d || ldx % 8 || !al16(dh) || !al16(x) || !al16(dx) || !al16(dres)))
    return HMOE_ERR_ARG;
  NormBwdArgs a = {dh, x, ldx, nullptr, nullptr, dres, dres_scale, dx, p, dweight, dscale, dshift, nullptr, nullptr,
                   {starts, (int)B, starts ? 0 : (int)(T / B), (int)T}, (int)d, 1, 1, 0, eps};
  return norm_bwd_run<false>(a, x_dtype, h_dtype, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

size_t hmoe_norm_residual_bwd_workspace_size(int64_t T, int64_t d, int64_t B) { return norm_bwd_ws(T, d, B, 1, true); }

int hmoe_norm_residual_bwd(const void* dout, int out_dtype, const void* y, const int32_t* inv_pos, int k,
                           const void* add, int y_dtype, const void* weight, int weight_dtype, const void* gate,
                           int gate_dtype, const int32_t* starts, int64_t B, int64_t T, int64_t d, int norm, float eps,
                           void* dy, void* dweight, void* dgate, void* workspace, size_t workspace_bytes,
                           hmoe_stream_t stream) {
  int rc = norm_sizes(T, d, B, starts);
  if (rc == HMOE_OK) rc = norm_types(out_dtype, y_dtype);
  const NormParams p = {weight, gate, nullptr, weight_dtype, gate_dtype, 0};
  if (rc == HMOE_OK) rc = norm_params(p);
  if (rc) return rc;
  if (k < 1 || (dweight && !weight) || (dgate && !gate) || !al16(dweight) || !al16(dgate)) return HMOE_ERR_ARG;
  if (T > 0 && (!dout || !y || !dy || !al16(dout) || !al16(y) || !al16(dy) || !al16(add))) return HMOE_ERR_ARG;
  NormBwdArgs a = {dout, y, d, inv_pos, add, nullptr, 0.0f, dy, p, dweight, dgate, nullptr, nullptr, nullptr,
                   {starts, (int)B, starts ? 0 : (int)(T / B), (int)T}, (int)d, k, norm, 0, eps};
  return norm_bwd_run<true>(a, out_dtype, y_dtype, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
