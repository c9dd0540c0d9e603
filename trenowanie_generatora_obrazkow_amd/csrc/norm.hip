// The norms around the routed block, with their C entry points: the RMS norm before it with weight and per-sample
// scale / shift, and the sum over the routed slots, RMS norm, gate and scaled residual after it; both with backward.
// A few operations per element: every kernel here is bound by the rows it reads and writes.  16384 x 1536 bf16, 4 samples:
// norm_in 22.9 us forward (101 MB, 4.4 TB/s), 36.4 backward (201 MB, 5.5 TB/s) and 4.7 for the sums; norm_out with two slots
// 44.2 (201 MB, 4.6 TB/s), 36.6 (201 MB, 5.5 TB/s) and 5.2.  A copy of 2 GB runs at 5.1 TB/s.
#include "hmoe_common.h"

namespace hmoe {

// ---------------------------------------------------------------------------------------------------------------
// Eight consecutive elements, 16 bytes aligned, at column col of the row that starts at element `row` of p: the row is the
// same for the whole wave, so it stays in scalar registers.  As fp32, of a type known at compile time (rows) or at run time
// (parameters: a branch that is uniform over the grid).
// ---------------------------------------------------------------------------------------------------------------
template <int DT>
constexpr int kSize = DT == HMOE_DT_F32 ? 4 : 2;
template <int DT>
__device__ __forceinline__ const void* at(const void* p, int64_t row, uint32_t col) {
  return static_cast<const char*>(p) + row * kSize<DT> + col * kSize<DT>;
}
template <int DT>
__device__ __forceinline__ void* at(void* p, int64_t row, uint32_t col) {
  return static_cast<char*>(p) + row * kSize<DT> + col * kSize<DT>;
}

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t row, uint32_t col, float (&v)[8]) {
  if constexpr (DT == HMOE_DT_F32) {
    const f32x4* q = static_cast<const f32x4*>(at<DT>(p, row, col));
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else {
    using X = Elt<DT == HMOE_DT_F16>;
    const uint4 u = *static_cast<const uint4*>(at<DT>(p, row, col));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = X::lo(w[i]);
      v[2 * i + 1] = X::hi(w[i]);
    }
  }
}

// The same eight elements as they lie in memory: a row waits for its sums in this form (half the registers of fp32 for
// 16-bit types) and is widened at each use.
template <int DT>
struct Raw8 {
  static constexpr int kRegs = DT == HMOE_DT_F32 ? 8 : 4;
  uint32_t w[kRegs];
  __device__ __forceinline__ void load(const void* p, int64_t row, uint32_t col) {
    const uint4* q = static_cast<const uint4*>(at<DT>(p, row, col));
#pragma unroll
    for (int i = 0; i < kRegs / 4; ++i) {
      const uint4 u = q[i];
      w[4 * i] = u.x;
      w[4 * i + 1] = u.y;
      w[4 * i + 2] = u.z;
      w[4 * i + 3] = u.w;
    }
  }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (DT == HMOE_DT_F32) return __uint_as_float(w[e]);
    else {
      using X = Elt<DT == HMOE_DT_F16>;
      return e & 1 ? X::hi(w[e >> 1]) : X::lo(w[e >> 1]);
    }
  }
  __device__ __forceinline__ void keep(bool on) {
#pragma unroll
    for (int i = 0; i < kRegs; ++i) w[i] = on ? w[i] : 0;
  }
  // the compiler must not keep the widened elements across this point
  __device__ __forceinline__ void hold() {
#pragma unroll
    for (int i = 0; i < kRegs; ++i) asm volatile("" : "+v"(w[i]));
  }
};

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t row, uint32_t col, const float (&v)[8]) {
  if constexpr (DT == HMOE_DT_F32) {
    f32x4* q = static_cast<f32x4*>(at<DT>(p, row, col));
    q[0] = f32x4{v[0], v[1], v[2], v[3]};
    q[1] = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    using X = Elt<DT == HMOE_DT_F16>;
    *static_cast<uint4*>(at<DT>(p, row, col)) =
        make_uint4(X::pack2(v[0], v[1]), X::pack2(v[2], v[3]), X::pack2(v[4], v[5]), X::pack2(v[6], v[7]));
  }
}

__device__ __forceinline__ void load8_rt(const void* p, int dt, int64_t row, uint32_t col, float (&v)[8]) {
  if (dt == HMOE_DT_F32)
    load8<HMOE_DT_F32>(p, row, col, v);
  else if (dt == HMOE_DT_F16)
    load8<HMOE_DT_F16>(p, row, col, v);
  else
    load8<HMOE_DT_BF16>(p, row, col, v);
}

__device__ __forceinline__ void store8_rt(void* p, int dt, int64_t row, uint32_t col, const float (&v)[8]) {
  if (dt == HMOE_DT_F32)
    store8<HMOE_DT_F32>(p, row, col, v);
  else if (dt == HMOE_DT_F16)
    store8<HMOE_DT_F16>(p, row, col, v);
  else
    store8<HMOE_DT_BF16>(p, row, col, v);
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

// The sample of row r (-1 or B: a padding row before the first / behind the last) and the end of its run of rows.  r is
// the same for the whole wave: a search down to 64 entries, which the lanes then read at once.
__device__ __forceinline__ int sample_of(const Samples& s, int r, int& end) {
  if (!s.starts) {
    const int b = (uint32_t)r / (uint32_t)s.L;
    end = (b + 1) * s.L;
    return b;
  }
  int lo = -1, hi = s.B + 1;  // starts[lo] <= r < starts[hi], with starts[-1] = 0 and starts[B + 1] = T
  while (hi - lo > 64) {
    const int m = (lo + hi) >> 1;
    if (s.starts[m] <= r)
      lo = m;
    else
      hi = m;
  }
  const int i = lo + 1 + wave_lane();
  const int v = i <= s.B && i <= hi ? s.starts[i] : INT32_MAX;
  const uint64_t past = ~__ballot(v <= r);
  const int n = past ? __builtin_ctzll(past) : 63;
  end = min(__builtin_amdgcn_readlane(v, n), s.T);
  end = end > r ? end : r + 1;
  return lo + n;
}

// ---------------------------------------------------------------------------------------------------------------
// A row is held by WPR waves, each lane VPL vectors of eight columns: vector i of lane l of the row's 64 WPR is
// l + 64 WPR i.  The backward's workgroups have eight waves (16 for WPR = 16) and hold several rows at once.  At most three
// vectors a lane: it keeps two column sums and the row's parameters in registers beside the rows.  by_width picks VPL and WPR
// so that only a lane's last vector can lie past the row (vec_in).  Loads are not predicated, which would make them wait for
// each other: such a vector reads the row's last one and a row past the end the last row, and both are dropped after.
// ---------------------------------------------------------------------------------------------------------------
constexpr int64_t kNormMaxD = 16 * 64 * 2 * 8;
template <int WPR>
constexpr int kNormThreads = WPR == 16 ? 1024 : 512;
template <int WPR>
constexpr int kNormGroups = kNormThreads<WPR> / 64 / WPR;
template <int WPR>
constexpr int kFwdThreads = WPR <= 2 ? 128 : 64 * WPR;  // the forward's: small, for an even share of the rows
template <int WPR>
constexpr int kFwdGroups = kFwdThreads<WPR> / 64 / WPR;

// whether vector c, a lane's i-th, lies in a row of nv vectors
template <int VPL>
__device__ __forceinline__ bool vec_in(int i, int c, int nv) {
  return i < VPL - 1 || c < nv;
}

// sums of two values over a row's waves; every lane of the row ends with both.  Successive calls alternate between the two
// halves of red (2 x 32 floats): one barrier each, since a wave comes back to a half only past the other half's barrier.
template <int WPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red, int& half) {
  a = wave_sum_butterfly(a);
  b = wave_sum_butterfly(b);
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x >> 6, row = wave / WPR * WPR;
    float* r = red + 32 * half;
    half ^= 1;
    if ((threadIdx.x & 63) == 0) {
      r[2 * wave] = a;
      r[2 * wave + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) {
      a += r[2 * (row + i)];
      b += r[2 * (row + i) + 1];
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
  int d, R;
  float eps;
};

// h = x r w (1 + scale_b) + shift_b, r = (mean(x^2) + eps)^-1/2, 0 on padding rows.  A workgroup takes R rows, each of its
// row groups every kFwdGroups-th; the parameters of a sample are read once, beside its first row, and the next row is
// on its way while a row is summed.
template <int ST, int HT, int VPL, int WPR>
__global__ __launch_bounds__(kFwdThreads<WPR>) void norm_in_kernel(NormInArgs a) {
  __shared__ float red[2 * 32];
  constexpr int G = kFwdGroups<WPR>;
  const int nv = a.d / 8, lane = threadIdx.x % (64 * WPR);
  const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WPR));
  const int r_end = min(a.s.T, (int)(blockIdx.x + 1) * a.R);
  int half = 0, b = 0, end = -1;
  bool live = false;
  Raw8<ST> x[VPL], nx[VPL];
  auto fetch = [&](int r, Raw8<ST> (&v)[VPL]) {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      v[i].load(a.x, (int64_t)min(r, r_end - 1) * a.ldx, 8 * min(lane + 64 * WPR * i, nv - 1));
  };
  float m[VPL][8], sh[VPL][8];
  const int r0 = blockIdx.x * a.R;
  fetch(r0 + grp, nx);
  for (int rg = r0; rg < r_end; rg += G) {  // (the same count for every wave: row_sum2 may hold a barrier)
    const int r = rg + grp;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      x[i] = nx[i];
      x[i].keep(vec_in<VPL>(i, lane + 64 * WPR * i, nv));
    }
    if (rg + G < r_end) fetch(r + G, nx);
    if (r < r_end && r >= end) {
      b = sample_of(a.s, r, end);
      live = b >= 0 && b < a.s.B;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int c = lane + 64 * WPR * i;
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          m[i][e] = 1.0f;
          sh[i][e] = 0.0f;
        }
        if (live && vec_in<VPL>(i, c, nv)) {
          if (a.p.weight) load8_rt(a.p.weight, a.p.weight_dt, 0, 8 * c, m[i]);
          if (a.p.scale) {
            load8_rt(a.p.scale, a.p.scale_dt, (int64_t)b * a.d, 8 * c, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) m[i][e] *= 1.0f + t[e];
          }
          if (a.p.shift) load8_rt(a.p.shift, a.p.shift_dt, (int64_t)b * a.d, 8 * c, sh[i]);
        }
      }
    }
    float sq = 0.0f, unused = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += x[i][e] * x[i][e];
    row_sum2<WPR>(sq, unused, red, half);
    const float rms = inv_rms(sq, a.d, a.eps);
    if (r >= r_end) continue;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
      if (!vec_in<VPL>(i, c, nv)) continue;
      float h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = live ? x[i][e] * rms * m[i][e] + sh[i][e] : 0.0f;
      store8<HT>(a.h, (int64_t)r * a.d, 8 * c, h);
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
  int d, k, norm, R;
  float eps, alpha;
};

// s = the sum over the k slots of row r in slot order in fp32, then the addend; a slot routed nowhere adds nothing (its row of
// y was never written).  KB slots are on their way at once.
template <int HT, int VPL, int WPR, int KB>
__device__ __forceinline__ void load_slots(const void* y, const int32_t* inv_pos, const void* add, int k, int d, int r,
                                           int lane, float (&s)[VPL][8]) {
  const int nv = d / 8;
  uint32_t col[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    col[i] = 8 * min(lane + 64 * WPR * i, nv - 1);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[i][e] = 0.0f;
  }
  Raw8<HT> ad[VPL];
  if (add) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) ad[i].load(add, (int64_t)r * d, col[i]);
  }
  for (int j0 = 0; j0 < k; j0 += KB) {
    Raw8<HT> t[KB][VPL];
    bool on[KB];
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      const int64_t f = (int64_t)r * k + min(j0 + j, k - 1);
      on[j] = j0 + j < k && (!inv_pos || inv_pos[f] >= 0);
#pragma unroll
      for (int i = 0; i < VPL; ++i) t[j][i].load(y, f * d, col[i]);
    }
#pragma unroll
    for (int j = 0; j < KB; ++j)
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        t[j][i].keep(on[j] && vec_in<VPL>(i, lane + 64 * WPR * i, nv));
#pragma unroll
        for (int e = 0; e < 8; ++e) s[i][e] += t[j][i][e];
      }
  }
  if (add) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      ad[i].keep(vec_in<VPL>(i, lane + 64 * WPR * i, nv));
#pragma unroll
      for (int e = 0; e < 8; ++e) s[i][e] += ad[i][e];
    }
  }
}

// out = alpha x + gate_b w s r(s), s the sum over the row's slots; alpha x on padding rows (whose y is not used).  Rows are
// dealt as in norm_in_kernel.
template <int ST, int HT, int VPL, int WPR, int KB>
__global__ __launch_bounds__(kFwdThreads<WPR>, ST == HMOE_DT_F32 || KB == 4 ? 2 : 4) void norm_out_kernel(NormOutArgs a) {
  __shared__ float red[2 * 32];
  constexpr int G = kFwdGroups<WPR>;
  const int nv = a.d / 8, lane = threadIdx.x % (64 * WPR);
  const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WPR));
  const int r_end = min(a.s.T, (int)(blockIdx.x + 1) * a.R);
  int half = 0, b = 0, end = -1;
  bool live = false;
  float m[VPL][8];
  for (int rg = blockIdx.x * a.R; rg < r_end; rg += G) {
    const int r = rg + grp;
    const bool row = r < r_end;
    Raw8<ST> x[VPL];
    float y[VPL][8];
    const int rc = min(r, r_end - 1);
#pragma unroll
    for (int i = 0; i < VPL; ++i) x[i].load(a.x, (int64_t)rc * a.ldx, 8 * min(lane + 64 * WPR * i, nv - 1));
    load_slots<HT, VPL, WPR, KB>(a.y, a.inv_pos, a.add, a.k, a.d, rc, lane, y);
    if (row && r >= end) {
      b = sample_of(a.s, r, end);
      live = b >= 0 && b < a.s.B;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int c = lane + 64 * WPR * i;
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) m[i][e] = 1.0f;
        if (live && vec_in<VPL>(i, c, nv)) {
          if (a.p.weight) load8_rt(a.p.weight, a.p.weight_dt, 0, 8 * c, m[i]);
          if (a.p.scale) {
            load8_rt(a.p.scale, a.p.scale_dt, (int64_t)b * a.d, 8 * c, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) m[i][e] *= t[e];
          }
        }
      }
    }
    float rms = 1.0f;
    if (a.norm) {
      float sq = 0.0f, unused = 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sq += y[i][e] * y[i][e];
      row_sum2<WPR>(sq, unused, red, half);
      rms = inv_rms(sq, a.d, a.eps);
    }
    if (!row) continue;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
      if (!vec_in<VPL>(i, c, nv)) continue;
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = a.alpha * x[i][e] + (live ? y[i][e] * rms * m[i][e] : 0.0f);
      store8<ST>(a.out, (int64_t)r * a.d, 8 * c, z);
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
// A sample inside one block's rows is finished by that block.  Of the others' pieces a block holds at most two: the end or
// middle of one that began before (slot 2 c of the workspace) and the beginning of one that goes on (slot 2 c + 1);
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
  float* part;    // 2 chunks x nsum x d
  float* wpart;   // chunks x d
  Samples s;
  int d, k, norm, R;
  float eps;
};

// KB: 0 for norm_in, else the slots loaded at once for norm_out.
// SHORT (equal samples of few rows): each row group takes whole samples, every G-th of the R / L of its block, and writes
// their sums itself; in the other form the groups share a piece's rows, and with fewer rows than groups most would wait.
template <int KB, int ST, int HT, int VPL, int WPR, bool SHORT>
__global__ __launch_bounds__(kNormThreads<WPR>) void norm_bwd_kernel(NormBwdArgs a) {
  constexpr bool OUT = KB > 0;
  constexpr int UT = OUT ? ST : HT, DT = OUT ? HT : ST;  // types of u and of dv
  // column vectors a thread adds up over the row groups: tid, tid + threads, ...
  constexpr int G = kNormGroups<WPR>, THREADS = kNormThreads<WPR>;
  constexpr int NC = (64 * WPR * VPL + THREADS - 1) / THREADS;
  __shared__ float red[2 * 32];
  extern __shared__ __align__(16) float colsum[];  // G x d
  const int nv = a.d / 8, lane = threadIdx.x % (64 * WPR);
  const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WPR));
  const int r_begin = blockIdx.x * a.R, r_end = min(a.s.T, r_begin + a.R);
  const int nsum = (a.dscale != nullptr) + (a.dshift != nullptr);
  int half = 0;
  float wacc[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) wacc[i][e] = 0.0f;
  // adds a column sum over the row groups and hands eight columns at a time to fin(i, column vector, sums)
  auto over_groups = [&](const float (&acc)[VPL][8], auto&& fin) {
    if constexpr (G == 1) {  // a thread's columns are its own sums
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = acc[i][e];
        if (lane + THREADS * i < nv) fin(i, lane + THREADS * i, t);
      }
      return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
      if (c < nv) store8<HMOE_DT_F32>(colsum, (int64_t)grp * a.d, 8 * c, acc[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = threadIdx.x + THREADS * i;
      if (c >= nv) continue;
      float t[8], q[8];
      load8<HMOE_DT_F32>(colsum, 0, 8 * c, t);
#pragma unroll
      for (int g = 1; g < G; ++g) {
        load8<HMOE_DT_F32>(colsum, (int64_t)g * a.d, 8 * c, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] += q[e];
      }
      fin(i, c, t);
    }
  };
  using VRaw = Raw8<OUT ? HMOE_DT_F32 : ST>;  // (the slots' sum stays fp32)
  auto load_rows = [&](int r, auto& ru, auto& rv, auto& rd) {
    r = min(r, a.s.T - 1);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const uint32_t col = 8 * min(lane + 64 * WPR * i, nv - 1);
      ru[i].load(a.u, (int64_t)r * a.d, col);
      if constexpr (!OUT) {
        rv[i].load(a.v, (int64_t)r * a.ldv, col);
        if (a.dres) rd[i].load(a.dres, (int64_t)r * a.d, col);
      }
    }
    if constexpr (OUT) {
      float t[VPL][8];
      load_slots<HT, VPL, WPR, KB>(a.v, a.inv_pos, a.add, a.k, a.d, r, lane, t);
#pragma unroll
      for (int i = 0; i < VPL; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) rv[i].w[e] = __float_as_uint(t[i][e]);
    }
  };
  float aacc[VPL][8], sacc[VPL][8], wm[VPL][8];
  // the parameters of sample b, and its sums from zero
  auto begin = [&](int b) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        aacc[i][e] = sacc[i][e] = 0.0f;
        wm[i][e] = 1.0f;
      }
      if (vec_in<VPL>(i, c, nv)) {
        float t[8];
        if (a.p.weight) load8_rt(a.p.weight, a.p.weight_dt, 0, 8 * c, wm[i]);
        if (a.p.scale) {
          load8_rt(a.p.scale, a.p.scale_dt, (int64_t)b * a.d, 8 * c, t);
#pragma unroll
          for (int e = 0; e < 8; ++e) wm[i][e] *= OUT ? t[e] : 1.0f + t[e];
        }
      }
    }
  };
  // one row of every row group (the row sums may hold a barrier: every wave comes here)
  auto one_row = [&](int r, bool row) {
    Raw8<UT> u[VPL];
    VRaw v[VPL];
    Raw8<ST> dr[OUT ? 1 : VPL];
    load_rows(r, u, v, dr);
    float sq = 0.0f, dot = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const bool in = vec_in<VPL>(i, lane + 64 * WPR * i, nv);
      u[i].keep(in);
      v[i].keep(in);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sq += v[i][e] * v[i][e];
        dot += u[i][e] * wm[i][e] * v[i][e];
      }
    }
    // (n = v r and mean(g n) before r again: r^3 and v r^3 would leave fp32's range for rows past 1e13 or rms below 1e-13)
    float rms = 1.0f, mean = 0.0f;  // mean(g n): dv = r (g - n mean)
    if (a.norm) {
      row_sum2<WPR>(sq, dot, red, half);
      rms = inv_rms(sq, a.d, a.eps);
      mean = dot * rms / (float)a.d;
    }
    if (!row) return;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = lane + 64 * WPR * i;
      if (!vec_in<VPL>(i, c, nv)) continue;
      float t[8];
      u[i].hold();
      v[i].hold();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float ue = u[i][e], n = v[i][e] * rms;
        aacc[i][e] += ue * n;
        if constexpr (!OUT) sacc[i][e] += ue;
        const float ge = ue * wm[i][e];
        t[e] = a.norm ? rms * (ge - n * mean) : ge;  // (without the norm the row, which may be inf or NaN, has no part)
      }
      if constexpr (!OUT)
        if (a.dres) {
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] += a.dres_scale * dr[i][e];
        }
      store8<DT>(a.dv, (int64_t)r * a.d, 8 * c, t);
    }
  };
  if constexpr (SHORT) {
    const int L = a.s.L, S = a.R / L;  // samples of this block
    float wsum[VPL][8];
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) wsum[i][e] = 0.0f;
    for (int s0 = 0; s0 < S; s0 += G) {
      const int b = blockIdx.x * S + s0 + grp;
      const bool on = s0 + grp < S && b < a.s.B;
      const int bc = min(b, a.s.B - 1);
      begin(bc);
      for (int l = 0; l < L; ++l) one_row(bc * L + l, on);
      if (!on) continue;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int c = lane + 64 * WPR * i;
        if (!vec_in<VPL>(i, c, nv)) continue;
        float q[8];
        if (a.dweight) {
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = OUT ? 1.0f : 0.0f;
          if (a.p.scale) load8_rt(a.p.scale, a.p.scale_dt, (int64_t)b * a.d, 8 * c, q);
#pragma unroll
          for (int e = 0; e < 8; ++e) wsum[i][e] += (OUT ? q[e] : 1.0f + q[e]) * aacc[i][e];
        }
        if (a.dscale) {
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = 1.0f;
          if (a.p.weight) load8_rt(a.p.weight, a.p.weight_dt, 0, 8 * c, q);
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] *= aacc[i][e];
          store8_rt(a.dscale, a.p.scale_dt, (int64_t)b * a.d, 8 * c, q);
        }
        if (!OUT && a.dshift) store8_rt(a.dshift, a.p.shift_dt, (int64_t)b * a.d, 8 * c, sacc[i]);
      }
    }
    if (a.dweight)
      over_groups(wsum, [&](int i, int, float (&t)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) wacc[i][e] = t[e];
      });
  } else {
    for (int r0 = r_begin; r0 < r_end;) {
      int end;
      const int b = sample_of(a.s, r0, end);
      const int piece_end = min(end, r_end);
      const bool live = b >= 0 && b < a.s.B;
      if (!live) {  // padding rows: no gradient from the norm
        for (int r = r0 + grp; r < piece_end; r += G)
          for (int c = lane; c < nv; c += 64 * WPR) {
            float t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = 0.0f;
            if (a.dres) {
              load8<ST>(a.dres, (int64_t)r * a.d, 8 * c, t);
#pragma unroll
              for (int e = 0; e < 8; ++e) t[e] *= a.dres_scale;
            }
            store8<DT>(a.dv, (int64_t)r * a.d, 8 * c, t);
          }
        r0 = piece_end;
        continue;
      }
      begin(b);
      for (int rg = r0; rg < piece_end; rg += G) one_row(rg + grp, rg + grp < piece_end);
      // (whole: this block holds every row of the sample)
      const int first = a.s.starts ? a.s.starts[b] : b * a.s.L;
      const bool whole = first >= r_begin && end <= r_end;
      float* slot = a.part + (2 * (int64_t)blockIdx.x + (first >= r_begin)) * nsum * a.d;
      if (a.dscale || a.dweight)
        over_groups(aacc, [&](int i, int c, float (&t)[8]) {
          float q[8];
          if (a.dweight) {  // A_b (1 + scale_b), or A_b gate_b
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = OUT ? 1.0f : 0.0f;
            if (a.p.scale) load8_rt(a.p.scale, a.p.scale_dt, (int64_t)b * a.d, 8 * c, q);
#pragma unroll
            for (int e = 0; e < 8; ++e) wacc[i][e] += (OUT ? q[e] : 1.0f + q[e]) * t[e];
          }
          if (!a.dscale) return;
          if (!whole) {
            store8<HMOE_DT_F32>(slot, 0, 8 * c, t);
            return;
          }
          if (a.p.weight) {
            load8_rt(a.p.weight, a.p.weight_dt, 0, 8 * c, q);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] *= q[e];
          }
          store8_rt(a.dscale, a.p.scale_dt, (int64_t)b * a.d, 8 * c, t);
        });
      if constexpr (!OUT) {
        if (a.dshift)
          over_groups(sacc, [&](int, int c, float (&t)[8]) {
            if (whole)
              store8_rt(a.dshift, a.p.shift_dt, (int64_t)b * a.d, 8 * c, t);
            else
              store8<HMOE_DT_F32>(slot, (int64_t)(nsum - 1) * a.d, 8 * c, t);
          });
      }
      r0 = piece_end;
    }
  }
  if (a.dweight) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = threadIdx.x + THREADS * i;
      if (c < nv) store8<HMOE_DT_F32>(a.wpart, (int64_t)blockIdx.x * a.d, 8 * c, wacc[i]);
    }
  }
}

// The column sums left in the workspace.  Workgroups walk the items: item b < B is sample b's sums, unless one chunk
// finished it (an empty sample gets zeros), item B the weight's over all chunks.  32 columns by SPLIT parts of the slots, each
// part reading every SPLIT-th with eight loads on their way, added in part order.
template <int SPLIT>
__global__ __launch_bounds__(32 * SPLIT) void norm_sums_kernel(NormBwdArgs a, int nchunk, int items) {
  __shared__ float lds[2][SPLIT][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, col = blockIdx.y * 32 + tx;
  const int nsum = (a.dscale != nullptr) + (a.dshift != nullptr);
  const bool in = col < a.d;
  auto put = [&](void* p, int dt, int64_t off, float v) {
    if (dt == HMOE_DT_F32)
      static_cast<float*>(p)[off] = v;
    else
      static_cast<uint16_t*>(p)[off] = (uint16_t)(dt == HMOE_DT_F16 ? cvt_h2(v, v) : cvt_bf2(v, v));
  };
  for (int b = blockIdx.x; b < items; b += gridDim.x) {
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
        continue;
    }
    const int64_t pitch = weight ? a.d : (int64_t)nsum * a.d;
    const float* src = weight ? a.wpart + col : a.part + col;
    const bool two = !weight && nsum == 2;
    auto slot = [&](int k) { return weight ? k : 2 * k + (k == c0); };
    float t0 = 0.0f, t1 = 0.0f;
    for (int c = c0 + ty; c <= c1; c += 8 * SPLIT) {
      float v[8], w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = c + i * SPLIT;
        const bool on = in && k <= c1;
        v[i] = on ? src[slot(k) * pitch] : 0.0f;
        w[i] = on && two ? src[slot(k) * pitch + a.d] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        t0 += v[i];
        t1 += w[i];
      }
    }
    __syncthreads();
    lds[0][ty][tx] = t0;
    lds[1][ty][tx] = t1;
    __syncthreads();
    if (ty != 0 || !in) continue;
#pragma unroll
    for (int i = 1; i < SPLIT; ++i) {
      t0 += lds[0][i][tx];
      t1 += lds[1][i][tx];
    }
    if (weight) {
      put(a.dweight, a.p.weight_dt, col, t0);
      continue;
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

// calls f(VPL, WPR) as integral constants for width d
template <class F>
static void by_width(int64_t d, F&& f) {
  const int64_t nv = d / 8;
#define HMOE_W(V, W) f(std::integral_constant<int, V>(), std::integral_constant<int, W>())
  if (nv <= 64) HMOE_W(1, 1);
  else if (nv <= 128) HMOE_W(2, 1);
  else if (nv <= 192) HMOE_W(3, 1);
  else if (nv <= 256) HMOE_W(2, 2);
  else if (nv <= 384) HMOE_W(3, 2);
  else if (nv <= 512) HMOE_W(2, 4);
  else if (nv <= 768) HMOE_W(3, 4);
  else if (nv <= 1024) HMOE_W(2, 8);
  else if (nv <= 1536) HMOE_W(3, 8);
  else HMOE_W(2, 16);
#undef HMOE_W
}

// row groups of a workgroup for width d
static int norm_groups(int64_t d) {
  int g = 0;
  by_width(d, [&](auto, auto w) { g = kNormGroups<decltype(w)::value>; });
  return g;
}

// calls f(KB) as an integral constant for k slots: how many are loaded at once, as far as the registers hold them
template <int HT, int WPR, class F>
static void by_slots_at_once(int k, F&& f) {
  if constexpr (WPR < 16) {
    if constexpr (HT != HMOE_DT_F32)
      if (k >= 4) return f(std::integral_constant<int, 4>());
    if (k >= 2) return f(std::integral_constant<int, 2>());
  }
  f(std::integral_constant<int, 1>());
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

// Rows per workgroup of the forward: a row for each of its row groups, or several (up to eight) where 16 waves on each of
// the 256 CUs have more than one.  16384 x 1536: 22 us (norm_in) and 41 us (norm_out, two slots) with workgroups of two
// waves, against 24 and 47 with four, 23 and 42 with eight; four rows a wave (16 waves a CU) against two or eight: within 5%.
static int fwd_rows(int64_t T, int64_t d) {
  int g = 1, wpr = 1;
  by_width(d, [&](auto, auto w) {
    g = kFwdGroups<decltype(w)::value>;
    wpr = decltype(w)::value;
  });
  const int64_t q = T * wpr / (256 * 16);
  return g * (int)(q < 1 ? 1 : q > 8 ? 8 : q);
}

// Rows per workgroup of the backward: what gives about 256 workgroups (one per CU: the registers of a row's sums leave room for
// eight waves), a multiple of the row groups.  16384 x 1536, norm_in: 256, 512 and 1024 workgroups 41, 47 and 60 us (all
// before the loads lost their predicates; with 256, 37 since); more of them also leave more column sums to write and add.
static int norm_rows(int64_t T, int groups) {
  int64_t r = (T + 255) / 256;
  r = (r + groups - 1) / groups * groups;
  return (int)(r > 0 ? r : groups);
}

// Whether the backward's row groups take whole samples (SHORT, equal samples only): where that leaves fewer steps one after the
// other.  A workgroup of R rows and G groups takes R / G batches of rows and R / L pieces, whose sums over the groups cost as
// much as six batches; SHORT takes L rows for each sample of a group.  16384 x 1536, norm_in, SHORT against the other, us: L = 1
// 158, 702; 2 85, 367; 4 60, 187; 8 47, 103; 16 44, 73; 32 68, 57; 64 121, 50.  4096 x 4096: 8 35, 71; 32 62, 56.  300 x 1536
// in 30 samples: 27, 21.
static bool norm_short(int64_t T, int64_t B, bool starts, int64_t R, int G) {
  if (starts || T == 0 || B < 2) return false;
  const int64_t L = T / B, pieces = R > L ? R / L : 1;
  return 6 * pieces + R / G > L * ((R + G * L - 1) / (G * L));
}

static size_t norm_bwd_ws(int64_t T, int64_t d, int64_t B, int nsum, bool weight) {
  if (T < 0 || d <= 0 || B < 1) return 0;
  const int64_t R = norm_rows(T, norm_groups(d)), nchunk = (T + R - 1) / R;
  return (size_t)(2 * nchunk * nsum + (weight ? nchunk : 0)) * (size_t)d * 4 + 16;
}

template <bool OUT>
static int norm_bwd_run(NormBwdArgs& a, int sdt, int hdt, void* workspace, size_t workspace_bytes, hipStream_t s) {
  const int nsum = (a.dscale != nullptr) + (a.dshift != nullptr);
  const int groups = norm_groups(a.d);
  // (SHORT: whole samples, and so never more workgroups than the other form has)
  a.R = norm_rows(a.s.T, groups);
  const bool brief = norm_short(a.s.T, a.s.B, a.s.starts != nullptr, a.R, groups);
  if (brief) a.R = (a.R + groups * a.s.L - 1) / (groups * a.s.L) * (groups * a.s.L);
  const int nchunk = (a.s.T + a.R - 1) / a.R;
  const bool final = nsum || a.dweight;
  if (final) {
    if (!workspace || workspace_bytes < norm_bwd_ws(a.s.T, a.d, a.s.B, nsum, a.dweight != nullptr))
      return HMOE_ERR_WORKSPACE;
    if (!al16(workspace)) return HMOE_ERR_ARG;
    a.part = static_cast<float*>(workspace);
    a.wpart = a.part + (int64_t)2 * nchunk * nsum * a.d;
  }
  if (nchunk) {
    const size_t lds = final && groups > 1 ? (size_t)groups * a.d * 4 : 0;  // at most 48 KB
    by_types(sdt, hdt, [&](auto st, auto ht) {
      by_width(a.d, [&](auto v, auto w) {
        constexpr int S = decltype(st)::value, H = decltype(ht)::value, V = decltype(v)::value, W = decltype(w)::value;
        auto launch = [&](auto kb) {
          constexpr int KB = decltype(kb)::value;
          if (brief)
            hipLaunchKernelGGL((norm_bwd_kernel<KB, S, H, V, W, true>), dim3(nchunk), dim3(kNormThreads<W>), lds, s, a);
          else
            hipLaunchKernelGGL((norm_bwd_kernel<KB, S, H, V, W, false>), dim3(nchunk), dim3(kNormThreads<W>), lds, s, a);
        };
        if constexpr (OUT)
          by_slots_at_once<H, W>(a.k, launch);
        else
          launch(std::integral_constant<int, 0>());
      });
    });
    HMOE_CHECK_LAUNCH();
  }
  if (final) {
    // (without sample sums to add, the weight's item comes first)
    NormBwdArgs f = a;
    if (!nsum || brief) f.s.B = 0;
    const int items = f.s.B + (a.dweight ? 1 : 0);
    if (items == 0) return HMOE_OK;
    // Up to 128 workgroups of a column block walk the items: with many samples most items are a chunk's own and left at once.
    // 128 against 1024, us: 16384 x 1536, 128 samples 15.2, 10.6; 1000 36, 40; 4000 97, 100; 16000 334, 326; 100000 x 64, 50000
    // samples 162, 53.
    const dim3 grid(items < 128 ? items : 128, (a.d + 31) / 32);
    // Many parts for long sums, few where the samples span a few chunks each.  32 against 8, us (256 chunks): 16384 x 1536, 1
    // sample 4.4, 6.4; 4 4.1, 5.1; 12 6.1, 5.5; 16 6.6, 5.6; 64 16.5, 7.8; 30000 x 512, 1 4.2, 6.2; 16 4.1, 5.1; 100 9.3, 5.8;
    // 4096 x 8192, 4 11.1, 7.5 (the side the rule does not take, as at 12 samples).
    if (nchunk > 16 * a.s.B)
      hipLaunchKernelGGL(norm_sums_kernel<32>, grid, dim3(32 * 32), 0, s, f, nchunk, items);
    else
      hipLaunchKernelGGL(norm_sums_kernel<8>, grid, dim3(32 * 8), 0, s, f, nchunk, items);
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
  const NormInArgs a = {x, ldx, h, p, {starts, (int)B, starts ? 0 : (int)(T / B), (int)T}, (int)d,
                        fwd_rows(T, d), eps};
  by_types(x_dtype, h_dtype, [&](auto st, auto ht) {
    by_width(d, [&](auto v, auto w) {
      constexpr int W = decltype(w)::value;
      hipLaunchKernelGGL((norm_in_kernel<decltype(st)::value, decltype(ht)::value, decltype(v)::value, W>),
                         dim3((unsigned)((T + a.R - 1) / a.R)), dim3(kFwdThreads<W>), 0,
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
                         k, norm, fwd_rows(T, d), eps, alpha};
  by_types(x_dtype, y_dtype, [&](auto st, auto ht) {
    by_width(d, [&](auto v, auto w) {
      constexpr int W = decltype(w)::value;
      by_slots_at_once<decltype(ht)::value, W>(k, [&](auto kb) {
        hipLaunchKernelGGL((norm_out_kernel<decltype(st)::value, decltype(ht)::value, decltype(v)::value, W,
                                            decltype(kb)::value>),
                           dim3((unsigned)((T + a.R - 1) / a.R)), dim3(kFwdThreads<W>), 0,
                           reinterpret_cast<hipStream_t>(stream), a);
      });
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
