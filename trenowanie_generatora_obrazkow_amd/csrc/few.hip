// A whole routed SwiGLU layer for a few tokens (up to 16) in two kernels.
//
//   few_up_kernel    the chosen experts' [g | u] = x Wgu (with up to 16 experts the softmax router as well)
//   few_down_kernel  act = silu(g) u, its product with Wd, the routing weights, the sum over the slots and an addend
//
// With so few tokens the layer is its chosen experts' weights read once, plus what a launch costs; the op-by-op form has five
// to seven dependent launches.  Here a workgroup of either kernel is one piece of one expert: a run of weight columns (one or
// two lines wide) and a part of the sum, so that many CUs stream weights however few experts were chosen.  Its four waves take
// steps of the sum in turn, weights straight from memory to registers with the next step's loads in flight (nothing is used
// twice, so nothing goes through the LDS), transposed there by byte permutes into fragments of the 16x16x32 matrix
// instruction, whose 16 columns are the expert's tokens.  The waves' sums meet in LDS, the parts of [g | u] in the second
// kernel's loads, the parts of the output in the workgroup that finishes a run of columns last: a counter, and no one waits.
//
// Measured, whole calls: one token with the router, 2 of 16 bf16 experts (d 1536, h 4096: 75 MB) 28.6 us (17.8 + 11.4); 16
// tokens over 51 of 64 8-bit experts (d 2048, h 1408: 441 MB) 105 to 109 us (64 + 40; 4.2 TB/s); seven over 9 fp16 experts (d
// 1000, h 712) 23 us (12 + 12); one over 8 int8 experts (d 2048, h 320) 19.7 us, the host's time (9 + 10).  Small ones are
// bound by a launch's steps one after another: start, grouping, the weights' latency, the sum over waves and parts.
//
// Numerics: fp32 sums throughout and one rounding, that of the output.  The activation enters its product as two bf16 numbers
// (16 significant bits; past bf16's largest number an infinity, as where a larger call rounds it), fp16 weights there as two as
// well (their 11 bits; an infinity, of either side, gives NaN); 8-bit experts (F8Stack) take x and the activation
// quantised as the grouped product does, widened exactly.
#include <algorithm>

#include "f8_common.h"
#include "route16.h"

namespace hmoe {

constexpr int kFewT = 16;                // tokens
constexpr int kFewK = 16;                // slots
constexpr int kFewM = kFewT * kFewK;     // routed rows
constexpr int kFewMaxS1 = 4, kFewMaxS2 = 16;
enum FewW { FW_BF16 = 0, FW_F16 = 1, FW_I8 = 2, FW_F8 = 3 };

// the first kernel leaves the grouping for the second
struct FewHead {
  int active;              // experts chosen
  int pad[3];
  int expert[kFewM], rows[kFewM], base[kFewM];  // each one's id, its routed rows, where they begin in `row`
  int row[kFewM];          // flat rows (token * k + slot), grouped by expert, in order
  int row16[kFewM][16];    // the first sixteen of each expert again, where they are found without `base`
  float w[kFewM];          // routing weights by flat row, 0 for an id that names no expert
  int flat_ok[kFewM];      // whether a flat row's id names an expert
};

struct FewParams {
  const uint16_t* x;
  int64_t ldx;
  int T, d, E, k, h, M;
  const void* ids;         // given routing
  int ids64;
  const void* tw;
  int tw_dt;
  const uint16_t* wr;      // or the router
  const float* bias;
  int renorm;
  float scaling;
  int32_t* out_ids;
  float* out_w;
  int32_t* n_invalid;
  const void *wgu, *wd;
  const void *s1, *s2;     // int8: scales per column; 8-bit floats: per block
  int s1_f32, s2_f32;
  const uint16_t* add;
  uint16_t* out;
  FewHead* head;
  unsigned* counter;       // one per column run of the output
  float *p1, *p2;          // (S1, M, 2, h), (S2, M, d)
  int S1, S2, runs1, runs2, per1, per2;  // parts, column runs, steps per part
};

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <bool F16>
__device__ __forceinline__ f32x4 few_mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// eight floats as bf16 pairs, and what they lose by it as bf16 pairs again; with INF, nothing where the first is infinite
// (so that an infinite number, or one past the largest bf16, stays an infinity instead of inf - inf)
template <bool INF>
__device__ __forceinline__ void split8(const float* v, u32x4& hi, u32x4& lo) {
  auto rest = [](float x, float h) { return !INF || __builtin_fabsf(h) < __builtin_inff() ? x - h : 0.0f; };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = cvt_bf2(v[2 * i], v[2 * i + 1]);
    lo[i] = cvt_bf2(rest(v[2 * i], bf_lo(hi[i])), rest(v[2 * i + 1], bf_hi(hi[i])));
  }
}

// Four weight columns of eight rows of k: 16 bytes of each row hold 8 (16-bit) or 16 (int8) columns; fragment j of a lane is
// its column j over the eight rows.
template <bool I8, bool F16>
__device__ __forceinline__ u32x4 few_column(const uint4 (&r)[8], int j) {
  u32x4 f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // rows 2 i, 2 i + 1
    const uint32_t a[4] = {r[2 * i].x, r[2 * i].y, r[2 * i].z, r[2 * i].w};
    const uint32_t b[4] = {r[2 * i + 1].x, r[2 * i + 1].y, r[2 * i + 1].z, r[2 * i + 1].w};
    if constexpr (I8) {
      const float p = (float)(int8_t)(a[j / 4] >> (8 * (j & 3))), q = (float)(int8_t)(b[j / 4] >> (8 * (j & 3)));
      f[i] = Elt<F16>::pack2(p, q);
    } else {
      f[i] = __builtin_amdgcn_perm(b[j / 2], a[j / 2], j & 1 ? 0x07060302u : 0x05040100u);
    }
  }
  return f;
}

// A lane's 32 values of a row's block of 128 (lanes l, l ^ 16, l ^ 32, l ^ 48 hold the block) quantised and widened again
__device__ __forceinline__ void f8_requant(const float (&v)[32], u32x4 (&f)[4]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = fmaxf(m, f8_abs(v[i]));
  m = bfly_max<32>(bfly_max<16>(m));
  const int e = f8_exp(m);
  const float inv = f8_inv(e), s = f8_pow(e);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    f[i] = f8_widen(make_uint2(f8_pack4(v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3], inv),
                               f8_pack4(v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7], inv)), s);
}

// ----------------------------------------------------------------------------------------------------------------
// Grouping: ids (flat rows, -1: none) -> the chosen experts in the order of their first rows, each with its rows in order
// ----------------------------------------------------------------------------------------------------------------
struct FewGroups {
  __attribute__((aligned(16))) int id[kFewM];
  int expert[kFewM], rows[kFewM], base[kFewM], row[kFewM];
  int wave_n[4], wave_rows[4];
};

__device__ __forceinline__ int few_group(FewGroups& g, int M) {
  const int i = threadIdx.x, lane = i & 63, wave = i >> 6;
  const int my = i < M ? g.id[i] : -1;
  int before = 0, all = 0, first = i;
  if (my >= 0) {
    for (int j = 0; j < M; j += 4) {  // (ids past M are -1)
      const int4 v = *reinterpret_cast<const int4*>(g.id + j);
      const int id[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bool same = id[t] == my;
        all += same;
        before += same && j + t < i;
        if (same) first = min(first, j + t);
      }
    }
  }
  const bool lead = my >= 0 && before == 0;
  const uint64_t leads = __ballot(lead);
  int n = lead ? all : 0;  // rows of the experts that begin up to here
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int o = __shfl_up(n, s, 64);
    if (lane >= s) n += o;
  }
  if (lane == 63) {
    g.wave_n[wave] = __builtin_popcountll(leads);
    g.wave_rows[wave] = n;
  }
  __syncthreads();
  int a = __builtin_popcountll(leads & ((1ull << lane) - 1)), b = n - (lead ? all : 0), total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) {
      a += g.wave_n[w];
      b += g.wave_rows[w];
    }
    total += g.wave_n[w];
  }
  if (lead) {
    g.expert[a] = my;
    g.rows[a] = all;
    g.base[a] = b;
    g.id[i] = -2 - b;  // (read back below: where the expert's rows begin)
  }
  __syncthreads();
  if (my >= 0) g.row[-2 - g.id[first] + before] = i;
  __syncthreads();
  return total;
}

// chain c of the router's logits of 16 tokens x 16 experts: the fixed order of hmoe_route_topk
__device__ __forceinline__ f32x4 few_router_chain(const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ wr,
                                                  int T, int d, int E, int lane, int c) {
#pragma clang fp contract(off)
  const int r = lane & 15, q = lane >> 4, nbf = d / 64;
  const uint16_t* xr = x + (int64_t)min(r, T - 1) * ldx + 16 * q;
  const uint16_t* wrow = wr + (int64_t)(r < E ? r : 0) * d + 16 * q;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  auto products = [&](const uint4 (&xv)[2], const uint4 (&wv)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t xw[4] = {xv[h].x, xv[h].y, xv[h].z, xv[h].w}, ww[4] = {wv[h].x, wv[h].y, wv[h].z, wv[h].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bf_lo(xw[i]), bf_lo(ww[i]), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bf_hi(xw[i]), bf_hi(ww[i]), acc, 0, 0, 0);
      }
    }
  };
  constexpr int PF = 8;  // blocks in flight
  for (int b0 = c; b0 < nbf; b0 += 4 * PF) {
    uint4 xs[PF][2], ws[PF][2];
#pragma unroll
    for (int p = 0; p < PF; ++p) {
      const int b = min(b0 + 4 * p, nbf - 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        xs[p][h] = *reinterpret_cast<const uint4*>(xr + 64 * b + 8 * h);
        ws[p][h] = *reinterpret_cast<const uint4*>(wrow + 64 * b + 8 * h);
      }
    }
#pragma unroll
    for (int p = 0; p < PF; ++p)
      if (b0 + 4 * p < nbf) products(xs[p], ws[p]);
  }
  if ((d & 63) && c == (nbf & 3)) {  // the partial block: -0 (x) and +0 (w) past d
    uint4 xv[2], wv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = 64 * nbf + 16 * q + 8 * h < d;
      const int off = in ? 64 * nbf + 8 * h : -16 * q;
      const uint4 xl = *reinterpret_cast<const uint4*>(xr + off), wl = *reinterpret_cast<const uint4*>(wrow + off);
      xv[h] = in ? xl : make_uint4(0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u);
      wv[h] = in ? wl : make_uint4(0, 0, 0, 0);
    }
    products(xv, wv);
  }
  return acc;
}

__device__ __forceinline__ float few_w(const void* w, int dt, int i) {
  if (dt == HMOE_DT_F32) return static_cast<const float*>(w)[i];
  const uint16_t h = static_cast<const uint16_t*>(w)[i];
  return dt == HMOE_DT_BF16 ? Elt<false>::one(h) : Elt<true>::one(h);
}

// ----------------------------------------------------------------------------------------------------------------
// [g | u] of one expert's rows over a run of columns and a part of d
// ----------------------------------------------------------------------------------------------------------------
// Fragments of a run and their columns.  Weights with columns side by side (16-bit, int8): a lane loads NC = 8 or 16 columns,
// lanes 0..7 of 16 gate ones and lanes 8..15 the same up ones, and its accumulator's element (j, v) is column
// 32 q + 8 v + j or 64 q + 16 v + j of the run's 16 NC (q = lane / 16).  8-bit floats (k side by side): fragments of 16 rows.
template <int W>
struct FewShape {
  static constexpr int NC = W == FW_I8 ? 16 : 8;
  static constexpr int FR = W == FW_F8 ? 4 : NC;             // accumulators of four
  static constexpr int COLS = W == FW_F8 ? 64 : 16 * NC;     // weight columns of a run
  static constexpr int STEP = W == FW_F8 ? 128 : 32;         // k per step
  static constexpr int RED = 4 * 16 * (COLS + 4) * 4;        // bytes of the waves' sums
  __device__ __forceinline__ static int col(int j, int v, int q) { return W == FW_F8 ? 16 * j + 4 * q + v : NC * (4 * q + v) + j; }
};

template <int W, bool F16, bool ROUTE>
__global__ __launch_bounds__(256, 1) void few_up_kernel(FewParams p) {
  using S = FewShape<W>;
  __shared__ FewGroups g;
  __shared__ float s_w[kFewM];
  extern __shared__ __attribute__((aligned(16))) float red[];  // [4][16][COLS + 4]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, q = lane >> 4;
  const int M = p.M;
  [[maybe_unused]] int chosen = -1;  // the router's id of flat row tid, as it goes out
  if constexpr (ROUTE) {
#pragma clang fp contract(off)
    const f32x4 acc = few_router_chain(p.x, p.ldx, p.wr, p.T, p.d, p.E, lane, wave);
#pragma unroll
    for (int i = 0; i < 4; ++i) red[wave * 256 + (4 * q + i) * 16 + l16] = acc[i];
    __syncthreads();
    const float* pt = red + (4 * wave + q) * 16 + l16;
    if (tid < kFewM) g.id[tid] = -1;
    __syncthreads();
    float lg[1] = {__fadd_rn(__fadd_rn(pt[0], pt[256]), __fadd_rn(pt[512], pt[768]))};
    if (p.bias && l16 < p.E) lg[0] = __fadd_rn(lg[0], p.bias[l16]);
    route_select16<1>(lg, 4 * wave, lane, p.T, p.E, p.k, p.renorm, p.scaling, nullptr, g.id, s_w);
    __syncthreads();
    // a token of NaN logits has the selection's empty mark in its later slots, which names no expert
    chosen = g.id[tid];
    g.id[tid] = chosen >= 0 && chosen < p.E ? chosen : -1;
    __syncthreads();
  } else {
    g.id[tid] = -1;
    if (tid < M) {
      const int64_t id = p.ids64 ? static_cast<const int64_t*>(p.ids)[tid] : (int64_t) static_cast<const int32_t*>(p.ids)[tid];
      g.id[tid] = id >= 0 && id < p.E ? (int)id : -1;
    }
    __syncthreads();
  }
  const int my = tid < M ? g.id[tid] : -1;  // (the grouping overwrites it)
  const int A = few_group(g, M);
  if (blockIdx.x == 0) {
    FewHead& h = *p.head;
    if (tid == 0) {
      h.active = A;
      if (p.n_invalid) *p.n_invalid = M - (A > 0 ? g.base[A - 1] + g.rows[A - 1] : 0);
    }
    if (tid < A) {
      h.expert[tid] = g.expert[tid];
      h.rows[tid] = g.rows[tid];
      h.base[tid] = g.base[tid];
    }
    if (tid < M) {
      if constexpr (ROUTE) {
        p.out_ids[tid] = chosen;
        p.out_w[tid] = s_w[tid];
      }
      h.w[tid] = ROUTE ? s_w[tid] : few_w(p.tw, p.tw_dt, tid);
      h.flat_ok[tid] = my >= 0;
      if (A > 0 && tid < g.base[A - 1] + g.rows[A - 1]) h.row[tid] = g.row[tid];
    }
    for (int i = tid; i < A * 16; i += 256) {
      const int x = i >> 4, r = i & 15;
      h.row16[x][r] = r < g.rows[x] ? g.row[g.base[x] + r] : 0;
    }
    for (int i = tid; i < p.runs2; i += 256) p.counter[i] = 0;
  }
  const int part = blockIdx.x % p.S1, run = blockIdx.x / p.S1 % p.runs1, a = blockIdx.x / (p.S1 * p.runs1);
  if (a >= A) return;
  const int e = g.expert[a], n = g.rows[a], base = g.base[a];
  const int steps = (p.d + S::STEP - 1) / S::STEP;
  const int k_end = min(steps, (part + 1) * p.per1);
  constexpr int HALF = S::COLS / 2;  // act columns of the run

  for (int r0 = 0; r0 < n; r0 += 16) {
    const int nr = min(16, n - r0);
    const bool has = l16 < nr;
    const uint16_t* px = p.x + (int64_t)(has ? g.row[base + r0 + l16] / p.k : 0) * p.ldx;
    f32x4 acc[S::FR];
#pragma unroll
    for (int j = 0; j < S::FR; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (W != FW_F8) {
      constexpr int ES = W == FW_I8 ? 1 : 2;
      const int ac = run * HALF + (l16 & 7) * S::NC;
      const bool cin = ac < p.h;
      const char* pw = static_cast<const char*>(p.wgu) + ((int64_t)e * p.d * 2 * p.h + (l16 >> 3) * p.h + ac) * ES;
      uint4 w[8], xv;
      auto load = [&](int st) __attribute__((always_inline)) {
        const int k = st * 32 + q * 8;
        const bool in = k < p.d;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = in && cin ? *reinterpret_cast<const uint4*>(pw + (int64_t)(k + i) * 2 * p.h * ES) : make_uint4(0, 0, 0, 0);
        xv = in && has ? *reinterpret_cast<const uint4*>(px + k) : make_uint4(0, 0, 0, 0);
      };
      int st = part * p.per1 + wave;
      if (st < k_end) load(st);
      for (; st < k_end; st += 4) {
        uint4 c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = w[i];
        const u32x4 xf = {xv.x, xv.y, xv.z, xv.w};
        if (st + 4 < k_end) load(st + 4);
#pragma unroll
        for (int j = 0; j < S::FR; ++j) acc[j] = few_mfma<F16>(few_column<W == FW_I8, F16>(c, j), xf, acc[j]);
      }
    } else {
      // rows of the stack: fragments 0, 1 gate, 2, 3 up; the lane's 32 values of k of each
      const uint8_t* pw[4];
      const uint8_t* ps[4];
      bool cin[4];
      const int nbs = (p.h + kF8Block - 1) / kF8Block;
      const int64_t lds = (p.d + 2047) / 2048 * 16;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ac = run * HALF + (j & 1) * 16 + l16;
        cin[j] = ac < p.h;
        pw[j] = static_cast<const uint8_t*>(p.wgu) + ((int64_t)e * 2 * p.h + (j >> 1) * p.h + min(ac, p.h - 1)) * p.d;
        ps[j] = static_cast<const uint8_t*>(p.s1) +
                ((int64_t)(e * 2 + (j >> 1)) * nbs + min(run * HALF + (j & 1) * 16, p.h - 1) / kF8Block) * lds;
      }
      uint4 w[4][2], xv[4];
      uint8_t sb[4];
      auto load = [&](int st) __attribute__((always_inline)) {
        const int k = st * 128 + q * 32;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            w[j][i] = cin[j] && k + 16 * i < p.d ? *reinterpret_cast<const uint4*>(pw[j] + k + 16 * i) : make_uint4(0, 0, 0, 0);
          sb[j] = ps[j][st];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          xv[i] = has && k + 8 * i < p.d ? *reinterpret_cast<const uint4*>(px + k + 8 * i) : make_uint4(0, 0, 0, 0);
      };
      int st = part * p.per1 + wave;
      if (st < k_end) load(st);
      for (; st < k_end; st += 4) {
        uint4 c[4][2];
        float sc[4], v[32];
        using X = Elt<F16>;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[j][0] = w[j][0];
          c[j][1] = w[j][1];
          sc[j] = f8_pow((int)sb[j] - 127);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u[4] = {xv[i].x, xv[i].y, xv[i].z, xv[i].w};
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            v[8 * i + 2 * t] = X::lo(u[t]);
            v[8 * i + 2 * t + 1] = X::hi(u[t]);
          }
        }
        if (st + 4 < k_end) load(st + 4);
        u32x4 xf[4];
        f8_requant(v, xf);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint2 b[4] = {make_uint2(c[j][0].x, c[j][0].y), make_uint2(c[j][0].z, c[j][0].w),
                              make_uint2(c[j][1].x, c[j][1].y), make_uint2(c[j][1].z, c[j][1].w)};
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j] = few_mfma<false>(f8_widen(b[i], sc[j]), xf[i], acc[j]);
        }
      }
    }
    // the waves' sums
    constexpr int LD = S::COLS + 4;
    if (r0 > 0 || ROUTE) __syncthreads();  // (the last chunk's, or the router's, reads of `red`)
    if (has) {
#pragma unroll
      for (int j = 0; j < S::FR; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) red[(wave * 16 + l16) * LD + S::col(j, v, q)] = acc[j][v];
    }
    __syncthreads();
    for (int i = tid; i < nr * S::COLS; i += 256) {
      const int r = i / S::COLS, c = i - r * S::COLS, up = c >= HALF, col = run * HALF + c - up * HALF;
      if (col >= p.h) continue;
      float v = (red[r * LD + c] + red[(16 + r) * LD + c]) + (red[(32 + r) * LD + c] + red[(48 + r) * LD + c]);
      if constexpr (W == FW_I8) {
        const int64_t at = (int64_t)e * 2 * p.h + up * p.h + col;
        v *= p.s1_f32 ? static_cast<const float*>(p.s1)[at] : Elt<false>::one(static_cast<const uint16_t*>(p.s1)[at]);
      }
      p.p1[(((int64_t)part * M + g.row[base + r0 + r]) * 2 + up) * p.h + col] = v;
    }
  }
}

// ----------------------------------------------------------------------------------------------------------------
// The output's columns of one expert's rows over a part of h; the last workgroup of a run of columns sums up
// ----------------------------------------------------------------------------------------------------------------
// The parts of the output pass between workgroups of one launch, on XCDs with an L2 each.  They are written and read as
// agent-scope atomics: these go through to memory and are read from there, so no workgroup has to write a whole L2 back or
// discard it (a release and an acquire fence per workgroup: 185 us instead of 40 for 16 tokens over 51 experts).
__device__ __forceinline__ void put_agent(float* p, float a, float b) {
  const uint64_t v = (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get_agent(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// act = silu(g) u of a chunk of kFewChunk columns of up to 16 rows, in LDS rows of kFewActLd numbers: the workgroup adds the parts
// of [g | u] once, eight columns a thread, all loads of a thread in flight together.  16-bit and int8 experts read it as two
// bf16 numbers; 8-bit floats as the one that Q(act) is (16 threads hold a block of 128).
constexpr int kFewChunk = 512, kFewActLd = kFewChunk + 8;
template <int S1, bool F8>
__device__ __forceinline__ void few_act(const float* __restrict__ p1, int64_t part_stride, const int* rows, int nr, int h, int k0,
                                        int k1, uint16_t* hi, uint16_t* lo) {
  const int pieces = (k1 - k0 + 7) / 8, all = F8 ? (pieces + 15) & ~15 : pieces;  // (whole blocks)
  for (int i = threadIdx.x; i < nr * all; i += 256) {
    const int r = i / all, c = (i - r * all) * 8, k = k0 + c;
    float4 x[S1][4];
    const float* pg = p1 + (int64_t)rows[r] * 2 * h + k;
    const bool in = k < h && c < k1 - k0;
#pragma unroll
    for (int s = 0; s < S1; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[s][j] = in ? *reinterpret_cast<const float4*>(pg + s * part_stride + (j >> 1) * h + (j & 1) * 4)
                     : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 1; s < S1; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[0][j].x += x[s][j].x; x[0][j].y += x[s][j].y; x[0][j].z += x[s][j].z; x[0][j].w += x[s][j].w;
      }
    float v[8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      v[4 * j] = silu_f(x[0][j].x) * x[0][j + 2].x;
      v[4 * j + 1] = silu_f(x[0][j].y) * x[0][j + 2].y;
      v[4 * j + 2] = silu_f(x[0][j].z) * x[0][j + 2].z;
      v[4 * j + 3] = silu_f(x[0][j].w) * x[0][j + 2].w;
    }
    u32x4 a, b;
    if constexpr (F8) {
      float m = 0.0f;
#pragma unroll
      for (int t = 0; t < 8; ++t) m = fmaxf(m, f8_abs(v[t]));
      m = bfly_max<8>(bfly_max<4>(bfly_max<2>(bfly_max<1>(m))));
      const int e = f8_exp(m);
      const float inv = f8_inv(e);
      a = f8_widen(make_uint2(f8_pack4(v[0], v[1], v[2], v[3], inv), f8_pack4(v[4], v[5], v[6], v[7], inv)), f8_pow(e));
    } else {
      split8<true>(v, a, b);
      *reinterpret_cast<u32x4*>(lo + r * kFewActLd + c) = b;
    }
    *reinterpret_cast<u32x4*>(hi + r * kFewActLd + c) = a;
  }
}

template <int W, bool F16>
__global__ __launch_bounds__(256, 1) void few_down_kernel(FewParams p) {
  using S = FewShape<W>;
  extern __shared__ __attribute__((aligned(16))) float red[];
  __shared__ __attribute__((aligned(16))) uint16_t s_hi[16 * kFewActLd], s_lo[W == FW_F8 ? 8 : 16 * kFewActLd];
  __shared__ int s_row[16];
  __shared__ float s_w[kFewM];
  __shared__ int s_ok[kFewM], s_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, q = lane >> 4;
  const int M = p.M;
  const FewHead& hd = *p.head;
  const int part = blockIdx.x % p.S2, run = blockIdx.x / p.S2 % p.runs2, a = blockIdx.x / (p.S2 * p.runs2);
  const int A = hd.active, e = hd.expert[a], n = hd.rows[a], base = hd.base[a];
  const int row16 = hd.row16[a][l16];  // (these loads are all under way together)
  if (tid < M) {
    s_w[tid] = hd.w[tid];
    s_ok[tid] = hd.flat_ok[tid];
  }
  if (a >= A && !(A == 0 && a == 0 && part == 0)) return;
  const int steps = (p.h + S::STEP - 1) / S::STEP;
  const int k_begin = part * p.per2, k_end = min(steps, (part + 1) * p.per2);
  constexpr int CS = kFewChunk / S::STEP;  // steps per chunk of act
  if (A > 0) {
    for (int r0 = 0; r0 < n; r0 += 16) {
      const int nr = min(16, n - r0);
      const bool has = l16 < nr;
      if (r0 > 0) __syncthreads();
      if (tid < 16) s_row[tid] = r0 == 0 ? row16 : hd.row[base + r0 + min(tid, nr - 1)];
      __syncthreads();
      f32x4 acc[S::FR];
#pragma unroll
      for (int j = 0; j < S::FR; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      // the weights of a step: 8 loads of 16 bytes a lane
      uint4 w[8];
      [[maybe_unused]] uint8_t sb[4];
      constexpr int ES = W == FW_I8 ? 1 : 2;
      const int col0 = run * S::COLS + l16 * S::NC;
      [[maybe_unused]] const char* pw16 = static_cast<const char*>(p.wd) + ((int64_t)e * p.h * p.d + col0) * ES;
      [[maybe_unused]] const uint8_t* pw8[4];
      [[maybe_unused]] const uint8_t* ps[4];
      if constexpr (W == FW_F8) {
        const int nbs = (p.d + kF8Block - 1) / kF8Block;
        const int64_t lds = (p.h + 2047) / 2048 * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pw8[j] = static_cast<const uint8_t*>(p.wd) + ((int64_t)e * p.d + min(run * S::COLS + j * 16 + l16, p.d - 1)) * p.h;
          ps[j] = static_cast<const uint8_t*>(p.s2) + ((int64_t)e * nbs + min(run * S::COLS + j * 16, p.d - 1) / kF8Block) * lds;
        }
      }
      auto load = [&](int st) __attribute__((always_inline)) {
        if constexpr (W != FW_F8) {
          const int k = st * 32 + q * 8;
          const bool in = k < p.h && col0 < p.d;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            w[i] = in ? *reinterpret_cast<const uint4*>(pw16 + (int64_t)(k + i) * p.d * ES) : make_uint4(0, 0, 0, 0);
        } else {
          const int k = st * 128 + q * 32;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool cin = run * S::COLS + j * 16 + l16 < p.d;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              w[2 * j + i] = cin && k + 16 * i < p.h ? *reinterpret_cast<const uint4*>(pw8[j] + k + 16 * i) : make_uint4(0, 0, 0, 0);
            sb[j] = ps[j][st];
          }
        }
      };
      if (k_begin + wave < k_end) load(k_begin + wave);
      for (int c0 = k_begin; c0 < k_end; c0 += CS) {
        const int c1 = min(k_end, c0 + CS);
        if (c0 > k_begin) __syncthreads();  // the last chunk has been read
        const int64_t ps1 = (int64_t)M * 2 * p.h;
        const int ka = c0 * S::STEP, kb = min(p.h, c1 * S::STEP);
        switch (p.S1) {
          case 1: few_act<1, W == FW_F8>(p.p1, ps1, s_row, nr, p.h, ka, kb, s_hi, s_lo); break;
          case 2: few_act<2, W == FW_F8>(p.p1, ps1, s_row, nr, p.h, ka, kb, s_hi, s_lo); break;
          case 3: few_act<3, W == FW_F8>(p.p1, ps1, s_row, nr, p.h, ka, kb, s_hi, s_lo); break;
          default: few_act<4, W == FW_F8>(p.p1, ps1, s_row, nr, p.h, ka, kb, s_hi, s_lo); break;
        }
        __syncthreads();
        // steps wave, wave + 4, ... of the part (a chunk is a multiple of four steps)
        for (int st = c0 + wave; st < c1; st += 4) {
          uint4 c[8];
          [[maybe_unused]] float sc[4];
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i] = w[i];
          if constexpr (W == FW_F8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[j] = f8_pow((int)sb[j] - 127);
          }
          if (st + 4 < k_end) load(st + 4);
          const u32x4 zero = {0, 0, 0, 0};
          if constexpr (W != FW_F8) {
            const int at = l16 * kFewActLd + (st - c0) * 32 + q * 8;
            const bool on = has && st * 32 + q * 8 < p.h;
            const u32x4 hi = on ? *reinterpret_cast<const u32x4*>(s_hi + at) : zero;
            const u32x4 lo = on ? *reinterpret_cast<const u32x4*>(s_lo + at) : zero;
#pragma unroll
            for (int j = 0; j < S::FR; ++j) {
              if constexpr (W == FW_F16) {  // the weights' 11 bits as two bf16 numbers
                const u32x4 v = few_column<false, true>(c, j);
                float f[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  f[2 * i] = h_lo(v[i]);
                  f[2 * i + 1] = h_hi(v[i]);
                }
                u32x4 wh, wl;
                split8<false>(f, wh, wl);
                acc[j] = few_mfma<false>(wl, hi, acc[j]);
                acc[j] = few_mfma<false>(wh, lo, acc[j]);
                acc[j] = few_mfma<false>(wh, hi, acc[j]);
              } else {
                const u32x4 v = few_column<W == FW_I8, false>(c, j);
                acc[j] = few_mfma<false>(v, lo, acc[j]);
                acc[j] = few_mfma<false>(v, hi, acc[j]);
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const u32x4 xf = has && st * 128 + q * 32 + 8 * i < p.h
                                   ? *reinterpret_cast<const u32x4*>(s_hi + l16 * kFewActLd + (st - c0) * 128 + q * 32 + 8 * i)
                                   : zero;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint4 v = c[2 * j + (i >> 1)];
                acc[j] = few_mfma<false>(f8_widen(i & 1 ? make_uint2(v.z, v.w) : make_uint2(v.x, v.y), sc[j]), xf, acc[j]);
              }
            }
          }
        }
      }
      constexpr int LD = S::COLS + 4;
      if (has) {
#pragma unroll
        for (int j = 0; j < S::FR; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) red[(wave * 16 + l16) * LD + S::col(j, v, q)] = acc[j][v];
      }
      __syncthreads();
      for (int i = tid; i < nr * (S::COLS / 2); i += 256) {
        const int r = i / (S::COLS / 2), c = (i - r * (S::COLS / 2)) * 2, col = run * S::COLS + c;
        if (col >= p.d) continue;
        float v[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          v[t] = (red[r * LD + c + t] + red[(16 + r) * LD + c + t]) + (red[(32 + r) * LD + c + t] + red[(48 + r) * LD + c + t]);
          if constexpr (W == FW_I8) {
            const int64_t at = (int64_t)e * p.d + col + t;
            v[t] *= p.s2_f32 ? static_cast<const float*>(p.s2)[at] : Elt<false>::one(static_cast<const uint16_t*>(p.s2)[at]);
          }
        }
        put_agent(p.p2 + ((int64_t)part * M + s_row[r]) * p.d + col, v[0], v[1]);
      }
    }
    // every thread's sums are in memory before the workgroup counts itself; the last of the run's A * S2 has all before it
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    __syncthreads();
    if (tid == 0)
      s_last = __hip_atomic_fetch_add(p.counter + run, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(A * p.S2 - 1);
    __syncthreads();
    if (!s_last) return;
    asm volatile("" ::: "memory");
  } else {
    __syncthreads();
  }
  // the run's columns of every token, two a thread: the terms (slot, part) are dealt to G groups of threads where there are
  // fewer columns than threads, each with eight loads in flight, and the groups' sums added in LDS, always in the same order
  using X = Elt<F16>;
  const int items = p.T * (S::COLS / 2);
  const int G = items * 4 <= 256 ? 4 : items * 2 <= 256 ? 2 : 1;
  const int terms = A > 0 ? p.k * p.S2 : 0;
  float2* s_sum = reinterpret_cast<float2*>(red);
  for (int i0 = 0; i0 < items * G; i0 += 256) {
    const int i = (i0 + tid) % items, grp = (i0 + tid) / items;
    const int t = i / (S::COLS / 2), col = run * S::COLS + (i - t * (S::COLS / 2)) * 2;
    const bool on = i0 + tid < items * G && col < p.d;
    float o0 = 0.0f, o1 = 0.0f;
    if (on) {
      for (int t0 = grp; t0 < terms; t0 += 8 * G) {
        float2 v[8];
        float wv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int term = t0 + j * G, s = term / p.S2, f = t * p.k + s;
          const bool ok = term < terms && s_ok[f];
          v[j] = ok ? get_agent(p.p2 + ((int64_t)(term - s * p.S2) * M + f) * p.d + col) : make_float2(0.0f, 0.0f);
          wv[j] = ok ? s_w[f] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o0 = __builtin_fmaf(wv[j], v[j].x, o0);
          o1 = __builtin_fmaf(wv[j], v[j].y, o1);
        }
      }
    }
    if (G > 1) {  // (one round: items * G <= 256)
      s_sum[tid] = make_float2(o0, o1);
      __syncthreads();
      for (int j = 1; j < G; ++j) {
        if (grp == 0 && on) {
          o0 += s_sum[tid + j * items].x;
          o1 += s_sum[tid + j * items].y;
        }
      }
    }
    if (on && grp == 0) {
      if (p.add) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p.add + (int64_t)t * p.d + col);
        o0 += X::lo(w);
        o1 += X::hi(w);
      }
      *reinterpret_cast<uint32_t*>(p.out + (int64_t)t * p.d + col) = X::pack2(o0, o1);
    }
  }
}

// ----------------------------------------------------------------------------------------------------------------
// Host
// ----------------------------------------------------------------------------------------------------------------
struct FewPlan {
  int S1, S2, runs1, runs2, per1, per2;
  size_t head, counter, p1, p2, total;
};

// How the work is cut: column runs of fixed width; the sums in parts until there is about one workgroup per CU in the first
// kernel and one for every other CU in the second (were every chosen expert another one), at least four steps to a part (one for
// each wave).  More parts cost more than they bring: with 512, 256 and 128 workgroups wanted one bf16 token over 2 experts of
// d 1536, h 4096 took 20.4, 17.6 and 20.4 us (with the router, which every workgroup runs) and 12.2, 11.4 and 11.4, seven fp16
// tokens over 9 experts of d 1000, h 712 11.4, 12.4 and 12.7 and 19.5, 15.8 and 11.9 (its last workgroups add 18, 12 and 6 parts).
// The rule counts workgroups and not bytes, and large layers would take more of them.  Whole calls, the weights from memory, with
// 256 and 128 wanted (these), 256 and 256, 256 and 512, 512 and 128, 128 and 128:
//   bf16  4 experts of 2304 x 4096, k 2, one token  35.4, 33.3, 37.3, 35.8, 45.8 us;  16 tokens  72.0, 64.2, 71.7, 74.1, 71.9
//         8 of 4096 x 8192, k 2, one token  104, 89, 88, 101, 104;  8 of 1024 x 2816, k 2, four tokens  36.5, 31.1, 31.0, 34.1, 36.3
//         16 of 1536 x 4096, k 2, 16 tokens  136, 124, 131, 136, 136;  64 of 1280 x 256, k 8, one and eight tokens  the same but for
//         34.8 -> 31.2 with 512 and 128 at eight
//   fp16  the 2304 x 4096 and 1024 x 2816 ones within 5% of bf16;  32 of 1536 x 768, k 4, 16 tokens  57.2, 57.2, 61.1, 56.3, 57.1
//   int8  32 of 1536 x 768, k 4, two tokens  19.8, 22.6, 22.6, 19.7, 20.0;  8 of 2560 x 6912, k 2, 16 tokens  109, 115, 123, 114,
//         109;  8 of 4096 x 8192, k 2, one token  65, 57, 60, 63, 82
//   8-bit floats  8 of 4096 x 8192, k 2, one token  81, 64, 57, 81, 81, eight tokens 170 each;  16 of 2048 x 1024, k 4, one token
//         18.7, 17.3, 17.2, 19.5, 20.9
static bool few_plan(int64_t T, int64_t d, int E, int k, int64_t h, int w, FewPlan& P) {
  if (T < 1 || T > kFewT || k < 1 || k > kFewK || E < 1 || d < 1 || h < 1 || d > (1 << 24) || h > (1 << 24)) return false;
  const int cols = w == FW_F8 ? 64 : w == FW_I8 ? 256 : 128, step = w == FW_F8 ? 128 : 32;
  const int64_t M = T * k, chosen = std::min<int64_t>(E, M);
  P.runs1 = (int)((h + cols / 2 - 1) / (cols / 2));
  P.runs2 = (int)((d + cols - 1) / cols);
  auto cut = [&](int64_t wanted, int64_t pieces, int64_t len, int most, int& parts, int& per) {
    const int64_t steps = (len + step - 1) / step;
    int64_t s = std::min<int64_t>({(wanted + pieces - 1) / pieces, most, (steps + 3) / 4});
    s = std::max<int64_t>(s, 1);
    per = (int)((steps + s - 1) / s);
    parts = (int)((steps + per - 1) / per);
  };
  cut(256, chosen * P.runs1, d, kFewMaxS1, P.S1, P.per1);
  cut(128, chosen * P.runs2, h, kFewMaxS2, P.S2, P.per2);
  size_t o = 0;
  auto take = [&](size_t n) {
    const size_t at = o;
    o += (n + 255) & ~(size_t)255;
    return at;
  };
  P.head = take(sizeof(FewHead));
  P.counter = take((size_t)P.runs2 * 4);
  P.p1 = take((size_t)P.S1 * M * 2 * h * 4);
  P.p2 = take((size_t)P.S2 * M * d * 4);
  P.total = o;
  return true;
}

static int few_type(int w_dtype, int dtype) {
  if (w_dtype == HMOE_DT_I8) return FW_I8;
  if (w_dtype == HMOE_DT_F8) return FW_F8;
  if (w_dtype == HMOE_DT_BF16 && dtype == HMOE_DT_BF16) return FW_BF16;
  if (w_dtype == HMOE_DT_F16 && dtype == HMOE_DT_F16) return FW_F16;
  return -1;
}

template <int W, bool F16>
static int few_launch(const FewParams& p, hipStream_t s) {
  const unsigned chosen = (unsigned)std::min(p.E, p.M);
  const size_t lds = FewShape<W>::RED;
  static_assert(FewShape<W>::RED + 2 * 16 * kFewActLd * 2 + 8 * kFewM <= 150 * 1024 && FewShape<W>::RED >= 4096, "LDS");
  auto big = [&](const void* f) {  // (beyond what a kernel gets unasked)
    return lds <= 16 * 1024 || hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) == hipSuccess;
  };
  const dim3 g1(chosen * (unsigned)(p.runs1 * p.S1)), g2(chosen * (unsigned)(p.runs2 * p.S2));
  if (p.wr) {
    if constexpr (W == FW_BF16) {
      auto k1 = few_up_kernel<W, F16, true>;
      if (!big(reinterpret_cast<const void*>(k1))) return HMOE_ERR_LAUNCH;
      hipLaunchKernelGGL(k1, g1, dim3(256), lds, s, p);
    } else {
      return HMOE_ERR_DTYPE;
    }
  } else {
    auto k1 = few_up_kernel<W, F16, false>;
    if (!big(reinterpret_cast<const void*>(k1))) return HMOE_ERR_LAUNCH;
    hipLaunchKernelGGL(k1, g1, dim3(256), lds, s, p);
  }
  HMOE_CHECK_LAUNCH();
  auto k2 = few_down_kernel<W, F16>;
  if (!big(reinterpret_cast<const void*>(k2))) return HMOE_ERR_LAUNCH;
  hipLaunchKernelGGL(k2, g2, dim3(256), lds, s, p);
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

static bool few_mis(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

static int few_check(const void* x, int64_t ldx, int dtype, const void* wgu, const void* wgu_s, int wgu_s_dtype, const void* wd,
                     const void* wd_s, int wd_s_dtype, int w_dtype, int64_t T, int64_t d, int E, int k, int64_t h,
                     const void* add, const void* out, const void* ws, size_t ws_bytes, FewPlan& P, int& w) {
  if (T < 0 || d <= 0 || E <= 0 || k <= 0 || h <= 0) return HMOE_ERR_ARG;
  if (dtype != HMOE_DT_BF16 && dtype != HMOE_DT_F16) return HMOE_ERR_DTYPE;
  w = few_type(w_dtype, dtype);
  if (w < 0) return HMOE_ERR_DTYPE;
  const bool scaled = w == FW_I8 || w == FW_F8;
  if (scaled != (wgu_s != nullptr) || scaled != (wd_s != nullptr)) return HMOE_ERR_ARG;
  if (w == FW_I8 && ((wgu_s_dtype != HMOE_DT_BF16 && wgu_s_dtype != HMOE_DT_F32) ||
                     (wd_s_dtype != HMOE_DT_BF16 && wd_s_dtype != HMOE_DT_F32)))
    return HMOE_ERR_DTYPE;
  const int gr = scaled ? 16 : 8;
  if (d % gr || h % gr || E > 1024 || T > kFewT || k > kFewK || d > (1 << 24) || h > (1 << 24)) return HMOE_ERR_SHAPE;
  if (T == 0) return HMOE_OK;
  if (!few_plan(T, d, E, k, h, w, P)) return HMOE_ERR_SHAPE;
  if ((int64_t)std::min<int64_t>(E, T * k) * std::max(P.runs1 * P.S1, P.runs2 * P.S2) >= (1 << 23)) return HMOE_ERR_SHAPE;
  if (!x || !wgu || !wd || !out || ldx < d || ldx % 8) return HMOE_ERR_ARG;
  if (few_mis(x, 16) || few_mis(wgu, 16) || few_mis(wd, 16) || few_mis(out, 16) || few_mis(add, 16) || few_mis(wgu_s, 4) ||
      few_mis(wd_s, 4))
    return HMOE_ERR_ARG;
  if (!ws || ws_bytes < P.total || few_mis(ws, 256)) return HMOE_ERR_WORKSPACE;
  return HMOE_OK;
}

static int few_run(FewParams p, const FewPlan& P, int w, int dtype, void* ws, hipStream_t s) {
  char* b = static_cast<char*>(ws);
  p.head = reinterpret_cast<FewHead*>(b + P.head);
  p.counter = reinterpret_cast<unsigned*>(b + P.counter);
  p.p1 = reinterpret_cast<float*>(b + P.p1);
  p.p2 = reinterpret_cast<float*>(b + P.p2);
  p.S1 = P.S1; p.S2 = P.S2; p.runs1 = P.runs1; p.runs2 = P.runs2; p.per1 = P.per1; p.per2 = P.per2;
  const bool f16 = dtype == HMOE_DT_F16;
  switch (w) {
    case FW_BF16: return few_launch<FW_BF16, false>(p, s);
    case FW_F16: return few_launch<FW_F16, true>(p, s);
    case FW_I8: return f16 ? few_launch<FW_I8, true>(p, s) : few_launch<FW_I8, false>(p, s);
    default: return f16 ? few_launch<FW_F8, true>(p, s) : few_launch<FW_F8, false>(p, s);
  }
}

}  // namespace hmoe

using namespace hmoe;

extern "C" {

size_t hmoe_few_workspace_size(int64_t T, int64_t d, int E, int k, int64_t h, int w_dtype, int dtype) {
  FewPlan P;
  const int w = few_type(w_dtype, dtype);
  return w >= 0 && few_plan(T, d, E, k, h, w, P) ? P.total : 0;
}

int hmoe_few_experts(const void* x, int64_t ldx, int dtype, const void* topk_ids, int ids_dtype, const void* topk_w,
                     int topk_w_dtype, const void* wgu, const void* wgu_s, int wgu_s_dtype, const void* wd, const void* wd_s,
                     int wd_s_dtype, int w_dtype, int64_t T, int64_t d, int E, int k, int64_t h, const void* add, void* out,
                     int32_t* n_invalid, void* workspace, size_t workspace_bytes, hmoe_stream_t stream) {
  FewPlan P;
  int w = 0;
  int rc = few_check(x, ldx, dtype, wgu, wgu_s, wgu_s_dtype, wd, wd_s, wd_s_dtype, w_dtype, T, d, E, k, h, add, out, workspace,
                     workspace_bytes, P, w);
  if (rc || T == 0) return rc;
  if (!topk_ids || !topk_w) return HMOE_ERR_ARG;
  if (ids_dtype != HMOE_DT_I32 && ids_dtype != HMOE_DT_I64) return HMOE_ERR_DTYPE;
  if (topk_w_dtype != HMOE_DT_F32 && topk_w_dtype != HMOE_DT_BF16 && topk_w_dtype != HMOE_DT_F16) return HMOE_ERR_DTYPE;
  FewParams p = {};
  p.x = static_cast<const uint16_t*>(x);
  p.ldx = ldx;
  p.T = (int)T; p.d = (int)d; p.E = E; p.k = k; p.h = (int)h; p.M = (int)T * k;
  p.ids = topk_ids;
  p.ids64 = ids_dtype == HMOE_DT_I64;
  p.tw = topk_w;
  p.tw_dt = topk_w_dtype;
  p.n_invalid = n_invalid;
  p.wgu = wgu; p.wd = wd; p.s1 = wgu_s; p.s2 = wd_s;
  p.s1_f32 = wgu_s_dtype == HMOE_DT_F32;
  p.s2_f32 = wd_s_dtype == HMOE_DT_F32;
  p.add = static_cast<const uint16_t*>(add);
  p.out = static_cast<uint16_t*>(out);
  return few_run(p, P, w, dtype, workspace, reinterpret_cast<hipStream_t>(stream));
}

int hmoe_few_forward(const void* x, int64_t ldx, const void* wr, const float* bias, const void* wgu, const void* wd, int64_t T,
                     int64_t d, int E, int k, int64_t h, int renorm, float scaling, const void* add, void* out,
                     int32_t* topk_ids, float* topk_w, void* workspace, size_t workspace_bytes, hmoe_stream_t stream) {
  FewPlan P;
  int w = 0;
  int rc = few_check(x, ldx, HMOE_DT_BF16, wgu, nullptr, 0, wd, nullptr, 0, HMOE_DT_BF16, T, d, E, k, h, add, out, workspace,
                     workspace_bytes, P, w);
  if (rc || T == 0) return rc;
  if (!wr || !topk_ids || !topk_w || few_mis(wr, 16)) return HMOE_ERR_ARG;
  if (k > E || E > 256) return HMOE_ERR_SHAPE;
  FewParams p = {};
  p.x = static_cast<const uint16_t*>(x);
  p.ldx = ldx;
  p.T = (int)T; p.d = (int)d; p.E = E; p.k = k; p.h = (int)h; p.M = (int)T * k;
  p.wgu = wgu;
  p.wd = wd;
  p.add = static_cast<const uint16_t*>(add);
  p.out = static_cast<uint16_t*>(out);
  if (E <= 16) {
    p.wr = static_cast<const uint16_t*>(wr);
    p.bias = bias;
    p.renorm = renorm;
    p.scaling = scaling;
    p.out_ids = topk_ids;
    p.out_w = topk_w;
  } else {
    // every workgroup would read the whole router weight: from 17 experts on it has its own launches, its logits where the
    // first kernel's sums will be
    float* logits = reinterpret_cast<float*>(static_cast<char*>(workspace) + P.p1);
    const bool fits = (size_t)T * E * 4 <= P.total - P.p1;
    rc = hmoe_route_topk(x, ldx, wr, bias, T, d, E, k, renorm, scaling, fits ? logits : nullptr, topk_ids, topk_w, stream);
    if (rc) return rc;
    p.ids = topk_ids;
    p.tw = topk_w;
    p.tw_dt = HMOE_DT_F32;
  }
  return few_run(p, P, w, HMOE_DT_BF16, workspace, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
