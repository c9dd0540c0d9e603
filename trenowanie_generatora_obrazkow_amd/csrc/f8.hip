// Products in 8-bit floating point with a scale per block of 128: quantisation of rows and of expert stacks, the grouped
// GEMM over them (plain, with row scale and scatter; SwiGLU with the activation quantised again), and the experts of a
// routed layer in one call.
//
//   y[r, n] = scale[r] * sum_k (a8[r, k] 2^ea[r, k / 128]) (w8[n, k] 2^ew[n / 128, k / 128])
//
// Both operands lie with k contiguous, so a k-slice of 128 is one 128-byte line of every row, and one slice has one scale
// per row of a and one per 128 columns of w.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "f8_common.h"
#include "gemm_common.h"

namespace hmoe {

// ----------------------------------------------------------------------------------------------------------------
// Quantisation
// ----------------------------------------------------------------------------------------------------------------
// eight consecutive values of a row as floats
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t at, float* v) {
  if constexpr (DT == HMOE_DT_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    using X = Elt<DT == HMOE_DT_F16>;
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = X::lo(u[i]);
      v[2 * i + 1] = X::hi(u[i]);
    }
  }
}

// Rows: 16 lanes hold a block of 128 columns, eight each, so a wave reads four blocks in 256-byte (16-bit input) pieces, and
// the block's largest value takes four exchanges within 16 lanes.  Memory-bound, M K (bytes + 1) bytes: 32768 x 8192 bf16 168
// us, 4.8 TB/s; 32768 x 1536 28 us, 5.5.  (Non-temporal stores: 160 us, but 6000 x 1008 and its product 31 -> 33.5.)
template <int DT>
__global__ __launch_bounds__(256) void quant_rows_kernel(const void* __restrict__ x, int64_t ldx, int64_t M, int K, int nb,
                                                         uint8_t* __restrict__ q, int64_t ldq, uint8_t* __restrict__ s,
                                                         int64_t lds) {
  const int sub = threadIdx.x & 15;
  const int64_t blocks = M * nb, step = (int64_t)gridDim.x * 16;
  for (int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); i < blocks; i += step) {
    const int64_t r = i / nb;
    const int b = (int)(i - r * nb), col = b * kF8Block + sub * 8;
    float v[8];
    float m = 0.0f;
    const bool in = col < K;
    if (in) {
      load8<DT>(x, r * ldx + col, v);
#pragma unroll
      for (int t = 0; t < 8; ++t) m = fmaxf(m, f8_abs(v[t]));
    }
    m = bfly_max<8>(bfly_max<4>(bfly_max<2>(bfly_max<1>(m))));
    const int e = f8_exp(m);
    if (in) {
      const float inv = f8_inv(e);
      *reinterpret_cast<uint2*>(q + r * ldq + col) =
          make_uint2(f8_pack4(v[0], v[1], v[2], v[3], inv), f8_pack4(v[4], v[5], v[6], v[7], inv));
    }
    if (sub == 0) s[r * lds + b] = (uint8_t)(e + 127);
  }
}

// A stack (K, N) per expert, N contiguous, in blocks of 128 x 128: a workgroup holds one block in registers (thread t: column
// piece t % 16, rows t / 16 + 16 i), finds its scale, and writes it as it lies (TR = false) or with k contiguous (TR = true,
// through LDS).  Done once for the weights' lifetime; 3 bytes a bf16 value: 16 x 1536 x 8192 183 us, 3.3 TB/s, with the
// gradient's layout too 302 us.
template <int DT, bool TR>
__global__ __launch_bounds__(256) void quant_stack_kernel(const void* __restrict__ w, int64_t stride_we, int64_t stride_wk,
                                                          int K, int Nh, int halves, uint8_t* __restrict__ q,
                                                          uint8_t* __restrict__ s, int64_t lds, int kb_n, int nb_h) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 144];  // [n][k], rows 16 bytes apart from a power of two
  __shared__ float wave_max[4];
  const int t = threadIdx.x;
  const int kb = (int)(blockIdx.x % kb_n), nb = (int)(blockIdx.x / kb_n), half = nb / nb_h;
  const int64_t e = blockIdx.y;
  const int c0 = (nb - half * nb_h) * kF8Block + (t & 15) * 8, k0 = kb * kF8Block + (t >> 4);
  const bool cin = c0 < Nh;
  float v[8][8];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int k = k0 + 16 * i;
    if (cin && k < K) {
      load8<DT>(w, e * stride_we + k * stride_wk + half * Nh + c0, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, f8_abs(v[i][j]));
  }
  m = wave_max_butterfly(m);
  if ((t & 63) == 0) wave_max[t >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
  const int ex = f8_exp(m);
  const float inv = f8_inv(ex);
  const int N = halves * Nh;
  if (t == 0) {
    const int rows = TR ? halves * nb_h : kb_n;
    s[(e * rows + (TR ? nb : kb)) * lds + (TR ? kb : nb)] = (uint8_t)(ex + 127);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t lo = f8_pack4(v[i][0], v[i][1], v[i][2], v[i][3], inv);
    const uint32_t hi = f8_pack4(v[i][4], v[i][5], v[i][6], v[i][7], inv);
    const int k = k0 + 16 * i;
    if constexpr (!TR) {
      if (cin && k < K) *reinterpret_cast<uint2*>(q + (e * K + k) * (int64_t)N + c0) = make_uint2(lo, hi);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        tile[((t & 15) * 8 + j) * 144 + (t >> 4) + 16 * i] = (uint8_t)(lo >> (8 * j));
        tile[((t & 15) * 8 + 4 + j) * 144 + (t >> 4) + 16 * i] = (uint8_t)(hi >> (8 * j));
      }
    }
  }
  if constexpr (TR) {
    __syncthreads();
    for (int i = t; i < 128 * 8; i += 256) {
      const int n = i >> 3, c = i & 7;
      const int col = (nb - half * nb_h) * kF8Block + n, k = kb * kF8Block + c * 16;
      if (col < Nh && k < K)
        *reinterpret_cast<uint4*>(q + (e * N + half * Nh + col) * (int64_t)K + k) =
            *reinterpret_cast<const uint4*>(tile + n * 144 + c * 16);
    }
  }
}

// The values of a quantised matrix, a scale per `block` columns (a power of two, at least 8).  Memory-bound: 32768 x 8192 to
// bf16 153 us, 5.3 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void dequant_rows_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                           const uint8_t* __restrict__ s, int64_t lds, int64_t M, int K8,
                                                           int shift, void* __restrict__ x, int64_t ldx) {
  const int64_t n = M * K8, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
    const int64_t r = i / K8;
    const int col = (int)(i - r * K8) * 8;
    const uint2 w = *reinterpret_cast<const uint2*>(q + r * ldq + col);
    const float sc = f8_pow((int)s[r * lds + (col >> shift)] - 127);
    float v[8];
    f8_unpack2<0>(w.x, v[0], v[1]);
    f8_unpack2<1>(w.x, v[2], v[3]);
    f8_unpack2<0>(w.y, v[4], v[5]);
    f8_unpack2<1>(w.y, v[6], v[7]);
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] *= sc;
    if constexpr (DT == HMOE_DT_F32) {
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(x) + r * ldx + col);
      o[0] = make_float4(v[0], v[1], v[2], v[3]);
      o[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      using X = Elt<DT == HMOE_DT_F16>;
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(x) + r * ldx + col) =
          make_uint4(X::pack2(v[0], v[1]), X::pack2(v[2], v[3]), X::pack2(v[4], v[5]), X::pack2(v[6], v[7]));
    }
  }
}

// ----------------------------------------------------------------------------------------------------------------
// Grouped GEMM
// ----------------------------------------------------------------------------------------------------------------
struct F8Params {
  const uint8_t* A;        // rows of a8 (sorted row r, or a_idx[r]), K bytes, row stride lda
  int64_t lda;
  const uint8_t* As;       // their scales, row stride ldas
  int64_t ldas;
  const int32_t* a_idx;
  const uint8_t* B;        // (E, halves N, K)
  const uint8_t* Bs;       // (E, halves nbs, ldbs): rows of 128 columns of one half
  int64_t ldbs;
  const void* counts;
  int counts64, E;
  int64_t M;
  int K, N, halves, nbs;   // N: columns of a half
  int nb;                  // n-tiles: of all halves (store), of act columns (SwiGLU)
  void* C;                 // store: y; SwiGLU: act as e4m3
  int64_t ldc;
  const int32_t* y_idx;
  const void* scale;       // per row, or NULL
  int scale_dt, scale_by_y;  // indexed by the sorted row, or by the row's place in y
  uint8_t* Cs;             // SwiGLU: act's scales
  int64_t ldcs;
};

constexpr int kF8Slice = 128;  // k per slice: one line of a row, one scale
constexpr int kF8BandM = 4;    // m-tiles of an expert that are walked together over the n-tiles (L2 reuse of the weights)

enum F8Epi { F8_STORE = 0, F8_SWIGLU = 1 };

// ONCE: each weight is copied once, past the caches (non-temporal)
template <int BM_, int BN_, int WM_, int WN_, int NS_, bool ONCE_ = false>
struct F8Cfg {
  static constexpr bool ONCE = ONCE_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_;
  static constexpr int NW = WM * WN, NT = 64 * NW, TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
  static constexpr int A_BYTES = BM * kF8Slice, B_BYTES = BN * kF8Slice, STAGE = A_BYTES + B_BYTES;
  static constexpr int LDS_BYTES = NS * STAGE;
  static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;  // copies of 8 rows per wave and slice
  static_assert(PA * 8 * NW == BM && PB * 8 * NW == BN && FM >= 1 && FN >= 2, "tile");
};

// LDS: a row of a slice is 128 bytes, its 16-byte chunk c at c ^ f8_swz(row), so that 16 rows' chunks of one number lie on
// distinct banks (two rows fill the 64 banks once).
__device__ __forceinline__ int f8_swz(int row) { return (row >> 1) & 7; }

// buf2lds (gemm_common.h) by LDS address
template <bool ONCE = false>
__device__ __forceinline__ void f8_copy(uint32_t voff, i32x4 rsrc, uint32_t soff, uint32_t lds32) {
  const uint32_t m0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds32);
  rsrc.x = __builtin_amdgcn_readfirstlane(rsrc.x);
  rsrc.y = __builtin_amdgcn_readfirstlane(rsrc.y);
  rsrc.z = __builtin_amdgcn_readfirstlane(rsrc.z);
  rsrc.w = __builtin_amdgcn_readfirstlane(rsrc.w);
  soff = (uint32_t)__builtin_amdgcn_readfirstlane((int)soff);
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds"
                 :: "s"(m0), "v"(voff), "s"(rsrc), "s"(soff) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :: "s"(m0), "v"(voff), "s"(rsrc), "s"(soff) : "memory", "m0");
}
// and buf2lds_inner, non-temporal
template <int OFF>
__device__ __forceinline__ void f8_copy_once(uint32_t voff, const i32x4& rsrc, uint32_t soff, uint32_t lds32) {
  asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds"
               :: "s"(lds32), "v"(voff), "s"(rsrc), "s"(soff), "i"(OFF) : "memory", "m0", "scc");
}

// The lane's number as a value of this place: what is computed from it is not moved out of the tile loop, where it would be
// kept, that is spilled, through the main loop (and a spill's reload waits for every store before it)
__device__ __forceinline__ int here(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

// A fragment of 32 rows x 64 k: the lane's row, 32 bytes
__device__ __forceinline__ i32x8 f8_frag(const char* rows, const int* off) {
  typedef int i32x4v __attribute__((ext_vector_type(4)));
  const i32x4v a = *reinterpret_cast<const i32x4v*>(rows + off[0]);
  const i32x4v b = *reinterpret_cast<const i32x4v*>(rows + off[1]);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The weights go in as the first operand, so a lane ends with one row of y (lane % 32) and, per group g of four, columns
// 8 g + 4 (lane / 32) + 0..3 of the fragment.  The scales are the words' lowest bytes.
__device__ __forceinline__ f32x16 f8_mfma(i32x8 w, i32x8 x, f32x16 c, uint32_t sw, uint32_t sx) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, 0, 0, 0, (int)sw, 0, (int)sx);
}
// 16 slices' scales of a row: to the next slice's
__device__ __forceinline__ void f8_next_scale(uint4& v) {
  v.x = __builtin_amdgcn_alignbit(v.y, v.x, 8);
  v.y = __builtin_amdgcn_alignbit(v.z, v.y, 8);
  v.z = __builtin_amdgcn_alignbit(v.w, v.z, 8);
  v.w >>= 8;
}

__device__ __forceinline__ float row_scale_at(const void* s, int dt, int64_t i) {
  if (dt == HMOE_DT_F32) return static_cast<const float*>(s)[i];
  const uint16_t h = static_cast<const uint16_t*>(s)[i];
  return dt == HMOE_DT_BF16 ? Elt<false>::one(h) : Elt<true>::one(h);
}

// One workgroup per CU (two with the tiles of up to 80 KB) walks tiles; the ring of two slices runs on from one tile into the
// next: the last slice's place in the copy stream is taken by the next tile's first slice, so that its latency and the tile
// search hide behind the last products and the epilogue, which parks its output in the stage that the last slice has left.
//
// Bound by the 8-bit matrix instructions for many rows per expert, by the weights' way from memory for few.  Warm, bf16 out:
// 8192^3 400 us, 2.75 PFLOP/s; 32768 rows over 16 experts, 1536 -> 8192 367 us, 2.24 (gate/up 364, 2.27), 4096 -> 1536 160 us,
// 2.58 (a plain library product of 8-bit matrices of these sizes: 360, 354 and 143 us).  In one run, even and warm, even and
// from memory, uneven and warm, uneven and from memory (an expert of none, others of twice the rows; loads of a gate in
// brackets): 1536 -> 8192 386, 434, 400 (415), 454 (463); gate/up 393, 430, 414 (429), 428 (438); 4096 -> 1536 170, 194, 193
// (192), 221 (228): the weights' and rows' first way costs as much as the load.  6000 rows over 12 experts, 1008 -> 2000: 24 to
// 25 whichever, one round of 240 tiles of eight slices.  12000 rows over 128 experts, 2048 -> 2 x 320 43 us, 320 -> 2048 31;
// 288 rows over 64 experts, 2048 -> 2 x 1408 64 us, 1408 -> 2048 30, 5.8 and 6.1 TB/s of weights.
//
// The outputs leave with non-temporal stores: a large one would push the rows and weights that the XCD's next tiles share out
// of its L2.  16 x 2048 rows, 1536 -> 8192: 465 -> 373 us (gate/up, half the columns of one byte, 408 -> 385), one expert 402 ->
// 380; 4096 -> 1536 185 -> 170; the layer of 16384 tokens with the sum over its rows 768 -> 745.  Outputs that the next kernel
// could have read from a cache are at most 1 us slower to it.
//
// WIDE: the operands are widened exactly to bf16 (their scales with them) and multiplied there, at half the rate.  The 8-bit
// instructions add eight products at the exponent of the largest and drop what lies below 2^-13 of it: some 2^-16 of a sum's
// size, nothing to a bf16 result, but where act is quantised again it moves a value in some thousand across a border of the 8
// bits, 1.4e-3 of the layer's output; fp16 outputs (rounded by 2.1e-4) are worth the wider products.
template <class C, int EPI, int CDT, bool WIDE>
__global__ __launch_bounds__(C::NT, C::LDS_BYTES > 81920 ? 1 : 2) void f8_gemm_kernel(F8Params p) {
  static_assert(C::NS == 2, "two stages");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  // behind the ring: where a tile's rows go and their scales, by turns of the tiles (the waves are at most one tile apart);
  // m-tiles up to and with expert e; expert e's first row, [E]: rows counted (at most M)
  constexpr int kRowTab = 2 * C::BM * 8;
  int* const s_tl = reinterpret_cast<int*>(smem + C::LDS_BYTES + kRowTab);
  int* const s_r0 = s_tl + p.E;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int E = p.E, per = (E + 63) / 64;

  // ---- the experts' rows and m-tiles: one wave scans the counts, E / 64 experts a lane ----
  if (wave == 0) {
    auto count = [&](int e) __attribute__((always_inline)) {
      return std::min(std::max(read_count(p.counts, p.counts64, e), (int64_t)0), p.M);
    };
    int64_t rs = 0;
    for (int i = 0; i < per; ++i) {
      const int e = lane * per + i;
      if (e < E) rs += count(e);
    }
    int64_t irs = rs;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int64_t a = __shfl_up(irs, s, 64);
      if (lane >= s) irs += a;
    }
    int64_t at = irs - rs;
    int tl = 0;
    for (int i = 0; i < per; ++i) {  // (rows past M do not exist)
      const int e = lane * per + i;
      if (e >= E) break;
      const int64_t end = at + count(e);
      const int lo = (int)std::min(at, p.M), hi = (int)std::min(end, p.M);
      tl += (hi - lo + C::BM - 1) / C::BM;
      s_r0[e] = lo;
      s_tl[e] = tl;
      at = end;
    }
    int itl = tl;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int a = __shfl_up(itl, s, 64);
      if (lane >= s) itl += a;
    }
    for (int i = 0; i < per; ++i) {
      const int e = lane * per + i;
      if (e < E) s_tl[e] += itl - tl;
    }
    if (lane == 63) s_r0[E] = (int)std::min(irs, p.M);
  }
  __syncthreads();
  const int counted = __builtin_amdgcn_readfirstlane(s_r0[E]);
  const int total = __builtin_amdgcn_readfirstlane(s_tl[E - 1]) * p.nb;
  const int share = (total + 7) >> 3;  // the tiles in runs of equal length over the 8 XCDs (workgroups go to them in turn)

  struct Tile {
    int e, nbi, row0, live;
  };
  // The workgroup's j-th tile: bands of kF8BandM m-tiles of an expert, n-tile by n-tile.  Where an XCD's last round has tiles
  // for at most half of its workgroups, 256-row tiles are halved by rows: waves without rows leave out their products (32768
  // rows over 16 experts of uneven load, 4096 -> 1536, 3.2 rounds: 205 -> 196 us).
  constexpr bool kHalve = C::BM == 256 && C::NW == 8;
  const int wgs = (int)gridDim.x >> 3, whole = kHalve && share % wgs * 2 <= wgs ? share / wgs * wgs : share;
  auto find = [&](int j, Tile& t) __attribute__((always_inline)) {
    const int v = (int)blockIdx.x + j * (int)gridDim.x, at = v >> 3;
    const bool halved = kHalve && at >= whole;
    const int mine = halved ? whole + ((at - whole) >> 1) : at, tile = (v & 7) * share + mine;
    if (mine >= share || tile >= total) return false;
    const int mt = tile / p.nb;
    int e = 0;
    for (int i = 0; i < per; ++i) {
      const int x = i * 64 + lane;
      e += __builtin_popcountll(__ballot((x < E ? s_tl[x] : INT32_MAX) <= mt));
    }
    const int m0 = e > 0 ? s_tl[e - 1] : 0, mt_e = s_tl[e] - m0, first = s_r0[e], end = s_r0[e + 1];
    const int local = tile - m0 * p.nb, band = local / (kF8BandM * p.nb) * kF8BandM;
    const int mc = min(kF8BandM, mt_e - band), r = local - band * p.nb;
    t.e = e;
    t.nbi = __builtin_amdgcn_readfirstlane(r / mc);
    t.row0 = __builtin_amdgcn_readfirstlane(first + (band + r % mc) * C::BM);
    t.live = __builtin_amdgcn_readfirstlane(min(end - t.row0, C::BM));
    if (halved) {
      const int skip = (at - whole) & 1 ? C::BM / 2 : 0;
      t.row0 += skip;
      t.live = min(t.live - skip, C::BM / 2);
    }
    return t.live > 0;  // (nothing follows the last round's)
  };
  const int nbh = EPI == F8_STORE ? p.nb / p.halves : p.nb;
  // the half a tile lies in, and its first column there (store), or its first column of act (SwiGLU)
  auto half_of = [&](const Tile& t) { return EPI == F8_STORE ? t.nbi / nbh : 0; };
  auto n0_of = [&](const Tile& t) { return (t.nbi - half_of(t) * nbh) * (EPI == F8_SWIGLU ? C::BN / 2 : C::BN); };

  // ---- copy sources of the tile whose slices are being copied ----
  const int K = p.K, nk = (K + kF8Slice - 1) / kF8Slice;
  i32x4 rsA, rsB;
  uint32_t vA[C::PA], vB[C::PB];
  auto chunk_of = [&](int ln, int rr) { return (ln & 7) ^ f8_swz(rr); };
  auto set_sources = [&](const Tile& t) __attribute__((always_inline)) {
    const int ln = here(lane);
    rsA = make_rsrc(p.a_idx ? p.A : p.A + (int64_t)t.row0 * p.lda);
    rsB = make_rsrc(p.B + (int64_t)t.e * p.halves * p.N * K);
    const int half = half_of(t), n0 = n0_of(t);
#pragma unroll
    for (int i = 0; i < C::PA; ++i) {
      const int rr = 8 * (wave * C::PA + i) + (ln >> 3);
      vA[i] = kOOB;
      if (rr < t.live) {
        const int64_t src = p.a_idx ? (int64_t)p.a_idx[t.row0 + rr] : (int64_t)rr;
        vA[i] = (uint32_t)(src * p.lda + chunk_of(ln, rr) * 16);
      }
    }
#pragma unroll
    for (int i = 0; i < C::PB; ++i) {
      const int rr = 8 * (wave * C::PB + i) + (ln >> 3);
      int col, row;  // column within the half, row of B
      if constexpr (EPI == F8_SWIGLU) {
        col = n0 + rr % (C::BN / 2);
        row = rr / (C::BN / 2) * p.N + col;
      } else {
        col = n0 + rr;
        row = half * p.N + col;
      }
      vB[i] = col < p.N ? (uint32_t)((int64_t)row * K + chunk_of(ln, rr) * 16) : kOOB;
    }
  };
  const uint32_t ring = lds_addr(smem);
  auto issue = [&](int kt, int stage) __attribute__((always_inline)) {  // slice kt, whole or not, into a stage
    const uint32_t slot = ring + stage * C::STAGE;
    const int k0 = kt * kF8Slice, ln = here(lane);
#pragma unroll
    for (int i = 0; i < C::PA; ++i)
      f8_copy(k0 + chunk_of(ln, 8 * (wave * C::PA + i) + (ln >> 3)) * 16 < K ? vA[i] : kOOB, rsA, (uint32_t)k0,
              slot + (wave * C::PA + i) * 1024);
#pragma unroll
    for (int i = 0; i < C::PB; ++i)
      f8_copy<C::ONCE>(k0 + chunk_of(ln, 8 * (wave * C::PB + i) + (ln >> 3)) * 16 < K ? vB[i] : kOOB, rsB, (uint32_t)k0,
              slot + C::A_BYTES + (wave * C::PB + i) * 1024);
  };

  int off[2][2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      off[ks][j] = (lane & 31) * 128 + (((ks * 4 + (lane >> 5) * 2 + j) ^ f8_swz(lane & 31)) * 16);
  auto b_row = [&](int b) {  // tile row of column fragment b
    if constexpr (EPI == F8_SWIGLU)
      return b < C::FN / 2 ? wn * (C::TN / 2) + b * 32 : C::BN / 2 + wn * (C::TN / 2) + (b - C::FN / 2) * 32;
    else
      return wn * C::TN + b * 32;
  };
  f32x16 acc[C::FM][C::FN];
  uint4 sA[C::FM], sB0, sB1;

  // One slice's products, the copies of the slice that follows dealt between them (FAST: one that lies inside K; otherwise
  // they have been issued)
  auto products = [&](auto fast_tag, int stage, int k0) __attribute__((always_inline)) {
    constexpr bool FAST = decltype(fast_tag)::value;
    constexpr int NM = 2 * C::FM * C::FN, NC = C::PA + C::PB;  // products, copies
    const char* sa = smem + stage * C::STAGE;
    const char* sb = sa + C::A_BYTES;
    const uint32_t fa = ring + (stage ^ 1) * C::STAGE + wave * (C::PA * 1024);
    const uint32_t fb = ring + (stage ^ 1) * C::STAGE + C::A_BYTES + wave * (C::PB * 1024);
    const uint32_t so = (uint32_t)k0;
    i32x8 xa[2][C::FM], wb[2][C::FN];
    auto read_a = [&](int ks, int a) { xa[ks][a] = f8_frag(sa + (wm * C::TM + a * 32) * 128, off[ks]); };
    auto read_b = [&](int ks, int b) { wb[ks][b] = f8_frag(sb + b_row(b) * 128, off[ks]); };
#pragma unroll
    for (int b = 0; b < C::FN; ++b) read_b(0, b);
#pragma unroll
    for (int a = 0; a < C::FM; ++a) read_a(0, a);
    static_for<NM>([&](auto n_tag) __attribute__((always_inline)) {
      constexpr int n = decltype(n_tag)::value, ks = n / (C::FM * C::FN), a = n / C::FN % C::FM, b = n % C::FN;
      acc[a][b] = f8_mfma(wb[ks][b], xa[ks][a], acc[a][b], EPI == F8_SWIGLU && b >= C::FN / 2 ? sB1.x : sB0.x, sA[a].x);
      if constexpr (FAST) {
        constexpr int PER = (NC + NM / 4 - 1) / (NM / 4);  // in the first half, to have the other half to arrive in
        constexpr int c0 = n * PER < NC ? n * PER : NC, c1 = (n + 1) * PER < NC ? (n + 1) * PER : NC;
        static_for<c1 - c0>([&](auto j) __attribute__((always_inline)) {
          constexpr int c = c0 + decltype(j)::value;
          if constexpr (c < C::PA)
            buf2lds_inner<c * 1024>(vA[c], rsA, so, fa);
          else if constexpr (C::ONCE)
            f8_copy_once<(c - C::PA) * 1024>(vB[c - C::PA], rsB, so, fb);
          else
            buf2lds_inner<(c - C::PA) * 1024>(vB[c - C::PA], rsB, so, fb);
        });
      }
      if constexpr (ks == 0) {  // the second half's fragments behind the first half's products
        if constexpr (b == 0) read_a(1, a);
        constexpr int per_b = (C::FN + C::FM - 1) / C::FM;
        if constexpr (b < per_b && a * per_b + b < C::FN) read_b(1, a * per_b + b);
      }
    });
  };

  auto products_wide = [&](int stage) __attribute__((always_inline)) {
    const char* sa = smem + stage * C::STAGE;
    const char* sb = sa + C::A_BYTES;
    auto scale_of = [](uint32_t w) { return f8_pow((int)(w & 0xffu) - 127); };
    float fa[C::FM];
#pragma unroll
    for (int a = 0; a < C::FM; ++a) fa[a] = scale_of(sA[a].x);
    const float f0 = scale_of(sB0.x), f1 = EPI == F8_SWIGLU ? scale_of(sB1.x) : f0;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // eight of the lane's 32 values of k
        u32x4 xa[C::FM], wb[C::FN];
        auto piece = [&](const char* rows) { return *reinterpret_cast<const uint2*>(rows + off[ks][i >> 1] + (i & 1) * 8); };
#pragma unroll
        for (int b = 0; b < C::FN; ++b)
          wb[b] = f8_widen(piece(sb + b_row(b) * 128), EPI == F8_SWIGLU && b >= C::FN / 2 ? f1 : f0);
#pragma unroll
        for (int a = 0; a < C::FM; ++a) xa[a] = f8_widen(piece(sa + (wm * C::TM + a * 32) * 128), fa[a]);
#pragma unroll
        for (int a = 0; a < C::FM; ++a)
#pragma unroll
          for (int b = 0; b < C::FN; ++b)
            acc[a][b] = mfma16<false>(__builtin_bit_cast(bf16x8, wb[b]), __builtin_bit_cast(bf16x8, xa[a]), acc[a][b]);
      }
  };

  // rows that no expert counts are zeros (where rows keep their places)
  auto zero_rows = [&]() __attribute__((always_inline)) {
    constexpr int ES = CDT == HMOE_DT_F32 ? 4 : 2;
    const int pieces = (int)((int64_t)p.halves * p.N * ES / 16);
    for (int64_t row = counted + (int64_t)blockIdx.x; row < p.M; row += gridDim.x)
      for (int i = threadIdx.x; i < pieces; i += C::NT)
        *reinterpret_cast<uint4*>(static_cast<char*>(p.C) + row * p.ldc * ES + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  };
  if constexpr (EPI == F8_STORE)
    if (!p.y_idx && counted < p.M) zero_rows();

  const uint8_t* pa[C::FM];  // scales of the lane's rows a*32 + lane%32 of the wave, and of the wave's columns
  const uint8_t *pb0, *pb1;
  auto set_scales = [&](const Tile& t) __attribute__((always_inline)) {
    const int lrow = here(lane) & 31;
#pragma unroll
    for (int a = 0; a < C::FM; ++a) {
      const int row = t.row0 + min(wm * C::TM + a * 32 + lrow, t.live - 1);  // (past the last row: its values are zeros)
      pa[a] = p.As + (p.a_idx ? (int64_t)p.a_idx[row] : (int64_t)row) * p.ldas;
    }
    // one 128-column block (store), the gate's and the up's (SwiGLU)
    const int sblk = min((n0_of(t) + wn * (EPI == F8_STORE ? C::TN : C::TN / 2)) / kF8Block, p.nbs - 1);
    pb0 = p.Bs + ((int64_t)(t.e * p.halves + half_of(t)) * p.nbs + sblk) * p.ldbs;
    pb1 = EPI == F8_SWIGLU ? pb0 + (int64_t)p.nbs * p.ldbs : pb0;
  };
  auto load_scales = [&](int kt) __attribute__((always_inline)) {  // of slices kt .. kt + 15
#pragma unroll
    for (int a = 0; a < C::FM; ++a) sA[a] = *reinterpret_cast<const uint4*>(pa[a] + kt);
    sB0 = *reinterpret_cast<const uint4*>(pb0 + kt);
    if constexpr (EPI == F8_SWIGLU) sB1 = *reinterpret_cast<const uint4*>(pb1 + kt);
  };

  Tile t;
  if (!find(0, t)) return;
  set_sources(t);
  issue(0, 0);
  set_scales(t);
  load_scales(0);
  wait_vm<0>();
  int stage = 0;
  for (int j = 1;; ++j) {  // (the tile's first slice and scales have landed)
    const int half = half_of(t), n0 = n0_of(t);
    [[maybe_unused]] int* const s_y = reinterpret_cast<int*>(smem + C::LDS_BYTES + (j & 1) * (C::BM * 8));
    [[maybe_unused]] float* const s_sc = reinterpret_cast<float*>(s_y + C::BM);
    if constexpr (EPI == F8_STORE) {  // where the tile's rows go, and their scales (read behind the main loop's barriers)
      for (int i = wave * 64 + here(lane); i < t.live; i += C::NT) {
        const int row = t.row0 + i, y = p.y_idx ? p.y_idx[row] : row;
        s_y[i] = y;
        s_sc[i] = p.scale ? row_scale_at(p.scale, p.scale_dt, p.scale_by_y ? y : row) : 1.0f;
      }
    }
#pragma unroll
    for (int a = 0; a < C::FM; ++a)
#pragma unroll
      for (int b = 0; b < C::FN; ++b)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[a][b][v] = 0.0f;

    // ---- main loop ----
    Tile next;
    bool more = false;
    auto begin_slice = [&](int kt) __attribute__((always_inline)) {
      if (kt > 0) {
        if ((kt & 15) == 0) load_scales(kt);
        wait_vm<0>();  // this wave's copies of slice kt have landed
      }
      lds_barrier();  // and the others'; all have read the slice before, whose stage is filled next
    };
    auto end_slice = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < C::FM; ++a) f8_next_scale(sA[a]);
      f8_next_scale(sB0);
      if constexpr (EPI == F8_SWIGLU) f8_next_scale(sB1);
      stage ^= 1;
    };
    int kt = 0;
    if (kHalve && wm * C::TM >= t.live) {  // no rows: this wave copies only
      for (; kt + 1 < nk; ++kt) {
        begin_slice(kt);
        issue(kt + 1, stage ^ 1);
        end_slice();
      }
    } else if constexpr (!WIDE) {
      for (; (kt + 2) * kF8Slice <= K; ++kt) {
        begin_slice(kt);
        products(std::true_type{}, stage, (kt + 1) * kF8Slice);
        end_slice();
      }
    }
    for (; kt < nk; ++kt) {
      begin_slice(kt);
      if (kt + 1 < nk) {
        issue(kt + 1, stage ^ 1);
      } else {
        more = find(j, next);
        if (more) {
          set_sources(next);
          issue(0, stage ^ 1);
        }
      }
      if constexpr (WIDE)
        products_wide(stage);
      else
        products(std::false_type{}, stage, 0);
      end_slice();
    }
    if (more) set_scales(next);
    if (more) load_scales(0);
    lds_barrier();  // all have read the last slice: its stage (the next tile's first slice goes to the other) takes the output
    char* const park = smem + (stage ^ 1) * C::STAGE;
    const int ln = here(lane), lrow = ln & 31, lcol = 4 * (ln >> 5);

    if constexpr (EPI == F8_STORE) {
      // 32 rows of the wave at a time go through its own part of the stage, chunk c of a row at c ^ row, and leave in whole
      // rows; in two turns where they fit, so that one's rows are written while the other's are read back
      constexpr int ES = CDT == HMOE_DT_F32 ? 4 : 2;
      constexpr int FP = ES == 4 ? C::FN / 2 : C::FN;  // column fragments of a pass
      constexpr int RB = FP * 32 * ES, CPR = RB / 16, RPI = 64 / CPR;
      constexpr int TURNS = 2 * 32 * RB * C::NW <= C::STAGE ? 2 : 1;
      static_assert(32 * RB * C::NW <= C::STAGE, "a pass of every wave in a stage");
      char* const own = park + wave * (TURNS * 32 * RB);
      if (wm * C::TM >= t.live) wait_vm<0>();  // (a wave without rows: see below)
#pragma unroll
      for (int a = 0; a < C::FM; ++a) {
        const int rbase = wm * C::TM + a * 32;
        if (rbase >= t.live) break;
        const float sc = s_sc[min(rbase + lrow, t.live - 1)];
#pragma unroll
        for (int b0 = 0; b0 < C::FN; b0 += FP) {
          char* const buf = own + (a * (C::FN / FP) + b0 / FP) % TURNS * (32 * RB);
#pragma unroll
          for (int b = 0; b < FP; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const f32x16& v = acc[a][b0 + b];
              const float o[4] = {v[4 * g] * sc, v[4 * g + 1] * sc, v[4 * g + 2] * sc, v[4 * g + 3] * sc};
              const int byte = (b * 32 + 8 * g + lcol) * ES;
              char* at = buf + lrow * RB + (((byte >> 4) ^ (lrow & (CPR - 1))) << 4) + (byte & 15);
              if constexpr (CDT == HMOE_DT_F32) {
                *reinterpret_cast<float4*>(at) = make_float4(o[0], o[1], o[2], o[3]);
              } else {
                using X = Elt<CDT == HMOE_DT_F16>;
                *reinterpret_cast<uint2*>(at) = make_uint2(X::pack2(o[0], o[1]), X::pack2(o[2], o[3]));
              }
            }
          __builtin_amdgcn_wave_barrier();
          // the next tile's first slice and scales have landed before the first store: that slice does not wait for the stores
          if (a == 0 && b0 == 0) wait_vm<0>();
#pragma unroll
          for (int i = 0; i < 32 / RPI; ++i) {
            const int rr = i * RPI + ln / CPR, c = ln % CPR;
            const u32x4 v = *reinterpret_cast<const u32x4*>(buf + rr * RB + ((c ^ (rr & (CPR - 1))) << 4));
            const int64_t y = s_y[min(rbase + rr, t.live - 1)];
            const int col = n0 + wn * C::TN + b0 * 32 + c * (16 / ES);
            if (rbase + rr < t.live && col < p.N)
              __builtin_nontemporal_store(
                  v, reinterpret_cast<u32x4*>(static_cast<char*>(p.C) + (y * p.ldc + half * p.N + col) * ES));
          }
          __builtin_amdgcn_wave_barrier();
        }
      }
    } else {
      // act = silu(g) u in fp32, in place of g; the largest of a row's 128 columns from the lanes l and l ^ 32 and, through
      // LDS, the waves side by side; then e4m3 through LDS into whole 128-byte rows
      float* s_max = reinterpret_cast<float*>(park);  // [WN][BM]
      char* const rows = park + C::WN * C::BM * 4;    // [BM][128]
      static_assert(C::BN / 2 == kF8Block && C::WN * C::BM * 4 + C::BM * 128 <= C::STAGE, "one block of act per tile");
#pragma unroll
      for (int a = 0; a < C::FM; ++a) {
        float m = 0.0f;
#pragma unroll
        for (int b = 0; b < C::FN / 2; ++b)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float act = silu_f(acc[a][b][v]) * acc[a][b + C::FN / 2][v];
            acc[a][b][v] = act;
            m = fmaxf(m, f8_abs(act));
          }
        m = bfly_max<32>(m);
        if (ln < 32) s_max[wn * C::BM + wm * C::TM + a * 32 + lrow] = m;
      }
      lds_barrier();
#pragma unroll
      for (int a = 0; a < C::FM; ++a) {
        const int rr = wm * C::TM + a * 32 + lrow;
        float m = 0.0f;
#pragma unroll
        for (int w = 0; w < C::WN; ++w) m = fmaxf(m, s_max[w * C::BM + rr]);
        const int ex = f8_exp(m);
        const float inv = f8_inv(ex);
        if (a == 0) wait_vm<0>();  // as above
        if (wn == 0 && ln < 32 && rr < t.live) p.Cs[(int64_t)(t.row0 + rr) * p.ldcs + t.nbi] = (uint8_t)(ex + 127);
#pragma unroll
        for (int b = 0; b < C::FN / 2; ++b)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x16& v = acc[a][b];
            const int byte = wn * (C::TN / 2) + b * 32 + 8 * g + lcol;
            *reinterpret_cast<uint32_t*>(rows + rr * 128 + (((byte >> 4) ^ f8_swz(rr)) << 4) + (byte & 15)) =
                f8_pack4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3], inv);
          }
      }
      lds_barrier();
      for (int i = wave * 64 + ln; i < t.live * 8; i += C::NT) {
        const int rr = i >> 3, c = i & 7;
        if (n0 + c * 16 < p.N)
          __builtin_nontemporal_store(
              *reinterpret_cast<const u32x4*>(rows + rr * 128 + ((c ^ f8_swz(rr)) << 4)),
              reinterpret_cast<u32x4*>(static_cast<char*>(p.C) + (int64_t)(t.row0 + rr) * p.ldc + n0 + c * 16));
      }
    }
    if (!more) break;
    t = next;
  }
}

static int f8_cus() {
  static std::atomic<int> n[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  int v = n[dev].load(std::memory_order_relaxed);
  if (v == 0) {
    if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0) return 0;
    n[dev].store(v, std::memory_order_relaxed);
  }
  return v;
}

template <class C, int EPI, int CDT, bool WIDE>
static int f8_launch(const F8Params& p, hipStream_t s) {
  auto kern = f8_gemm_kernel<C, EPI, CDT, WIDE>;
  constexpr int kLds = C::LDS_BYTES + 2 * C::BM * 8 + 16;  // and 8 bytes per expert
  static std::atomic<bool> attr_set[64];  // per device
  int dev = 0;
  const int cus = f8_cus();
  if (cus <= 0 || hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return HMOE_ERR_DEVICE;
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                            kLds + kMaxEGemm * 8) !=
        hipSuccess)
      return HMOE_ERR_LAUNCH;
    attr_set[dev].store(true, std::memory_order_release);
  }
  F8Params q = p;
  q.nb = EPI == F8_SWIGLU ? (p.N + C::BN / 2 - 1) / (C::BN / 2) : p.halves * ((p.N + C::BN - 1) / C::BN);
  // an m-tile for every expert with rows and at most M / BM further ones; the workgroups in eights (one per XCD)
  const int64_t tiles = (std::min<int64_t>(p.E, p.M) + p.M / C::BM) * q.nb;
  if (tiles >= (1 << 28)) return HMOE_ERR_SHAPE;
  const int64_t wgs = std::min<int64_t>(tiles, (int64_t)cus * (C::LDS_BYTES > 81920 ? 1 : 2));
  hipLaunchKernelGGL(kern, dim3((unsigned)((wgs + 7) / 8 * 8)), dim3(C::NT), kLds + p.E * 8, s, q);
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

// Tiles: 32 x 256 (two workgroups per CU: few rows per expert, the launch streams weights); 128 x 128, two workgroups per CU,
// one's epilogue under the other's products (gate/up, whose tile makes one block of act: 128 x 256, one workgroup of 8 waves);
// 256 x 256.  Each is priced by its rounds over the CUs, a round by its slices; the prices (us) follow 76 launches of each kind:
// 1 to 128 experts of random load, 4 to 8192 rows each, d 768-8192, h 320-8192, every tile timed in turn.  Over these the
// choice takes 1% more than the fastest tile on average (gate/up 2%) and at most 15% (17%; wide 40%, where 1.4 rounds of 32
// rows would have been one of 128).  A line by rows per expert took up to 1.9 times the fastest: 1024 -> 1024 x 2048 rows over
// 8 experts of 300 31 instead of 19 us.
// 8 waves for a tile of 256 x 256: twice the LDS reads per product of 4 waves, but two waves per SIMD, of which one computes
// while the other waits or is in the epilogue: gate/up 16 x 2048 rows, 1536 -> 8192, 482 -> 440 us, in 16 bits 788 -> 738;
// plain outputs 510 -> 504 there, 600 rows of 1024 x 768 over 32 experts 41 -> 35 (4 waves are 4% ahead where K is 8192).
// With at most 32 rows per expert the weights go past the caches, which leaves these to the rows and the outputs: 64 experts of
// 4 rows, 2048 -> 2 x 1408 70 -> 64 us, 1408 -> 2048 35 -> 32, 16 of 4, 1536 -> 2 x 4096 34 -> 31 (layers whose weights the 256
// MB cache holds lose up to 1 us of 16).  Uneven loads gain as well, though an expert of several row tiles reads its weights
// several times (14 launches of 8 to 256 experts, 4 to 32 rows an expert on average, the weights from memory; past the caches
// and through them): loads by 1 / (e + 1), 16 rows on average and 212 at most, 2048 -> 2 x 1408 65.5 and 71.7; 32 and 413 83.4
// and 86.5; 1408 -> 2048 44.6 and 47.5; 256 experts, 2048 -> 2 x 256, 16 and 657 56.8 and 61.1; none of the 56 slower.  Not
// where further row tiles read them again (128 experts of 96 rows, 2048 -> 2 x 320 64 -> 76), nor where a row's end shares its
// line with the next one's begin (320 -> 2048, 4 rows: 22 -> 27).
template <int EPI, int CDT, bool WIDE = false>
static int f8_pick(const F8Params& p, hipStream_t s) {
  const int cus = f8_cus();
  if (cus <= 0) return HMOE_ERR_DEVICE;
  const double hit = (double)std::min<int64_t>(p.E, p.M), rows = (double)p.M / hit, nk = (p.K + kF8Slice - 1) / kF8Slice;
  auto price = [&](double bm, double bn, double slots, double fixed, double slice) {
    const double nb = EPI == F8_SWIGLU ? std::ceil(p.N / (bn / 2)) : p.halves * std::ceil(p.N / bn);
    // (uneven counts make some tiles more)
    const double rounds = 1.08 * hit * std::max(1.0, rows / bm + 0.5) * nb / slots;
    return (rounds < 4 ? std::ceil(rounds) : rounds) * (fixed + slice * nk);
  };
  double t32, t128, t256;
  if constexpr (EPI == F8_STORE) {
    t32 = price(32, 256, 2 * cus, 7, 0.7), t128 = price(128, 128, 2 * cus, 5, 0.7), t256 = price(256, 256, cus, 8, 1.15);
  } else if constexpr (WIDE) {
    t32 = price(32, 256, 2 * cus, 3, 1.3), t128 = price(128, 256, cus, 4, 1.65), t256 = price(256, 256, cus, 8, 2.75);
  } else {
    t32 = price(32, 256, 2 * cus, 2.5, 1.1), t128 = price(128, 256, cus, 2, 1.3), t256 = price(256, 256, cus, 5, 1.75);
  }
  if (t32 <= t128 && t32 <= t256) {
    if (rows <= 32 && p.K % kF8Slice == 0) return f8_launch<F8Cfg<32, 256, 1, 4, 2, true>, EPI, CDT, WIDE>(p, s);
    return f8_launch<F8Cfg<32, 256, 1, 4, 2>, EPI, CDT, WIDE>(p, s);
  }
  if constexpr (EPI == F8_STORE) {
    if (t128 <= t256) return f8_launch<F8Cfg<128, 128, 2, 2, 2>, EPI, CDT, WIDE>(p, s);
  } else {
    if (t128 <= t256) return f8_launch<F8Cfg<128, 256, 2, 4, 2>, EPI, CDT, WIDE>(p, s);
  }
  return f8_launch<F8Cfg<256, 256, 2, 4, 2>, EPI, CDT, WIDE>(p, s);
}

static bool al(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

static int f8_check(const void* a, int64_t lda, const uint8_t* a_s, int64_t lda_s, const int32_t* a_idx, int64_t a_rows,
                    const void* w, const uint8_t* w_s, int64_t E, int64_t K, int64_t N, int halves, const void* counts, int counts_dtype,
                    int64_t M) {
  if (!counts || E <= 0 || M < 0) return HMOE_ERR_ARG;
  if (E > kMaxEGemm || M > INT32_MAX - 256) return HMOE_ERR_SHAPE;
  if (counts_dtype != HMOE_DT_I32 && counts_dtype != HMOE_DT_I64) return HMOE_ERR_DTYPE;
  if (M == 0) return HMOE_OK;
  if (!a || !a_s || !w || !w_s || K <= 0 || N <= 0 || halves < 1 || halves > 2 || N % halves) return HMOE_ERR_ARG;
  if (K % 16 || N / halves % 16) return HMOE_ERR_SHAPE;
  if (lda < K || lda % 16 || lda_s < f8_scale_ld(K) || lda_s % 16 || !al(a, 16) || !al(a_s, 16) || !al(w, 16) || !al(w_s, 16))
    return HMOE_ERR_ARG;
  // 32-bit copy offsets: one expert's weights, the rows of a tile, all of a where its rows are gathered
  const int64_t lim = ((int64_t)1 << 31) - 32768;
  if (K > lim / N || lda > lim / 256 || (a_idx && a_rows > lim / lda)) return HMOE_ERR_SHAPE;
  if (a_rows < (a_idx ? 1 : M)) return HMOE_ERR_ARG;
  return HMOE_OK;
}

static F8Params f8_params(const void* a, int64_t lda, const uint8_t* a_s, int64_t lda_s, const int32_t* a_idx, const void* w,
                          const uint8_t* w_s, int64_t E, int64_t K, int64_t N, int halves, const void* counts,
                          int counts_dtype, int64_t M) {
  F8Params p = {};
  p.A = static_cast<const uint8_t*>(a);
  p.lda = lda;
  p.As = a_s;
  p.ldas = lda_s;
  p.a_idx = a_idx;
  p.B = static_cast<const uint8_t*>(w);
  p.Bs = w_s;
  p.ldbs = f8_scale_ld(K);
  p.counts = counts;
  p.counts64 = counts_dtype == HMOE_DT_I64;
  p.E = (int)E;
  p.M = M;
  p.K = (int)K;
  p.N = (int)(N / halves);
  p.halves = halves;
  p.nbs = (p.N + kF8Block - 1) / kF8Block;
  return p;
}

}  // namespace hmoe

using namespace hmoe;

extern "C" {

size_t hmoe_f8_scale_ld(int64_t K) { return K > 0 ? static_cast<size_t>(f8_scale_ld(K)) : 0; }

int hmoe_f8_quant_rows(const void* x, int64_t ldx, int dtype, int64_t M, int64_t K, void* q, int64_t ldq, uint8_t* s,
                       int64_t lds, hmoe_stream_t stream) {
  if (M < 0 || K <= 0) return HMOE_ERR_ARG;
  if (dtype != HMOE_DT_BF16 && dtype != HMOE_DT_F16 && dtype != HMOE_DT_F32) return HMOE_ERR_DTYPE;
  if (M == 0) return HMOE_OK;
  if (!x || !q || !s) return HMOE_ERR_ARG;
  if (K % 16 || K > INT32_MAX - 256) return HMOE_ERR_SHAPE;
  if (ldx < K || ldx % 8 || ldq < K || ldq % 16 || lds < f8_scale_ld(K) || lds % 16 || !al(x, 16) || !al(q, 16) || !al(s, 16))
    return HMOE_ERR_ARG;
  const int nb = (int)((K + kF8Block - 1) / kF8Block);
  const int64_t groups = (M * nb + 15) / 16;
  const dim3 grid((unsigned)std::min<int64_t>(groups, 4096));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto* q8 = static_cast<uint8_t*>(q);
  if (dtype == HMOE_DT_BF16)
    hipLaunchKernelGGL(quant_rows_kernel<HMOE_DT_BF16>, grid, dim3(256), 0, st, x, ldx, M, (int)K, nb, q8, ldq, s, lds);
  else if (dtype == HMOE_DT_F16)
    hipLaunchKernelGGL(quant_rows_kernel<HMOE_DT_F16>, grid, dim3(256), 0, st, x, ldx, M, (int)K, nb, q8, ldq, s, lds);
  else
    hipLaunchKernelGGL(quant_rows_kernel<HMOE_DT_F32>, grid, dim3(256), 0, st, x, ldx, M, (int)K, nb, q8, ldq, s, lds);
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

int hmoe_f8_dequant_rows(const void* q, int64_t ldq, const uint8_t* s, int64_t lds, int64_t M, int64_t K, int block, void* x,
                         int64_t ldx, int dtype, hmoe_stream_t stream) {
  if (M < 0 || K <= 0) return HMOE_ERR_ARG;
  if (dtype != HMOE_DT_BF16 && dtype != HMOE_DT_F16 && dtype != HMOE_DT_F32) return HMOE_ERR_DTYPE;
  if (block != 128 && block != 32) return HMOE_ERR_SHAPE;
  if (M == 0) return HMOE_OK;
  if (!q || !s || !x) return HMOE_ERR_ARG;
  if (K % 8 || K > INT32_MAX - 256) return HMOE_ERR_SHAPE;
  if (ldq < K || ldq % 8 || lds < (K + block - 1) / block || ldx < K || ldx % 8 || !al(q, 8) || !al(x, 16)) return HMOE_ERR_ARG;
  const int k8 = (int)(K / 8), shift = block == 128 ? 7 : 5;
  const dim3 grid((unsigned)std::min<int64_t>((M * k8 + 255) / 256, 8192));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto* q8 = static_cast<const uint8_t*>(q);
  if (dtype == HMOE_DT_BF16)
    hipLaunchKernelGGL(dequant_rows_kernel<HMOE_DT_BF16>, grid, dim3(256), 0, st, q8, ldq, s, lds, M, k8, shift, x, ldx);
  else if (dtype == HMOE_DT_F16)
    hipLaunchKernelGGL(dequant_rows_kernel<HMOE_DT_F16>, grid, dim3(256), 0, st, q8, ldq, s, lds, M, k8, shift, x, ldx);
  else
    hipLaunchKernelGGL(dequant_rows_kernel<HMOE_DT_F32>, grid, dim3(256), 0, st, q8, ldq, s, lds, M, k8, shift, x, ldx);
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

int hmoe_f8_quant_stack(const void* w, int dtype, int64_t E, int64_t K, int64_t N, int64_t stride_we, int64_t stride_wk,
                        int halves, int transpose, void* q, uint8_t* s, hmoe_stream_t stream) {
  if (E <= 0 || K <= 0 || N <= 0 || halves < 1 || halves > 2 || N % halves) return HMOE_ERR_ARG;
  if (dtype != HMOE_DT_BF16 && dtype != HMOE_DT_F16 && dtype != HMOE_DT_F32) return HMOE_ERR_DTYPE;
  if (!w || !q || !s) return HMOE_ERR_ARG;
  if (K % 16 || N / halves % 16 || E > kMaxEGemm || K > INT32_MAX - 256 || N > INT32_MAX - 256) return HMOE_ERR_SHAPE;
  if (!transpose && halves != 1) return HMOE_ERR_SHAPE;  // blocks of a reduction run over all of it
  if (stride_wk < N || stride_wk % 8 || stride_we % 8 || !al(w, 16) || !al(q, 16)) return HMOE_ERR_ARG;
  const int kb = (int)((K + kF8Block - 1) / kF8Block), nh = (int)(N / halves), nbh = (nh + kF8Block - 1) / kF8Block;
  if ((int64_t)kb * halves * nbh >= ((int64_t)1 << 23)) return HMOE_ERR_SHAPE;
  const int64_t lds = f8_scale_ld(transpose ? K : N);
  const dim3 grid((unsigned)(kb * halves * nbh), (unsigned)E);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto* q8 = static_cast<uint8_t*>(q);
  auto go = [&](auto dt, auto tr) {
    hipLaunchKernelGGL((quant_stack_kernel<decltype(dt)::value, decltype(tr)::value>), grid, dim3(256), 0, st, w, stride_we,
                       stride_wk, (int)K, nh, halves, q8, s, lds, kb, nbh);
  };
  auto by_dt = [&](auto tr) {
    if (dtype == HMOE_DT_BF16) go(std::integral_constant<int, HMOE_DT_BF16>{}, tr);
    else if (dtype == HMOE_DT_F16) go(std::integral_constant<int, HMOE_DT_F16>{}, tr);
    else go(std::integral_constant<int, HMOE_DT_F32>{}, tr);
  };
  if (transpose) by_dt(std::true_type{});
  else by_dt(std::false_type{});
  HMOE_CHECK_LAUNCH();
  return HMOE_OK;
}

int hmoe_f8_grouped_mm(const void* a, int64_t lda, const uint8_t* a_s, int64_t lda_s, int64_t a_rows, const void* w,
                       const uint8_t* w_s, int64_t E, int64_t K, int64_t N, int halves, const void* counts, int counts_dtype,
                       int64_t M, const int32_t* a_idx, const int32_t* y_idx, const void* scale, int scale_dtype, int scale_by_y, void* y,
                       int64_t ldy, int y_dtype, hmoe_stream_t stream) {
  int rc = f8_check(a, lda, a_s, lda_s, a_idx, a_rows, w, w_s, E, K, N, halves, counts, counts_dtype, M);
  if (rc) return rc;
  if (y_dtype != HMOE_DT_BF16 && y_dtype != HMOE_DT_F16 && y_dtype != HMOE_DT_F32) return HMOE_ERR_DTYPE;
  if (scale && scale_dtype != HMOE_DT_BF16 && scale_dtype != HMOE_DT_F16 && scale_dtype != HMOE_DT_F32) return HMOE_ERR_DTYPE;
  if (M == 0) return HMOE_OK;
  if (!y || !al(y, 16) || ldy < N || ldy % 8) return HMOE_ERR_ARG;
  F8Params p = f8_params(a, lda, a_s, lda_s, a_idx, w, w_s, E, K, N, halves, counts, counts_dtype, M);
  p.C = y;
  p.ldc = ldy;
  p.y_idx = y_idx;
  p.scale = scale;
  p.scale_dt = scale_dtype;
  p.scale_by_y = scale_by_y && y_idx;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (y_dtype == HMOE_DT_BF16) return f8_pick<F8_STORE, HMOE_DT_BF16>(p, s);
  if (y_dtype == HMOE_DT_F16) return f8_pick<F8_STORE, HMOE_DT_F16>(p, s);
  return f8_pick<F8_STORE, HMOE_DT_F32>(p, s);
}

size_t hmoe_f8_quant_mm_workspace_size(int64_t rows, int64_t K) {
  if (rows < 0 || K <= 0 || K > INT32_MAX - 256 || rows > INT32_MAX) return 0;
  return static_cast<size_t>(rows) * static_cast<size_t>((K + 15) / 16 * 16 + f8_scale_ld(K)) + 16;
}

int hmoe_f8_quant_mm(const void* x, int64_t ldx, int x_dtype, int64_t rows, const void* w, const uint8_t* w_s, int64_t E,
                     int64_t K, int64_t N, int halves, const void* counts, int counts_dtype, int64_t M, const int32_t* a_idx,
                     const int32_t* y_idx, const void* scale, int scale_dtype, int scale_by_y, void* y, int64_t ldy, int y_dtype,
                     void* workspace, size_t workspace_bytes, hmoe_stream_t stream) {
  if (rows < 0 || K <= 0) return HMOE_ERR_ARG;
  const size_t need = hmoe_f8_quant_mm_workspace_size(rows, K);
  if (!workspace || need == 0 || workspace_bytes < need || !al(workspace, 16)) return HMOE_ERR_WORKSPACE;
  auto* q = static_cast<uint8_t*>(workspace);
  auto* s = q + rows * ((K + 15) / 16 * 16);
  // the product's limits ahead of the first launch, so that a refused call launches nothing
  int rc = f8_check(q, K, s, f8_scale_ld(K), a_idx, rows, w, w_s, E, K, N, halves, counts, counts_dtype, M);
  if (rc) return rc;
  if (y_dtype != HMOE_DT_BF16 && y_dtype != HMOE_DT_F16 && y_dtype != HMOE_DT_F32) return HMOE_ERR_DTYPE;
  if (scale && scale_dtype != HMOE_DT_BF16 && scale_dtype != HMOE_DT_F16 && scale_dtype != HMOE_DT_F32) return HMOE_ERR_DTYPE;
  if (M > 0 && (!y || !al(y, 16) || ldy < N || ldy % 8)) return HMOE_ERR_ARG;
  rc = hmoe_f8_quant_rows(x, ldx, x_dtype, M == 0 ? 0 : rows, K, q, K, s, f8_scale_ld(K), stream);
  if (rc) return rc;
  return hmoe_f8_grouped_mm(q, K, s, f8_scale_ld(K), rows, w, w_s, E, K, N, halves, counts, counts_dtype, M, a_idx, y_idx, scale,
                            scale_dtype, scale_by_y, y, ldy, y_dtype, stream);
}

int hmoe_f8_gate_up_swiglu(const void* x, int64_t ldx, const uint8_t* x_s, int64_t ldx_s, int64_t x_rows, const int32_t* a_idx,
                           const void* wgu, const uint8_t* wgu_s, int64_t E, int64_t d, int64_t h, const void* counts, int counts_dtype,
                           int64_t M, int wide, void* act, uint8_t* act_s, hmoe_stream_t stream) {
  if (h <= 0) return HMOE_ERR_ARG;
  int rc = f8_check(x, ldx, x_s, ldx_s, a_idx, x_rows, wgu, wgu_s, E, d, 2 * h, 2, counts, counts_dtype, M);
  if (rc || M == 0) return rc;
  if (!act || !act_s || !al(act, 16)) return HMOE_ERR_ARG;
  F8Params p = f8_params(x, ldx, x_s, ldx_s, a_idx, wgu, wgu_s, E, d, 2 * h, 2, counts, counts_dtype, M);
  p.C = act;
  p.ldc = h;
  p.Cs = act_s;
  p.ldcs = f8_scale_ld(h);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return wide ? f8_pick<F8_SWIGLU, HMOE_DT_F8, true>(p, s) : f8_pick<F8_SWIGLU, HMOE_DT_F8>(p, s);
}

}  // extern "C"

// The experts of a routed layer for given routing: x quantised, dispatch, gate/up with SwiGLU and act quantised, down with the
// routing weights (fp32 as given) and scatter, over one workspace.
namespace {

size_t al256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

struct F8Layout {
  size_t x8, xs, counts, starts, order, a_idx, dws, act, act_s, total, dws_bytes;
};

bool f8_layout(int64_t T, int64_t d, int E, int k, int64_t h, F8Layout& L) {
  if (T < 0 || d <= 0 || E <= 0 || k <= 0 || h <= 0 || T > INT32_MAX || d > INT32_MAX || h > INT32_MAX || k > 1024) return false;
  const size_t t = static_cast<size_t>(T), M = t * static_cast<size_t>(k);
  L.dws_bytes = hmoe_dispatch_workspace_size(T, k, E);
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += al256(bytes > 0 ? bytes : 1);
    return at;
  };
  L.x8 = take(t * static_cast<size_t>(d));
  L.xs = take(t * static_cast<size_t>(f8_scale_ld(d)));
  L.counts = take(static_cast<size_t>(E) * 4);
  L.starts = take(static_cast<size_t>(E + 1) * 4);
  L.order = take(M * 4);
  L.a_idx = take(M * 4);
  L.dws = take(L.dws_bytes);
  L.act = take(M * static_cast<size_t>(h));
  L.act_s = take(M * static_cast<size_t>(f8_scale_ld(h)));
  L.total = o;
  return true;
}

}  // namespace

extern "C" {

size_t hmoe_f8_moe_experts_workspace_size(int64_t T, int64_t d, int E, int k, int64_t h) {
  F8Layout L;
  return f8_layout(T, d, E, k, h, L) ? L.total : 0;
}

int hmoe_f8_moe_experts(const void* x, int64_t ldx, int dtype, const void* topk_ids, int ids_dtype, const void* topk_w,
                        int topk_w_dtype, const void* wgu, const uint8_t* wgu_s, const void* wd, const uint8_t* wd_s, int64_t T,
                        int64_t d, int E, int k, int64_t h, void* y, int32_t* inv_pos, int32_t* n_invalid, void* workspace,
                        size_t workspace_bytes, hmoe_stream_t stream) {
  F8Layout L;
  if (!f8_layout(T, d, E, k, h, L)) return HMOE_ERR_ARG;
  if (dtype != HMOE_DT_BF16 && dtype != HMOE_DT_F16) return HMOE_ERR_DTYPE;
  if (topk_w_dtype != HMOE_DT_F32 && topk_w_dtype != HMOE_DT_BF16 && topk_w_dtype != HMOE_DT_F16) return HMOE_ERR_DTYPE;
  if (!workspace || workspace_bytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return HMOE_ERR_WORKSPACE;
  // every launch's limits ahead of the first, so that a refused call launches nothing (an empty input only runs the dispatch)
  if (T > 0 && (!x || !topk_ids || !topk_w || !wgu || !wgu_s || !wd || !wd_s || !y || ldx < d || ldx % 8 || !al(x, 16) ||
                !al(wgu, 16) || !al(wgu_s, 16) || !al(wd, 16) || !al(wd_s, 16) || !al(y, 16)))
    return HMOE_ERR_ARG;
  const int64_t lim = ((int64_t)1 << 31) - 32768, M = T * k;
  if (d % 16 || h % 16 || E > kMaxEGemm || M > INT32_MAX - 256 || d > lim / (2 * h) || d > lim / 256 || h > lim / 256 ||
      T > lim / d)
    return HMOE_ERR_SHAPE;
  char* ws = static_cast<char*>(workspace);
  auto* counts = reinterpret_cast<int32_t*>(ws + L.counts);
  auto* order = reinterpret_cast<int32_t*>(ws + L.order);
  auto* a_idx = reinterpret_cast<int32_t*>(ws + L.a_idx);
  auto* xs = reinterpret_cast<uint8_t*>(ws + L.xs);
  auto* act_s = reinterpret_cast<uint8_t*>(ws + L.act_s);
  int rc = hmoe_dispatch_tiles(topk_ids, ids_dtype, topk_w, topk_w_dtype, T, k, E, nullptr, 0, 0, nullptr, nullptr, counts,
                               nullptr, reinterpret_cast<int32_t*>(ws + L.starts), order, a_idx, inv_pos, nullptr, n_invalid,
                               ws + L.dws, L.dws_bytes, dtype, stream);
  if (rc != HMOE_OK || M == 0) return rc;
  rc = hmoe_f8_quant_rows(x, ldx, dtype, T, d, ws + L.x8, d, xs, f8_scale_ld(d), stream);
  if (rc != HMOE_OK) return rc;
  rc = hmoe_f8_gate_up_swiglu(ws + L.x8, d, xs, f8_scale_ld(d), T, a_idx, wgu, wgu_s, E, d, h, counts, HMOE_DT_I32, M,
                              dtype == HMOE_DT_F16, ws + L.act, act_s, stream);
  if (rc != HMOE_OK) return rc;
  return hmoe_f8_grouped_mm(ws + L.act, h, act_s, f8_scale_ld(h), M, wd, wd_s, E, h, d, 1, counts, HMOE_DT_I32, M, nullptr, order,
                            topk_w, topk_w_dtype, 1, y, d, dtype, stream);
}

}  // extern "C"
