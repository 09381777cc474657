// i8.hip -- products of 8-bit integers with a scale for each row of either side:
// Y[m][n] = sx[m] sw[n] sum_k Xq[m][k] Wq[n][k] (+ bias[n]), and the quantizer that
// makes such rows.  No reference function (the reference's own 8-bit form is q8_0,
// whose activations stay fp32).
//
// The sum is a whole number.  Codes of the quantizer are -127 to 127, and their sums exact in
// int32 for K <= 133144 (2^31 / 127^2); a code of -128, which rows from elsewhere may hold, leaves
// room for K <= 132104 on one side and 131071 on both.  So neither the tile, the order of K nor a
// split of it changes a result: one rounding of the sum to fp32, two products, the bias, and the
// output's own rounding.
//
// An int8 row is padded with zeros to whole 128-byte steps (i8_row_bytes), so no kernel
// has a K tail: padding of x adds zeros whatever the padding of W holds.
#include "tm_i8.h"
#include "tm_tiles.h"

#include <algorithm>
#include <cmath>

namespace tiermm {
int device_cus(int* cus);
namespace {

typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

// ------------------------------------------------------------------- quantizer
// One row a workgroup of NT threads.  R > 0: the row has at most R * NT units of 16 bytes and
// stays in registers, all its loads on their way at once; R = 0: any row, read twice.
template <int XT, int NT, int R>
__global__ __launch_bounds__(NT) void i8_quant_kernel(const uint8_t* __restrict__ x, size_t ldx,
                                                      int8_t* __restrict__ q, size_t rb, float* __restrict__ scale,
                                                      int K, int Kp) {
  using X = Rows<XT>;
  __shared__ uint32_t red[NT / 64];
  const uint8_t* row = x + (size_t)blockIdx.x * ldx;
  const int k0 = threadIdx.x * X::EPU, step = NT * X::EPU;
  u32x4 u[R > 0 ? R : 1];
  uint32_t top = 0;
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) u[i] = k0 + i * step < K ? X::get(row, k0 + i * step, K) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float v[X::EPU];
      X::widen(u[i], v);
      top = top_bits(v, top);
    }
  } else {
    for (int k = k0; k < K; k += step) {
      float v[X::EPU];
      X::widen(X::get(row, k, K), v);
      top = top_bits(v, top);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) top = max(top, red[w]);
  const RowScale r = row_scale_of(top);
  int8_t* out = q + (size_t)blockIdx.x * rb;
  auto put = [&](int k, const u32x4& c) __attribute__((always_inline)) {
    float v[X::EPU];
    X::widen(c, v);
    if constexpr (X::EPU == 8) *(u32x2*)(out + k) = u32x2{codes4(v, r), codes4(v + 4, r)};
    else *(uint32_t*)(out + k) = codes4(v, r);
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (k0 + i * step < Kp) put(k0 + i * step, u[i]);
  } else {
    for (int k = k0; k < Kp; k += step) put(k, k < K ? X::get(row, k, K) : u32x4{0u, 0u, 0u, 0u});
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = r.sc;
}

// --------------------------------------------------------------------- product
struct I8Args {
  const uint8_t* X;     // M (grouped: xrows) rows of rbx bytes
  const float* sx;
  const uint8_t* W;     // N rows of rbw bytes (grouped: E times)
  const float* sw;
  const float* bias;    // or null
  uint8_t* Y;
  size_t rbx, rbw, ldy;  // bytes
  int M, N, K, nk;       // nk steps of K
  // grouped: rows [off[e], off[e + 1]) of Y belong to expert e
  const int32_t* off;
  const int32_t* rows;  // row p of Y reads row rows[p] / topk of X (null: row p)
  int E, topk, xrows;
  int share;  // tiles that an XCD takes at a time
};

// What a workgroup computes: rows [m0, m1) of Y, column tile tn.
struct Tile {
  int m0, m1, tn;
  int e;      // expert; E: rows that no expert has, which become zeros (zero_tile)
  bool once;  // no other tile reads these rows of W
};

// Tile `bid` over the experts' rows, expert by expert, and in each column by column; false past
// the last.  XCD x (bid % 8) takes `share` tiles at a time: their rows of W and X meet in its L2.
// Each wave finds it from the offsets, 64 experts a step.
template <int BM>
__device__ __forceinline__ bool grouped_tile(const I8Args& a, int ntn, int bid, Tile& tl) {
  const int lane = threadIdx.x & 63, P = a.M, i = bid >> 3;
  const int t = ((i / a.share) * 8 + (bid & 7)) * a.share + i % a.share;
  int run = 0;
  for (int e0 = 0; e0 <= a.E; e0 += 64) {
    // rows of expert e (E: those from off[E] to P), whatever the offsets hold within [0, P]
    const int e = e0 + lane, b = e <= a.E ? min(max(a.off[e], 0), P) : P;
    const int end = e < a.E ? min(max(a.off[e + 1], 0), P) : P;
    const int rows = max(end - b, 0), n = (rows + BM - 1) / BM * ntn;
    int s = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(s, o, 64);
      s += lane >= o ? up : 0;
    }
    const uint64_t hit = __ballot(t >= run + s - n && t < run + s);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      const int r0 = __shfl(b, l, 64), nr = __shfl(rows, l, 64), t0 = run + __shfl(s - n, l, 64);
      const int ntm = (nr + BM - 1) / BM, in = t - t0;
      tl.e = e0 + l;
      tl.tn = in / ntm;
      tl.m0 = r0 + (in % ntm) * BM;
      tl.m1 = min(tl.m0 + BM, r0 + nr);
      tl.once = ntm == 1;
      return true;
    }
    run += __shfl(s, 63, 64);
  }
  // rows in front of off[0], counted from P (zero_tile)
  const int lead = min(max(a.off[0], 0), P), ntm = (lead + BM - 1) / BM, in = t - run;
  if (in >= ntm * ntn) return false;
  tl.e = a.E;
  tl.tn = in / ntm;
  tl.m0 = P + (in % ntm) * BM;
  tl.m1 = min(tl.m0 + BM, P + lead);
  tl.once = false;
  return true;
}

// The tile of this workgroup; false past the last.  Dense tiles go in groups of 4 tile rows,
// column by column.
template <int BM, int BN, bool GROUPED>
__device__ __forceinline__ bool find_tile(const I8Args& a, Tile& tl) {
  const int ntn = (a.N + BN - 1) / BN;
  if constexpr (GROUPED) return grouped_tile<BM>(a, ntn, blockIdx.x, tl);
  const int ntm = (a.M + BM - 1) / BM, t = xcd_share(blockIdx.x, ntm * ntn);
  if (t < 0) return false;
  constexpr int GM = 4;
  const int grp = t / (GM * ntn), first = grp * GM, gm = min(GM, ntm - first), in = t - grp * GM * ntn;
  tl.m0 = (first + in % gm) * BM;
  tl.m1 = min(tl.m0 + BM, a.M);
  tl.tn = in / gm;
  tl.e = 0;
  tl.once = ntm == 1;
  return true;
}

// Row of X behind row p of Y, or -1.
template <bool GROUPED>
__device__ __forceinline__ int source_row(const I8Args& a, int p) {
  if constexpr (!GROUPED) return p;
  if (!a.rows) return p < a.xrows ? p : -1;
  const int i = a.rows[p];
  const int r = i < 0 ? -1 : i / a.topk;
  return r < a.xrows ? r : -1;
}

// Start of row r of a stage of BM rows of X and BN of W (rows past the tile: its last one).
template <int BM, bool GROUPED>
__device__ __forceinline__ const uint8_t* stage_row(const I8Args& a, const Tile& tl, int n0, int r) {
  if (r < BM) return a.X + (size_t)max(source_row<GROUPED>(a, min(tl.m0 + r, tl.m1 - 1)), 0) * a.rbx;
  const uint8_t* W = a.W + (GROUPED ? (size_t)tl.e * a.N * a.rbw : 0);
  return W + (size_t)min(n0 + r - BM, a.N - 1) * a.rbw;
}

// Columns n0 .. n0 + BN - 1 of rows that no expert has become zeros: rows [m0, m1), those from P up
// being the ones in front of off[0].
template <class Y, int BN, int THREADS>
__device__ __forceinline__ void zero_tile(const I8Args& a, const Tile& tl, int n0) {
  const int cols = min(BN, a.N - n0);
  for (int i = tl.m0; i < tl.m1; ++i) {
    const int m = i < a.M ? i : i - a.M;
    for (int c = threadIdx.x * Y::EPU; c < cols; c += THREADS * Y::EPU)
      Y::set(a.Y + (size_t)m * a.ldy + (size_t)n0 * Y::ES, c, cols, u32x4{0u, 0u, 0u, 0u});
  }
}

// Scales are far where one is not 0 and below 2^-63, or from 2^63 up.
struct ScaleRange {
  float least = 1.f, most = 0.f;
  __device__ __forceinline__ void add(float v) {
    least = fminf(least, v == 0.f ? 1.f : fabsf(v));
    most = fmaxf(most, fabsf(v));
  }
  __device__ __forceinline__ bool far() const { return least < 0x1p-63f || most >= 0x1p63f; }
};

// BM rows of X times BN rows of W by WVM x WVN waves of WM x WN blocks of 32 x 32.
//
// A stage is 128 bytes of every row, brought to LDS by global_load_lds; S stages take
// turns.  A row's 16-byte chunk c lies at slot c ^ ((row >> 1) & 7): the 16 rows that one
// cycle of a fragment read touches then cover all the banks (c ^ (row & 7) spent half of the
// LDS cycles on conflicts).  A stage is four MFMA steps of K = 32.  While the products of one
// step run, the fragments of the next come in, one read between two MFMAs, and the loads of
// stage kt + S go out, spread the same way from the step after the barrier that frees their
// place on (256 x 256, a stage: 2993 -> 2760 cycles; the MFMAs alone take 2048).
//
// W is the MFMA's first operand, so a lane holds four neighbouring columns of one row of Y;
// rows leave through LDS in 16-byte units (stored from the lanes, element by element, the
// epilogue took 12 us a tile; so it takes 4).
//
// Measured: 4096 x 14336 x 5120, bf16 out, 256 x 320 tiles: 244-252 us, 2.4-2.5 PFLOP/s (a
// library's int8 product of this size without scales: 2.12).  The card's power limit bounds
// it: the clock falls to 1.6-1.7 GHz and the MFMAs alone, on operands that stay put, take 175
// of the K loop's 240 us; on zeros the clock stays at 2.36 GHz and the call takes 224 us.
// Larger tiles cost less power for loads and LDS reads a product: 256 x 256 266, 128 x 128 315.
// No faster: 64-byte stages in rings of 4 and 5 (312, 326), four waves of 128 x 128 (337).
template <int YT, int BM, int BN, int WVM, int WVN, int S, bool GROUPED>
__global__ __launch_bounds__(64 * WVM * WVN) void i8_gemm_kernel(const I8Args a) {
  constexpr int NW = WVM * WVN, WM = BM / WVM / 32, WN = BN / WVN / 32, NF = WM + WN;
  constexpr int STAGE = (BM + BN) * kStep, INST = STAGE / 1024 / NW;
  static_assert(WM * WVM * 32 == BM && WN * WVN * 32 == BN && INST * NW * 1024 == STAGE, "whole blocks and loads a wave");
  static_assert(WM <= 2, "row blocks that step() tells apart");
  // loads of a stage by the step that issues them: 3 (of the stage before last), 0 and 1
  constexpr int D0 = (INST + 2) / 3, D1 = (INST - D0 + 1) / 2, D2 = INST - D0 - D1;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  float* col_scale = (float*)(lds + S * STAGE);
  float* col_bias = col_scale + BN;
  float* row_scale = col_bias + BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Tile tl;
  if (!find_tile<BM, BN, GROUPED>(a, tl)) return;
  const int n0 = tl.tn * BN;
  using Y = Rows<YT>;
  if (GROUPED && tl.e == a.E) return zero_tile<Y, BN, 64 * NW>(a, tl, n0);
  const float* sw = a.sw + (GROUPED ? (size_t)tl.e * a.N : 0);

  // load u of this wave: rows 8 * (wave + NW * u) .. + 7 of the stage (X's, then W's)
  const uint8_t* src[INST];
#pragma unroll
  for (int u = 0; u < INST; ++u) {
    const int r = 8 * (wave + NW * u) + (lane >> 3);
    src[u] = stage_row<BM, GROUPED>(a, tl, n0, r) + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
  }
  const uint32_t lds0 = lds_addr(lds);
  auto ring = [](int kt) { return S == 2 ? kt & 1 : S == 4 ? kt & 3 : kt % S; };
  auto issue = [&](int kt, int u) __attribute__((always_inline)) {
    dma16(src[u] + (size_t)kt * kStep, lds0 + ring(kt) * STAGE + (wave + NW * u) * 1024);
  };
#pragma unroll
  for (int t = 0; t < S - 1; ++t)
    if (t < a.nk) {
#pragma unroll
      for (int u = 0; u < INST; ++u) issue(t, u);
    }

  // the scales of the tile's rows and columns, for the end; a far one where a row has no source, so
  // that store() looks
  for (int i = tid; i < BN; i += 64 * NW) {
    const int n = min(n0 + i, a.N - 1);
    col_scale[i] = sw[n];
    col_bias[i] = a.bias ? a.bias[n] : 0.f;
  }
  for (int i = tid; i < BM; i += 64 * NW) {
    const int xr = source_row<GROUPED>(a, min(tl.m0 + i, tl.m1 - 1));
    row_scale[i] = xr < 0 ? 0x1p-127f : a.sx[xr];
  }

  i32x16 acc[WN][WM];
#pragma unroll
  for (int j = 0; j < WN; ++j)
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0;

  const int wm = wave % WVM, wn = wave / WVM, fr = lane & 31, fh = lane >> 5, turn = (fr >> 1) & 7;
  const uint32_t xrow = (uint32_t)(wm * 32 + fr) * kStep, wrow = (uint32_t)(BM + wn * WN * 32 + fr) * kStep;
  i32x4 xf[2][WM], wf[2][WN];
  // fragment v of step kk of stage kt into set f: W's first, the m of X, W's others, as the
  // products need them
  auto fragment = [&](int m, int kt, int kk, int f, int v) __attribute__((always_inline)) {
    const uint8_t* s = lds + ring(kt) * STAGE + ((2 * kk + fh) ^ turn) * 16;
    if (v >= 1 && v <= m) xf[f][v - 1] = *(const i32x4*)(s + xrow + (v - 1) * WVM * 32 * kStep);
    else wf[f][v == 0 ? 0 : v - m] = *(const i32x4*)(s + wrow + (v == 0 ? 0 : v - m) * 32 * kStep);
  };
  // Grouped: the blocks of this wave that hold rows of the expert.  A wave's blocks of 32 rows lie
  // WVM blocks apart, so a tile of 256 rows that holds 128 or fewer keeps every SIMD half busy:
  // 512 tokens x 8 over 64 experts, 2816 x 2048, 256 x 256 tiles 102 us; with neighbouring blocks,
  // and waves that have all their work or none, 112.
  const int live = GROUPED ? (tl.m1 - tl.m0 - wm * 32 + WVM * 32 - 1) / (WVM * 32) : WM;
  // The products of fragments f, with the fragments (kt, kk) into the other set and loads
  // u0 .. u0 + n - 1 of stage `dt` between them; of the first m blocks of rows.
  auto products = [&](auto mc, int f, int kt, int kk, int dt, int u0, int n) __attribute__((always_inline)) {
    constexpr int m = decltype(mc)::value, nm = m * WN, nf = m + WN;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < nm; ++q) {
#pragma unroll
      for (int v = 0; v < nf; ++v)
        if (std::max(v * (nm - 2) / nf, 0) == q) fragment(m, kt, kk, f ^ 1, v);
#pragma unroll
      for (int d = 0; d < n; ++d)
        if (std::min(1 + d * (nm - 1) / n, nm - 1) == q && dt < a.nk) issue(dt, u0 + d);
      const int j = q / m, i = q % m;
      acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[f][j], xf[f][i], acc[j][i], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto step = [&](int f, int kt, int kk, int dt, int u0, int n) __attribute__((always_inline)) {
    if (live >= WM) return products(std::integral_constant<int, WM>(), f, kt, kk, dt, u0, n);
    if constexpr (WM == 2)
      if (live == 1) return products(std::integral_constant<int, 1>(), f, kt, kk, dt, u0, n);
#pragma unroll
    for (int d = 0; d < n; ++d)
      if (dt < a.nk) issue(dt, u0 + d);
  };
  // waits until stage kt has landed, those up to kt + S - 2 being on their way too
  auto landed = [&](int kt) __attribute__((always_inline)) {
    const int behind = a.nk - 1 - kt;
    if (behind >= S - 2) vm_wait<(S - 2) * INST>();
    else wait_stages<S - 3, INST>(behind);
  };
  landed(0);
  __syncthreads();
  if (S - 1 < a.nk) {
#pragma unroll
    for (int u = 0; u < D0; ++u) issue(S - 1, u);
  }
  // scales of this wave's elements, to see at the end whether one is far
  float scale_x[WM], scale_w[WN];
#pragma unroll
  for (int i = 0; i < WM; ++i) scale_x[i] = row_scale[(i * WVM + wm) * 32 + fr];
#pragma unroll
  for (int j = 0; j < WN; ++j) scale_w[j] = col_scale[(wn * WN + j) * 32 + fr];
  __builtin_amdgcn_sched_barrier(0);  // the first fragments in the loop's own order, one wait for each
#pragma unroll
  for (int v = 0; v < NF; ++v) {
    fragment(WM, 0, 0, 0, v);
    __builtin_amdgcn_sched_barrier(0);
  }
  for (int kt = 0; kt < a.nk; ++kt) {
    step(0, kt, 1, kt + S - 1, D0, D1);
    step(1, kt, 2, kt + S - 1, D0 + D1, D2);
    step(0, kt, 3, 0, 0, 0);
    landed(kt + 1);
    __syncthreads();  // stage kt + 1 has landed for every wave, and stage kt is read
    // (past the end: the fragments of what the place holds, which nothing uses)
    step(1, kt + 1, 0, kt + S, 0, D0);
  }

  // Element r of a block is column 8 * (r / 4) + 4 * fh + r % 4 of row fr: a lane's own
  // stores would be 4 columns wide.  Each wave passes 32 rows of one or two blocks at a
  // time through its part of LDS and stores whole 16-byte units, 8 of them a row.
  constexpr int JB = Y::ES == 2 ? 2 : 1, PART = 4096;
  static_assert(NW * PART <= S * STAGE, "rows of the epilogue in LDS");
  uint8_t* part = lds + wave * PART;
  auto store = [&](auto far_scales, auto jn, int j0) __attribute__((always_inline)) {
    constexpr bool FAR = decltype(far_scales)::value;
    constexpr int J = decltype(jn)::value, CH = J * 32 * Y::ES / 16;
    const int cw = (wn * WN + j0) * 32, nw = n0 + cw;
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      const int rw = (i * WVM + wm) * 32, mb = tl.m0 + rw;
      if (mb >= tl.m1) break;
      const float s = row_scale[rw + fr];
      // rows without a source are zeros, whatever the columns' scales are
      const bool none = FAR && GROUPED && source_row<GROUPED>(a, min(mb + fr, tl.m1 - 1)) < 0;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int c = j * 32 + 8 * b + 4 * fh;
          const f32x4 cs = *(const f32x4*)(col_scale + cw + c), cb = *(const f32x4*)(col_bias + cw + c);
          f32x4 v;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int sum = acc[j0 + j][i][4 * b + k];
            v[k] = none ? 0.f : FAR ? scaled(sum, s, cs[k], cb[k]) : scaled_near(sum, s, cs[k], cb[k]);
          }
          Y::set4(part + out_place<CH>(fr, c * Y::ES), v);
        }
      wave_lds_wait();
#pragma unroll
      for (int u = 0; u < CH / 2; ++u) {
        const int r = u * (64 / CH) + lane / CH, c = lane % CH, col = nw + c * Y::EPU;
        const u32x4 v = *(const u32x4*)(part + out_place<CH>(r, c * 16));
        if (mb + r < tl.m1 && col < a.N) Y::set(a.Y + (size_t)(mb + r) * a.ldy, col, a.N, v);
      }
      wave_lds_wait();
    }
  };
  auto store_all = [&](auto far_scales) __attribute__((always_inline)) {
#pragma unroll
    for (int j0 = 0; j0 + JB <= WN; j0 += JB) store(far_scales, std::integral_constant<int, JB>(), j0);
    if constexpr (WN % JB) store(far_scales, std::integral_constant<int, WN % JB>(), WN - WN % JB);
  };
  ScaleRange range;
#pragma unroll
  for (int i = 0; i < WM; ++i) range.add(scale_x[i]);
#pragma unroll
  for (int j = 0; j < WN; ++j) range.add(scale_w[j]);
  const bool wave_far = __ballot(range.far()) != 0;
  __syncthreads();  // every wave has read its last stage
  if (__builtin_expect(wave_far, 0)) return store_all(std::true_type());
  store_all(std::false_type());
}

// Launches fn over the tiles; grouped, every expert, and the rows in front of the first and behind
// the last, may end in a partly filled one.
template <class Fn>
int launch(Fn* fn, std::atomic<uint64_t>& done, I8Args a, bool grouped, int bm, int bn, int threads, int lds,
           hipStream_t s, const char* who) {
  const int st = lds_attr_once(done, (const void*)fn, lds, who);
  if (st != TIERMM_OK) return st;
  const long long ntn = (a.N + bn - 1) / bn;
  const long long ntm = grouped ? a.M / bm + std::min(a.E + 2, a.M) : (a.M + bm - 1) / bm;
  a.share = (int)std::min(32ll, (ntm * ntn + 7) / 8);
  const long long step = grouped ? 8ll * a.share : 8, grid = (ntm * ntn + step - 1) / step * step;
  if (grid > (1ll << 22)) return set_error(TIERMM_UNSUPPORTED, "%s: %lld tiles", who, ntm * ntn);
  fn<<<(unsigned)grid, threads, lds, s>>>(a);
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

template <int YT, int BM, int BN, int WVM, int WVN, int S, bool GROUPED>
int launch_gemm(const I8Args& a, hipStream_t s, const char* who) {
  constexpr int LDS = S * (BM + BN) * kStep + (BM + 2 * BN) * 4;
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static std::atomic<uint64_t> done{0};
  return launch(i8_gemm_kernel<YT, BM, BN, WVM, WVN, S, GROUPED>, done, a, GROUPED, BM, BN, 64 * WVM * WVN, LDS, s, who);
}

// ----------------------------------------------------------------- single tokens
// Sum of two wave-wide vectors' halves (32) or rows of 16 lanes (16): the lanes of one half
// then hold a's sums, the others' b's.
__device__ __forceinline__ int merge32(int a, int b) {
  const auto t = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  return (int)t[0] + (int)t[1];
}
__device__ __forceinline__ int merge16(int a, int b) {
  const auto t = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  return (int)t[0] + (int)t[1];
}
template <int CTRL>
__device__ __forceinline__ int add_ror(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
// Wave-wide sums of v[0 .. R): lanes 16 g .. + 15 hold that of v[g * R / 4].
template <int R>
__device__ __forceinline__ int wave_sums(const int (&v)[R]) {
  int s;
  if constexpr (R == 2) { const int h = merge32(v[0], v[1]); s = merge16(h, h); }
  else { const int h = merge32(v[0], v[0]); s = merge16(h, h); }
  return add_ror<0x121>(add_ror<0x122>(add_ror<0x124>(add_ror<0x128>(s))));  // row_ror 8, 4, 2, 1
}

// Up to MX rows of x, quantized by each workgroup into LDS while its first weights are on the
// way.  A wave takes R rows of W in 1 KiB pieces, 16 bytes a lane, so each load is eight whole
// lines of one row; v_dot4 on 16 bytes a lane costs a tenth of what the bytes take to come.
//
// Bound by the stream of W, and by x's preparation in front of it (some 2 us): 1 x 28672 x 14336
// bf16 59-61 us (6.7-7.0 TB/s), 1 x 14336 x 5120 13.0-13.5 (5.4-5.6), 1 x 1024 x 5120 fp32
// 4.1-4.6.  Two rows a wave and 16 waves: each CU prepares x once or twice; 4 waves 15.6 us, four
// rows and 4 waves 14.6, at 14336 rows; one row a wave and 8 waves at 1024: 4.5 against 7.0.  On
// MFMA 16x16x64 with W straight from memory, 16 rows of 64 bytes a load: 16.7.
template <int YT, int XT, int MX, int R, int NW>
__global__ __launch_bounds__(64 * NW) void i8_gemv_kernel(const I8Args a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t codes[];  // [MX][whole KiB]
  __shared__ float row_scale[MX];
  __shared__ uint32_t red[MX][NW];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Kp = a.nk * kStep, nc = (Kp + 1023) >> 10, ldc = nc << 10;
  const int n0 = (blockIdx.x * NW + wave) * R;
  const uint8_t* wp[R];
#pragma unroll
  for (int r = 0; r < R; ++r) wp[r] = a.W + (size_t)min(n0 + r, a.N - 1) * a.rbw + 16 * lane;
  constexpr int U = 4;  // pieces in flight
  i32x4 q[U][R];
  auto load = [&](int u, int c) __attribute__((always_inline)) {
    const bool in = (c << 10) + 16 * lane < Kp;
#pragma unroll
    for (int r = 0; r < R; ++r)
      q[u][r] = in ? __builtin_nontemporal_load((const i32x4*)(wp[r] + ((size_t)c << 10))) : i32x4{0, 0, 0, 0};
  };
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < nc) load(u, u);

  using X = Rows<XT>;
  // With one row of W a wave, x is held in registers (all its loads on their way at once) where
  // they have room: 1 x 1024 x 5120 fp32 5.1 -> 4.5 us, two tokens 6.6 -> 5.5.  With two rows, whose
  // 16 waves would then need more than the 64 registers of two workgroups a CU, it is read twice:
  // 13.4 against 15.7 us at 1 x 14336 x 5120 bf16.
  constexpr int XR = 4, STEP = 64 * NW * X::EPU;
  const int k0 = tid * X::EPU;
  const bool held = R == 1 && a.K <= XR * STEP;
  auto row = [&](int m) { return a.X + (size_t)min(m, a.M - 1) * a.rbx; };
  u32x4 xu[MX][XR];
  uint32_t top[MX] = {};
  auto more = [&](int m, const u32x4& u) __attribute__((always_inline)) {
    float v[X::EPU];
    X::widen(u, v);
    top[m] = top_bits(v, top[m]);
  };
  if (held) {
#pragma unroll
    for (int m = 0; m < MX; ++m)
#pragma unroll
      for (int i = 0; i < XR; ++i) {
        const int k = k0 + i * STEP;
        xu[m][i] = k < a.K ? X::get(row(m), k, a.K) : u32x4{0u, 0u, 0u, 0u};
      }
#pragma unroll
    for (int m = 0; m < MX; ++m)
#pragma unroll
      for (int i = 0; i < XR; ++i) more(m, xu[m][i]);
  } else {
    for (int k = k0; k < a.K; k += STEP)
#pragma unroll
      for (int m = 0; m < MX; ++m) more(m, X::get(row(m), k, a.K));
  }
#pragma unroll
  for (int m = 0; m < MX; ++m) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top[m] = max(top[m], (uint32_t)__shfl_xor((int)top[m], o, 64));
    if (lane == 0) red[m][wave] = top[m];
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MX; ++m) {
#pragma unroll
    for (int w = 0; w < NW; ++w) top[m] = max(top[m], red[m][w]);
    const RowScale s = row_scale_of(top[m]);
    if (tid == 0) row_scale[m] = s.sc;
    auto put = [&](int k, const u32x4& u) __attribute__((always_inline)) {
      float v[X::EPU];
      X::widen(u, v);
      uint8_t* to = codes + m * ldc + k;
      if constexpr (X::EPU == 8) *(u32x2*)to = u32x2{codes4(v, s), codes4(v + 4, s)};
      else *(uint32_t*)to = codes4(v, s);
    };
    if (held) {
#pragma unroll
      for (int i = 0; i < XR; ++i)
        if (k0 + i * STEP < Kp) put(k0 + i * STEP, xu[m][i]);
    } else {
      for (int k = k0; k < Kp; k += STEP) put(k, k < a.K ? X::get(row(m), k, a.K) : u32x4{0u, 0u, 0u, 0u});
    }
  }
  __syncthreads();

  // this lane's channel.  Two rows a wave ask for its scale while W comes (1 x 14336 x 5120 13.4 -> 13.3
  // us); with one, asking at the end was faster (1 x 1024 x 5120 4.15 us against 4.26).
  const int n = n0 + (lane >> 4) * R / 4;
  const bool stores = (lane & 15) == 0 && lane % (64 / R) == 0 && n < a.N;
  const float early_s = R > 1 && stores ? a.sw[n] : 0.f, early_b = R > 1 && stores && a.bias ? a.bias[n] : 0.f;
  int acc[MX][R] = {};
  for (int c0 = 0; c0 < nc; c0 += U)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u;
      if (c >= nc) break;
#pragma unroll
      for (int m = 0; m < MX; ++m) {
        // past the padded row both sides may be anything but the weight, which is 0
        const i32x4 x = *(const i32x4*)(codes + m * ldc + (c << 10) + 16 * lane);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][r] = __builtin_amdgcn_sdot4(q[u][r][i], x[i], acc[m][r], false);
      }
      if (c + U < nc) load(u, c + U);
    }
  using Y = Rows<YT>;
#pragma unroll
  for (int m = 0; m < MX; ++m) {
    const int sum = wave_sums<R>(acc[m]);
    if (m < a.M && stores) {
      const float cs = R > 1 ? early_s : a.sw[n], cb = R > 1 ? early_b : a.bias ? a.bias[n] : 0.f;
      const float v[4] = {scaled(sum, row_scale[m], cs, cb), 0.f, 0.f, 0.f};
      Y::put4(a.Y + (size_t)m * a.ldy + (size_t)n * Y::ES, v, 1);
    }
  }
}

template <int YT, int XT, int MX, int R, int NW>
int launch_gemv(const I8Args& a, hipStream_t s, const char* who) {
  const int ldc = (a.nk * kStep + 1023) / 1024 * 1024;
  i8_gemv_kernel<YT, XT, MX, R, NW><<<(a.N + NW * R - 1) / (NW * R), 64 * NW, MX * ldc, s>>>(a);
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

// Few rows: the product is bound by the bytes of W.  A workgroup takes a BM x BN tile; its
// WVN x WVK waves share the columns and the 64-byte steps of a stage, which holds KS * 128 bytes
// of every row.  A ring of S stages keeps S - 1 on their way by global_load_lds, whole lines of
// eight rows a load; one barrier a stage.
//
// A lone workgroup streams 60-80 GB/s into its CU (a plain loop of such loads out of L2: 131; 16
// rows of 64 bytes straight to registers: 38), so few columns take small tiles, and long stages,
// whose steps the waves share: 8 x 1024 x 5120 5.0 us on 16 x 16, 10.6 on 16 x 64, 14.1 on 128 x 64.
// With columns enough W's bytes bound it: 8 x 14336 x 5120 12.2 us (6.0 TB/s), routed experts of
// 8 tokens (16 x 64) 5.5 TB/s.  Waves that share only K read each operand once: 32 x 32 1 x 8
// waves 6.4 us against 7.1 of 2 x 8 at 8 x 1024 x 5120.  Rings of 6 and 8 stages were no faster.
template <int YT, int BM, int BN, int WVN, int WVK, int KS, int S, bool GROUPED>
__global__ __launch_bounds__(64 * WVN * WVK) void i8_tile_kernel(const I8Args a) {
  constexpr int NW = WVN * WVK, MB = BM / 16, NB = BN / WVN / 16, KK = 2 * KS / WVK;
  constexpr int SUB = (BM + BN) * kStep, STAGE = KS * SUB, INST = STAGE / 1024 / NW;
  static_assert(INST * NW * 1024 == STAGE && KK * WVK == 2 * KS && NB * WVN * 16 == BN, "whole loads, steps and blocks a wave");
  constexpr int LDO = BN + 4;  // dwords of a row of sums
  static_assert(WVK * BM * LDO * 4 <= S * STAGE, "sums in LDS");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Tile tl;
  if (!find_tile<BM, BN, GROUPED>(a, tl)) return;
  const int n0 = tl.tn * BN;
  using Y = Rows<YT>;
  if (GROUPED && tl.e == a.E) return zero_tile<Y, BN, 64 * NW>(a, tl, n0);
  const float* sw = a.sw + (GROUPED ? (size_t)tl.e * a.N : 0);

  // load u of this wave: eight rows of a sub-stage (X's, then W's)
  const uint8_t* src[INST];
#pragma unroll
  for (int u = 0; u < INST; ++u) {
    const int r = (8 * (wave + NW * u) + (lane >> 3)) % (BM + BN);
    src[u] = stage_row<BM, GROUPED>(a, tl, n0, r) + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
  }
  const uint32_t lds0 = lds_addr(lds);
  const int ns = (a.nk + KS - 1) / KS;
  int put = 0;
  auto issue = [&](int st) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < INST; ++u) {
      const int i = 8 * (wave + NW * u), r = i % (BM + BN);
      // steps past the end load the last one again, and are not multiplied
      const size_t k = (size_t)(KS == 1 ? st : min(st * KS + i / (BM + BN), a.nk - 1)) * kStep;
      const uint32_t to = lds0 + put * STAGE + (wave + NW * u) * 1024;
      if (tl.once && r >= BM) dma16_nt(src[u] + k, to);
      else dma16(src[u] + k, to);
    }
    put = put + 1 == S ? 0 : put + 1;
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < ns) issue(i);

  i32x4 acc[NB][MB] = {};
  const int wn = wave % WVN, wk = wave / WVN, fr = lane & 15, fg = lane >> 4, turn = (fr >> 1) & 7;
  int get = 0;
  for (int st = 0; st < ns; ++st) {
    const int after = ns - 1 - st;  // stages on their way behind this one
    if (after >= S - 2) vm_wait<(S - 2) * INST>();
    else wait_stages<S - 3, INST>(after);
    __syncthreads();  // stage st has landed for every wave, and the one before it is read
    if (st + S - 1 < ns) issue(st + S - 1);
    const uint8_t* s = lds + get * STAGE;
    get = get + 1 == S ? 0 : get + 1;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      const int step = wk * KK + k, sub = step >> 1;
      if (KS > 1 && st * KS + sub >= a.nk) break;
      const uint8_t* p = s + sub * SUB + fr * kStep + ((4 * (step & 1) + fg) ^ turn) * 16;
      i32x4 xf[MB], wf[NB];
#pragma unroll
      for (int i = 0; i < MB; ++i) xf[i] = *(const i32x4*)(p + i * 16 * kStep);
#pragma unroll
      for (int j = 0; j < NB; ++j) wf[j] = *(const i32x4*)(p + (BM + (wn * NB + j) * 16) * kStep);
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
          acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[i], acc[j][i], 0, 0, 0);
    }
  }
  __syncthreads();
  // a lane's sum is columns 4 * fg .. + 3 of row fr of each block
  int32_t* sums = (int32_t*)lds;
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i)
      *(i32x4*)(sums + (wk * BM + i * 16 + fr) * LDO + (wn * NB + j) * 16 + 4 * fg) = acc[j][i];
  __syncthreads();
  for (int q = tid; q < BM * BN / 4; q += 64 * NW) {
    const int r = q / (BN / 4), c = q % (BN / 4) * 4, m = tl.m0 + r, n = n0 + c;
    if (m >= tl.m1 || n >= a.N) continue;
    i32x4 v = *(const i32x4*)(sums + r * LDO + c);
#pragma unroll
    for (int w = 1; w < WVK; ++w) v += *(const i32x4*)(sums + (w * BM + r) * LDO + c);
    const int xr = source_row<GROUPED>(a, m);
    const float sc = xr < 0 ? 0.f : a.sx[xr];
    float o[4], cs[4], cb[4];
    bool near = true;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int nn = min(n + k, a.N - 1);
      cs[k] = sw[nn];
      cb[k] = a.bias ? a.bias[nn] : 0.f;
      o[k] = scaled_near(v[k], sc, cs[k], cb[k]);
      near &= normal(sc * cs[k]);
    }
    if (__builtin_expect(!near, 0)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = xr < 0 ? 0.f : scaled(v[k], sc, cs[k], cb[k]);
    }
    Y::put4(a.Y + (size_t)m * a.ldy + (size_t)n * Y::ES, o, min(4, a.N - n));
  }
}

template <int YT, int BM, int BN, int WVN, int WVK, int KS, int S, bool GROUPED>
int launch_tile(const I8Args& a, hipStream_t s, const char* who) {
  constexpr int LDS = S * KS * (BM + BN) * kStep;
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static std::atomic<uint64_t> done{0};
  return launch(i8_tile_kernel<YT, BM, BN, WVN, WVK, KS, S, GROUPED>, done, a, GROUPED, BM, BN, 64 * WVN * WVK, LDS, s,
                who);
}

// The tiles, and what one costs: a call takes about t0 + K / 1024 * max(one, each * n) us, n the
// tiles that the fullest CU runs.  `one` is a tile alone on its CU (its loads' latency),
// `each` what another adds (the CU's share of the stream, or its MFMAs).  Fitted to measured
// times of 104 sizes (8 to 4096 rows, 500 to 28672 columns, K of 1000 to 14336) on weights that
// the last-level cache holds; the tile with the least such time is within 2 % of the best of
// twenty in the mean, 19 % at worst.  Example, 5120 x 5120, us: 8 rows 16 x 32 tiles 6.1, 64 x 64
// 11.4, 128 x 128 17.9; 64 rows 32 x 64 9.1, 64 x 64 11.8, 16 x 16 13.6; 512 rows 128 x 128 19.8,
// 64 x 64 28.2, 256 x 256 55.9; 4096 rows 256 x 320 89.7, 128 x 128 120, 256 x 256 124.
struct TileCost {
  int bm, bn;
  float t0, one, each;
};
constexpr TileCost kTiles[] = {
    {16, 16, 3.4f, 0.39f, 0.50f},  {16, 32, 3.2f, 0.77f, 0.92f},   {16, 64, 3.1f, 1.54f, 1.33f},
    {32, 32, 3.3f, 0.74f, 0.93f},  {32, 64, 3.8f, 1.19f, 1.43f},   {64, 64, 3.2f, 1.86f, 1.75f},
    {128, 64, 2.8f, 2.55f, 2.80f}, {128, 128, 2.9f, 3.30f, 3.75f}, {256, 128, 3.5f, 5.83f, 6.75f},
    {256, 192, 2.2f, 6.62f, 9.86f}, {256, 256, 4.6f, 0.18f, 11.6f}, {256, 320, 4.3f, 11.1f, 14.1f},
};

int pick_tile(const I8Args& a, int cus) {
  int best = 0;
  float least = 1e30f;
  for (int i = 0; i < (int)(sizeof kTiles / sizeof kTiles[0]); ++i) {
    const TileCost& c = kTiles[i];
    const float n = std::ceil(std::ceil((float)a.M / c.bm) * ((a.N + c.bn - 1) / c.bn) / cus);
    const float t = c.t0 + a.nk * (kStep / 1024.f) * std::max(c.one, c.each * n);
    if (t < least) least = t, best = i;
  }
  return best;
}

// Grouped, a call takes about max(n * (fix + K / 1024 * each), stream * MB of W) us and the launch: the
// experts' weights come from memory, past the last-level cache, and a tile costs the MFMAs of its
// filled blocks and, around its K loop, `fix`.  Fitted to 60 sizes (1 to 160 experts, 1 to 1300 rows
// each, K of 130 to 14336, W of 0.1 to 1300 MB) and to uniform routing: the tile with the least such
// time is within 1.7 % of the best in the mean, 21 % at worst; with the costs above, 8 and 58 %.
// The other tiles were hardly ever the best here.  Example, 64 experts of 2816 x 2048, us:
// 4 rows each 16 x 64 tiles 63, 64 x 64 72, 256 x 256 90; 32 rows 64 x 64 82, 128 x 128 93; 188 rows
// 256 x 256 130, 128 x 128 181, 64 x 64 240.
struct GroupedCost {
  int tile;  // of kTiles
  float fix, each, stream;
};
constexpr GroupedCost kGroupedTiles[] = {
    {0, 0.85f, 0.52f, 0.23f}, {2, 1.15f, 1.35f, 0.175f}, {5, 1.1f, 1.88f, 0.18f},  {7, 2.5f, 5.2f, 0.20f},
    {8, 4.0f, 6.6f, 0.22f},   {9, 2.9f, 10.7f, 0.23f},   {10, 3.7f, 12.1f, 0.235f}, {11, 4.3f, 14.3f, 0.28f},
};

// Tiles of bm rows that an expert of `mean` rows is expected to need where every row chooses by
// itself, its rows then spread by sqrt(mean) (the normal distribution's tail as a logistic one).
float tiles_of(float mean, int bm) {
  const float j = std::floor(mean / bm);
  auto above = [&](float rows) { return 1.f / (1.f + std::exp(-1.7f * (mean - rows) / std::sqrt(mean))); };
  return j + (j > 0.f ? above(j * bm) : 1.f) + above((j + 1) * bm);
}

// The offsets are on the device: the rows are taken as independent choices of the experts, dropped
// ones among them.  Measured where they are not: 2048 tokens, top 8 of 64, 2816 x 2048 169 us, with
// experts' logits of a spread of 1 (the fullest 5 to 7 times the mean) 165, with half of the pairs
// dropped 157 (their rows of Y are cleared).
int pick_grouped_tile(const I8Args& a, int cus) {
  const float used = a.E * (1.f - std::exp(-(float)a.M / a.E)), mean = a.M / used;
  const float mb = used * a.N * a.nk * (kStep * 1e-6f);
  int best = 0;
  float least = 1e30f;
  for (const GroupedCost& c : kGroupedTiles) {
    const TileCost& z = kTiles[c.tile];
    const float n = std::ceil(used * tiles_of(mean, z.bm) * ((a.N + z.bn - 1) / z.bn) / cus);
    const float t = std::max(n * (c.fix + a.nk * (kStep / 1024.f) * c.each), c.stream * mb);
    if (t < least) least = t, best = c.tile;
  }
  return best;
}

template <int YT, bool GROUPED>
int launch_picked(int tile, const I8Args& a, hipStream_t s, const char* who) {
  if constexpr (!GROUPED) switch (tile) {
      case 1: return launch_tile<YT, 16, 32, 1, 8, 4, 4, false>(a, s, who);
      case 3: return launch_tile<YT, 32, 32, 1, 8, 4, 4, false>(a, s, who);
      case 4: return launch_tile<YT, 32, 64, 1, 8, 4, 3, false>(a, s, who);
      case 6: return launch_gemm<YT, 128, 64, 4, 2, 4, false>(a, s, who);
    }
  switch (tile) {
    case 0: return launch_tile<YT, 16, 16, 1, 8, 4, 4, GROUPED>(a, s, who);
    case 2: return launch_tile<YT, 16, 64, 2, 2, 2, 4, GROUPED>(a, s, who);
    case 5: return launch_gemm<YT, 64, 64, 2, 2, 4, GROUPED>(a, s, who);
    case 7: return launch_gemm<YT, 128, 128, 2, 4, 4, GROUPED>(a, s, who);
    case 8: return launch_gemm<YT, 256, 128, 4, 2, 3, GROUPED>(a, s, who);
    case 9: return launch_gemm<YT, 256, 192, 4, 2, 2, GROUPED>(a, s, who);
    case 10: return launch_gemm<YT, 256, 256, 4, 2, 2, GROUPED>(a, s, who);
    default: return launch_gemm<YT, 256, 320, 4, 2, 2, GROUPED>(a, s, who);
  }
}

int gemm(const I8Args& a, int ytype, bool grouped, hipStream_t s, const char* who) {
  int cus = 0, st = device_cus(&cus);
  if (st != TIERMM_OK) return st;
  const int tile = grouped ? pick_grouped_tile(a, cus) : pick_tile(a, cus);
  with_rows(ytype, [&](auto yt) {
    constexpr int YT = decltype(yt)::value;
    st = grouped ? launch_picked<YT, true>(tile, a, s, who) : launch_picked<YT, false>(tile, a, s, who);
  });
  return st;
}

// One or two rows of x are quantized by the product's own workgroups (the GEMV): a launch less,
// and each byte of W in whole lines.
constexpr int kGemvLds = 60 * 1024;
bool fuses(int M, int K) { return M <= 2 && M * (padded(K) + 1024) <= kGemvLds; }

// Below 5120 columns a wave takes one row of W and a workgroup is 8 waves, from there up two and
// 16.  Of 96 sizes (1 and 2 tokens, 512 to 14336 columns, K of 2048 to 14336, bf16 and fp32) this
// takes the faster form in 84 and is 1 to 14 % behind it in 12 (the most at 1 x 5120 x 14336 bf16, 16.6
// us against 14.6).  Us of one row and of two, bf16: 1 x 1024 x 5120 4.6 and 6.3, 1 x 4096 x 5120 6.6
// and 7.1, 1 x 5120 x 5120 7.8 and 7.6, 2 x 5120 x 5120 10.1 and 8.8, 1 x 14336 x 5120 15.5 and 14.1.
int fused(const I8Args& a, int xtype, int ytype, hipStream_t s, const char* who) {
  int st = TIERMM_OK;
  with_rows(ytype, [&](auto yt) {
    with_rows(xtype, [&](auto xt) {
      constexpr int YT = decltype(yt)::value, XT = decltype(xt)::value;
      auto rows = [&](auto mx) {
        constexpr int MX = decltype(mx)::value;
        if (a.N < 5120) st = launch_gemv<YT, XT, MX, 1, 8>(a, s, who);
        else st = launch_gemv<YT, XT, MX, 2, 16>(a, s, who);
      };
      if (a.M == 1) rows(std::integral_constant<int, 1>());
      else rows(std::integral_constant<int, 2>());
    });
  });
  return st;
}

// Rows up to which a row gets 1024 threads: few rows wait for their latency.  4096 rows of
// 5120 bf16: 11.5 us (5.5 TB/s) with 256 threads a row, 16.3 with 1024; of 14336 fp32, whose
// registers 256 threads do not hold: 20.8 (2000 rows, 6.9 TB/s) against 27.7 read twice.
constexpr int kQuantWide = 512;

int quant(const void* x, int xtype, size_t ldx, int8_t* q, size_t rb, float* scale, int M, int K, hipStream_t s,
          const char* who) {
  const size_t ld = ldx * row_elem_bytes(xtype);
  const uint8_t* p = (const uint8_t*)x;
  const int Kp = padded(K);
  with_rows(xtype, [&](auto xt) {
    constexpr int XT = decltype(xt)::value;
    const int units = Kp / Rows<XT>::EPU;
#define QUANT(NT, R) i8_quant_kernel<XT, NT, R><<<M, NT, 0, s>>>(p, ld, q, rb, scale, K, Kp)
    if (M <= kQuantWide) {
      if (units <= 1024) QUANT(1024, 1);
      else if (units <= 2048) QUANT(1024, 2);
      else if (units <= 4096) QUANT(1024, 4);
      else QUANT(1024, 0);
    } else {
      if (units <= 512) QUANT(256, 2);
      else if (units <= 1024) QUANT(256, 4);
      else if (units <= 2048) QUANT(256, 8);
      else if (units <= 4096) QUANT(1024, 4);
      else QUANT(1024, 0);
    }
#undef QUANT
  });
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

// Checks of the sizes, and of one side's rows.
int check_size(const char* who, int M, int N, int K) {
  if (M < 0 || N < 0 || K < 1) return set_error(TIERMM_EINVAL, "%s: bad size %d x %d x %d", who, M, N, K);
  if (K > kMaxK) return set_error(TIERMM_UNSUPPORTED, "%s: K = %d, at most %d", who, K, kMaxK);
  if (M > (1 << 23)) return set_error(TIERMM_UNSUPPORTED, "%s: %d rows, at most %d", who, M, 1 << 23);
  if (N > (1 << 26)) return set_error(TIERMM_UNSUPPORTED, "%s: %d columns, at most %d", who, N, 1 << 26);
  return TIERMM_OK;
}
int check_i8_rows(const char* who, const char* what, const void* p, size_t rb, int K) {
  if (!p) return set_error(TIERMM_EINVAL, "%s: null %s", who, what);
  if (bad_stride(rb, padded(K)) || rb % 16 || misaligned(p, 16))
    return set_error(TIERMM_EINVAL, "%s: %s rows of %zu bytes (whole 16-byte units from %d up, 16-byte aligned)", who,
                     what, rb, padded(K));
  return TIERMM_OK;
}
int check_out(const char* who, const void* Y, int ytype, size_t ldy, int N) {
  const int es = row_elem_bytes(ytype);
  if (!es) return set_error(TIERMM_UNSUPPORTED, "%s: output of type %d", who, ytype);
  if (bad_stride(ldy, N)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, N);
  if (!Y || misaligned(Y, es)) return set_error(TIERMM_EINVAL, "%s: null or misaligned output", who);
  return TIERMM_OK;
}

}  // namespace
}  // namespace tiermm

using namespace tiermm;

extern "C" {

size_t tiermm_i8_row_bytes(int K) { return K < 1 || K > kMaxK ? 0 : (size_t)padded(K); }

int tiermm_i8_quant(const void* x, int xtype, size_t ldx, int8_t* q, size_t rb, float* scale, int M, int K,
                    tiermm_stream_t stream) {
  const char* who = "tiermm_i8_quant";
  int st = check_size(who, M, 0, K);
  if (st != TIERMM_OK) return st;
  const int es = row_elem_bytes(xtype);
  if (!es) return set_error(TIERMM_UNSUPPORTED, "%s: rows of type %d", who, xtype);
  if (bad_stride(ldx, K)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, K);
  if (M == 0) return TIERMM_OK;
  if (!x || misaligned(x, es) || !scale || misaligned(scale, 4))
    return set_error(TIERMM_EINVAL, "%s: null or misaligned buffer", who);
  st = check_i8_rows(who, "int8", q, rb, K);
  if (st != TIERMM_OK) return st;
  return quant(x, xtype, ldx, q, rb, scale, M, K, (hipStream_t)stream, who);
}

int tiermm_i8_gemm(const int8_t* Xq, size_t rbx, const float* sx, const int8_t* W, size_t rbw, const float* sw,
                   const float* bias, void* Y, int ytype, size_t ldy, int M, int N, int K, tiermm_stream_t stream) {
  const char* who = "tiermm_i8_gemm";
  int st = check_size(who, M, N, K);
  if (st != TIERMM_OK || M == 0 || N == 0) return st;
  if ((st = check_out(who, Y, ytype, ldy, N)) != TIERMM_OK) return st;
  if ((st = check_i8_rows(who, "x", Xq, rbx, K)) != TIERMM_OK) return st;
  if ((st = check_i8_rows(who, "weight", W, rbw, K)) != TIERMM_OK) return st;
  if (!sx || !sw || misaligned(sx, 4) || misaligned(sw, 4) || misaligned(bias, 4))
    return set_error(TIERMM_EINVAL, "%s: null or misaligned scales", who);
  const I8Args a = {(const uint8_t*)Xq, sx, (const uint8_t*)W, sw, bias, (uint8_t*)Y, rbx, rbw,
                    ldy * row_elem_bytes(ytype), M, N, K, padded(K) / kStep, nullptr, nullptr, 0, 1, M, 1};
  return gemm(a, ytype, false, (hipStream_t)stream, who);
}

size_t tiermm_i8_linear_ws_bytes(int M, int N, int K) {
  if (M < 1 || N < 1 || K < 1 || K > kMaxK) return 0;
  return (size_t)M * padded(K) + ((size_t)M * 4 + 15) / 16 * 16;
}

int tiermm_i8_linear(const void* x, int xtype, size_t ldx, const int8_t* W, size_t rbw, const float* sw,
                     const float* bias, void* Y, int ytype, size_t ldy, int M, int N, int K, void* ws, size_t ws_bytes,
                     tiermm_stream_t stream) {
  const char* who = "tiermm_i8_linear";
  int st = check_size(who, M, N, K);
  if (st != TIERMM_OK) return st;
  const int es = row_elem_bytes(xtype);
  if (!es) return set_error(TIERMM_UNSUPPORTED, "%s: x of type %d", who, xtype);
  if (bad_stride(ldx, K)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, K);
  if (M == 0 || N == 0) return TIERMM_OK;
  if (!x || misaligned(x, es)) return set_error(TIERMM_EINVAL, "%s: null or misaligned x", who);
  if ((st = check_out(who, Y, ytype, ldy, N)) != TIERMM_OK) return st;
  if ((st = check_i8_rows(who, "weight", W, rbw, K)) != TIERMM_OK) return st;
  if (!sw || misaligned(sw, 4) || misaligned(bias, 4))
    return set_error(TIERMM_EINVAL, "%s: null or misaligned scales", who);
  if (misaligned(ws, 16)) return set_error(TIERMM_EINVAL, "%s: workspace not 16-byte aligned", who);
  I8Args a = {(const uint8_t*)x, nullptr, (const uint8_t*)W, sw, bias, (uint8_t*)Y, ldx * es, rbw,
              ldy * row_elem_bytes(ytype), M, N, K, padded(K) / kStep, nullptr, nullptr, 0, 1, M, 1};
  if (fuses(M, K)) return fused(a, xtype, ytype, (hipStream_t)stream, who);
  void* w = nullptr;
  if ((st = get_workspace(ws, ws_bytes, tiermm_i8_linear_ws_bytes(M, N, K), &w, who)) != TIERMM_OK) return st;
  int8_t* q = (int8_t*)w;
  float* sx = (float*)(q + (size_t)M * padded(K));
  if ((st = quant(x, xtype, ldx, q, padded(K), sx, M, K, (hipStream_t)stream, who)) != TIERMM_OK) return st;
  a.X = (const uint8_t*)q;
  a.sx = sx;
  a.rbx = padded(K);
  return gemm(a, ytype, false, (hipStream_t)stream, who);
}

int tiermm_i8_gemm_grouped(const int8_t* Xq, size_t rbx, const float* sx, const int32_t* rows, int n_rows, int topk,
                           const int32_t* expert_offsets, int n_experts, const int8_t* W, size_t rbw, const float* sw,
                           void* Y, int ytype, size_t ldy, int P, int N, int K, tiermm_stream_t stream) {
  const char* who = "tiermm_i8_gemm_grouped";
  int st = check_size(who, P, N, K);
  if (st != TIERMM_OK) return st;
  if (n_rows < 0 || n_experts < 1 || topk < 1) return set_error(TIERMM_EINVAL, "%s: bad size", who);
  if (n_experts > TIERMM_MOE_MAX_EXPERTS)
    return set_error(TIERMM_UNSUPPORTED, "%s: %d experts, at most %d", who, n_experts, TIERMM_MOE_MAX_EXPERTS);
  if (P == 0 || N == 0) return TIERMM_OK;
  if ((st = check_out(who, Y, ytype, ldy, N)) != TIERMM_OK) return st;
  if (n_rows == 0) return set_error(TIERMM_EINVAL, "%s: no rows of x", who);
  if ((st = check_i8_rows(who, "x", Xq, rbx, K)) != TIERMM_OK) return st;
  if ((st = check_i8_rows(who, "weight", W, rbw, K)) != TIERMM_OK) return st;
  if (!expert_offsets || !sx || !sw || misaligned(sx, 4) || misaligned(sw, 4) || misaligned(expert_offsets, 4) ||
      misaligned(rows, 4))
    return set_error(TIERMM_EINVAL, "%s: null or misaligned table", who);
  const I8Args a = {(const uint8_t*)Xq, sx, (const uint8_t*)W, sw, nullptr, (uint8_t*)Y, rbx, rbw,
                    ldy * row_elem_bytes(ytype), P, N, K, padded(K) / kStep, expert_offsets, rows, n_experts, topk, n_rows, 1};
  return gemm(a, ytype, true, (hipStream_t)stream, who);
}

}  // extern "C"
