// i8.hip -- products of 8-bit integers with a scale for each row of either side:
// Y[m][n] = sx[m] sw[n] sum_k Xq[m][k] Wq[n][k] (+ bias[n]), and the quantizer that
// makes such rows.  No reference function (the reference's own 8-bit form is q8_0,
// whose activations stay fp32).
//
// The sum is a whole number, exact in int32 for K <= 133152 (2^31 / 127^2), so neither
// the tile, the order of K nor a split of it changes a result: one rounding of the sum
// to fp32, two products, the bias, and the output's own rounding.
//
// An int8 row is padded with zeros to whole 128-byte steps (i8_row_bytes), so no kernel
// has a K tail: padding of x adds zeros whatever the padding of W holds.
#include "tm_rows.h"

#include <algorithm>

namespace tiermm {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 128;          // bytes of K a row holds a step
constexpr int kMaxK = 133120;       // whole steps below 2^31 / 127^2

constexpr int padded(int K) { return (K + kStep - 1) / kStep * kStep; }

// ------------------------------------------------------------------- quantizer
// Scale of a row whose largest magnitude has the fp32 bits `top`, and what its elements
// are multiplied with: inv = 127 / max, sc = max / 127.  A NaN or an infinity makes the
// scale NaN and the codes 0, so every product of the row is NaN.  Magnitudes under
// 2^-100 are first scaled up (exactly) by 2^100: 127 / max would overflow.
struct RowScale {
  float pre, inv, sc;
};
__device__ __forceinline__ RowScale row_scale_of(uint32_t top) {
  RowScale r = {1.f, 0.f, 0.f};
  if (top >= 0x7f800000u) {
    r.sc = __uint_as_float(0x7fc00000u);
  } else if (top) {
    const float m = __uint_as_float(top);
    r.pre = m < 0x1p-100f ? 0x1p100f : 1.f;
    r.inv = 127.f / (m * r.pre);
    r.sc = m / 127.f;
  }
  return r;
}

// Codes of 4 elements, packed: rint(x * inv), nearest even.
__device__ __forceinline__ uint32_t codes4(const float* v, const RowScale& r) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // a scale of 0 or NaN has inv = 0: codes 0, whatever the element
    const float f = r.inv == 0.f ? 0.f : __builtin_rintf((v[i] * r.pre) * r.inv);
    w |= ((uint32_t)(int)f & 0xffu) << (8 * i);
  }
  return w;
}

template <int N>
__device__ __forceinline__ uint32_t top_bits(const float (&v)[N], uint32_t top) {
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  return top;
}

// One row a workgroup, read twice.
template <int XT>
__global__ __launch_bounds__(256) void i8_quant_kernel(const uint8_t* __restrict__ x, size_t ldx,
                                                       int8_t* __restrict__ q, size_t rb, float* __restrict__ scale,
                                                       int K, int Kp) {
  using R = Rows<XT>;
  __shared__ uint32_t red[4];
  const uint8_t* row = x + (size_t)blockIdx.x * ldx;
  uint32_t top = 0;
  for (int c = threadIdx.x * R::EPU; c < K; c += 256 * R::EPU) {
    float v[R::EPU];
    R::widen(R::get(row, c, K), v);
    top = top_bits(v, top);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  const RowScale r = row_scale_of(max(max(red[0], red[1]), max(red[2], red[3])));
  int8_t* out = q + (size_t)blockIdx.x * rb;
  for (int c = threadIdx.x * R::EPU; c < Kp; c += 256 * R::EPU) {
    float v[R::EPU] = {};
    if (c < K) R::widen(R::get(row, c, K), v);
#pragma unroll
    for (int i = 0; i < R::EPU; i += 4) *(uint32_t*)(out + c + i) = codes4(v + i, r);
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
};

// The rows of Y that a workgroup's tile covers.
struct Tile {
  int m0, m1, tn;   // rows [m0, m1), column tile
  int e;            // expert; E: rows that no expert has, which become zeros
};

// Tile `t` of the workgroups' sequence in which XCD x (blockIdx % 8) walks the x-th
// contiguous share, or -1 past the end.
__device__ __forceinline__ int xcd_share(int bid, int total) {
  const int x = bid & 7, i = bid >> 3, each = total >> 3, more = total & 7;
  return i < each + (x < more) ? x * each + min(x, more) + i : -1;
}

template <int BM>
__device__ __forceinline__ bool grouped_tile(const I8Args& a, int ntn, int bid, Tile& tl) {
  const int lane = threadIdx.x & 63, P = a.M;
  auto begin = [&](int e) { return min(max(a.off[e], 0), P); };
  // rows of group e0 + lane (group E: from off[E] to P)
  auto rows_of = [&](int e, int& b) {
    b = e <= a.E ? begin(e) : P;
    const int n = e < a.E ? begin(e + 1) - b : e == a.E ? P - b : 0;
    return max(n, 0);
  };
  int total = 0;
  for (int e0 = 0; e0 <= a.E; e0 += 64) {
    int b;
    int n = (rows_of(e0 + lane, b) + BM - 1) / BM;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    total += n;
  }
  const int t = xcd_share(bid, total * ntn);
  if (t < 0) return false;
  int run = 0;
  for (int e0 = 0; e0 <= a.E; e0 += 64) {
    int b;
    const int rows = rows_of(e0 + lane, b), n = (rows + BM - 1) / BM * ntn;
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
      return true;
    }
    run += __shfl(s, 63, 64);
  }
  return false;
}

// Row of X behind row p of Y, or -1.
__device__ __forceinline__ int source_row(const I8Args& a, int p) {
  if (!a.rows) return p < a.xrows ? p : -1;
  const int i = a.rows[p];
  const int r = i < 0 ? -1 : i / a.topk;
  return r < a.xrows ? r : -1;
}

// One element of Y: the sum rounded to fp32, times sx * sw, plus the bias (0: none).
__device__ __forceinline__ float scaled(int sum, float sx, float sw, float bias) {
  return fmaf((float)sum, sx * sw, bias);
}

// LDS place of byte `o` of row r of CH 16-byte chunks: neighbouring rows' chunks are
// spread over the 16 chunks that the banks span.
template <int CH>
__device__ __forceinline__ int out_place(int r, int o) {
  const int c = o >> 4, turn = CH >= 16 ? r : r / (16 / CH);
  return r * CH * 16 + ((c ^ (turn & (CH - 1))) << 4) + (o & 15);
}
// One wave's LDS operations are in order; the compiler must keep them so too.
__device__ __forceinline__ void wave_lds_wait() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// BM rows of X times BN rows of W by WVM x WVN waves of WM x WN blocks of 32 x 32.
//
// A stage is 128 bytes of every row, brought to LDS by global_load_lds; two stages take
// turns.  A row's 16-byte chunk c lies at slot c ^ ((row >> 1) & 7): the 16 rows that one
// cycle of a fragment read touches then cover all the banks.  A stage is four MFMA
// steps of K = 32.  While the products of one step run, the fragments of the next come in,
// one read between two MFMAs, and the loads of the stage after next go out, spread the same
// way from the step after the barrier that frees their place on.
//
// W is the MFMA's first operand, so a lane holds four neighbouring columns of one row of Y.
template <int YT, int BM, int BN, int WVM, int WVN, bool GROUPED>
__global__ __launch_bounds__(64 * WVM * WVN) void i8_gemm_kernel(const I8Args a) {
  constexpr int NW = WVM * WVN, WM = BM / WVM / 32, WN = BN / WVN / 32, NM = WM * WN, NF = WM + WN;
  constexpr int STAGE = (BM + BN) * kStep, INST = STAGE / 1024 / NW;
  static_assert(WM * WVM * 32 == BM && WN * WVN * 32 == BN && INST * NW * 1024 == STAGE, "whole blocks and loads a wave");
  // loads of a stage by the step that issues them: 3 (of the stage before last), 0 and 1
  constexpr int D0 = (INST + 2) / 3, D1 = (INST - D0 + 1) / 2, D2 = INST - D0 - D1;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  float* col_scale = (float*)(lds + 2 * STAGE);
  float* col_bias = col_scale + BN;
  float* row_scale = col_bias + BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ntn = (a.N + BN - 1) / BN;

  Tile tl;
  if constexpr (GROUPED) {
    if (!grouped_tile<BM>(a, ntn, blockIdx.x, tl)) return;
  } else {
    const int ntm = (a.M + BM - 1) / BM, t = xcd_share(blockIdx.x, ntm * ntn);
    if (t < 0) return;
    constexpr int GM = 4;  // groups of 4 tile rows, column by column
    const int grp = t / (GM * ntn), first = grp * GM, gm = min(GM, ntm - first), in = t - grp * GM * ntn;
    tl.m0 = (first + in % gm) * BM;
    tl.m1 = min(tl.m0 + BM, a.M);
    tl.tn = in / gm;
    tl.e = 0;
  }
  const int n0 = tl.tn * BN;
  using Y = Rows<YT>;

  if (GROUPED && tl.e == a.E) {  // rows of no expert
    const int cols = min(BN, a.N - n0);
    for (int m = tl.m0; m < tl.m1; ++m)
      for (int c = tid * Y::EPU; c < cols; c += 64 * NW * Y::EPU)
        Y::set(a.Y + (size_t)m * a.ldy + (size_t)n0 * Y::ES, c, cols, u32x4{0u, 0u, 0u, 0u});
    return;
  }
  const uint8_t* W = a.W + (GROUPED ? (size_t)tl.e * a.N * a.rbw : 0);
  const float* sw = a.sw + (GROUPED ? (size_t)tl.e * a.N : 0);

  // load u of this wave: rows 8 * (wave + NW * u) .. + 7 of the stage (X's, then W's)
  const uint8_t* src[INST];
  const int slot = lane & 7, lr = lane >> 3;
#pragma unroll
  for (int u = 0; u < INST; ++u) {
    const int r = 8 * (wave + NW * u) + lr, c = slot ^ ((r >> 1) & 7);
    if (r < BM) {
      const int m = min(tl.m0 + r, tl.m1 - 1);
      const int xr = GROUPED ? max(source_row(a, m), 0) : m;
      src[u] = a.X + (size_t)xr * a.rbx + c * 16;
    } else {
      src[u] = W + (size_t)min(n0 + r - BM, a.N - 1) * a.rbw + c * 16;
    }
  }
  const uint32_t lds0 = lds_addr(lds);
  auto issue = [&](int kt, int u) __attribute__((always_inline)) {
    dma16(src[u] + (size_t)kt * kStep, lds0 + (kt & 1) * STAGE + (wave + NW * u) * 1024);
  };
#pragma unroll
  for (int u = 0; u < INST; ++u) issue(0, u);

  // the scales of the tile's rows and columns, for the end; NaN-free zeros where a row has no source
  for (int i = tid; i < BN; i += 64 * NW) {
    const int n = min(n0 + i, a.N - 1);
    col_scale[i] = sw[n];
    col_bias[i] = a.bias ? a.bias[n] : 0.f;
  }
  for (int i = tid; i < BM; i += 64 * NW) {
    const int m = min(tl.m0 + i, tl.m1 - 1), xr = GROUPED ? source_row(a, m) : m;
    row_scale[i] = xr < 0 ? 0.f : a.sx[xr];
  }

  i32x16 acc[WN][WM];
#pragma unroll
  for (int j = 0; j < WN; ++j)
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0;

  const int wm = wave % WVM, wn = wave / WVM, fr = lane & 31, fh = lane >> 5, turn = (fr >> 1) & 7;
  const uint32_t xrow = (uint32_t)(wm * WM * 32 + fr) * kStep, wrow = (uint32_t)(BM + wn * WN * 32 + fr) * kStep;
  i32x4 xf[2][WM], wf[2][WN];
  // fragment v of step kk of stage kt into set f: W's first, X's, W's others, as the products need them
  auto fragment = [&](int kt, int kk, int f, int v) __attribute__((always_inline)) {
    const uint8_t* s = lds + (kt & 1) * STAGE + ((2 * kk + fh) ^ turn) * 16;
    if (v >= 1 && v <= WM) xf[f][v - 1] = *(const i32x4*)(s + xrow + (v - 1) * 32 * kStep);
    else wf[f][v == 0 ? 0 : v - WM] = *(const i32x4*)(s + wrow + (v == 0 ? 0 : v - WM) * 32 * kStep);
  };
  // The products of fragments f, with the fragments (kt, kk) into the other set and loads
  // u0 .. u0 + n - 1 of stage `dt` between them.
  auto step = [&](int f, int kt, int kk, int dt, int u0, int n) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < NM; ++q) {
#pragma unroll
      for (int v = 0; v < NF; ++v)
        if (v * (NM - 2) / NF == q) fragment(kt, kk, f ^ 1, v);
#pragma unroll
      for (int d = 0; d < n; ++d)
        if (1 + d * (NM - 1) / n == q && dt < a.nk) issue(dt, u0 + d);
      const int j = q / WM, i = q % WM;
      acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[f][j], xf[f][i], acc[j][i], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  vm_wait<0>();
  __syncthreads();
  if (a.nk > 1) {
#pragma unroll
    for (int u = 0; u < D0; ++u) issue(1, u);
  }
#pragma unroll
  for (int v = 0; v < NF; ++v) fragment(0, 0, 0, v);
  for (int kt = 0; kt < a.nk; ++kt) {
    step(0, kt, 1, kt + 1, D0, D1);
    step(1, kt, 2, kt + 1, D0 + D1, D2);
    step(0, kt, 3, kt + 1, 0, 0);
    vm_wait<0>();
    __syncthreads();  // stage kt + 1 has landed for every wave, and stage kt is read
    // (past the end: the fragments of what the place holds, which nothing uses)
    step(1, kt + 1, 0, kt + 2, 0, D0);
  }

  // Element r of a block is column 8 * (r / 4) + 4 * fh + r % 4 of row fr: a lane's own
  // stores would be 4 columns wide.  Each wave passes 32 rows of one or two blocks at a
  // time through its part of LDS and stores whole 16-byte units, 8 of them a row.
  constexpr int JB = Y::ES == 2 ? 2 : 1, PART = 4096;
  static_assert(NW * PART <= 2 * STAGE, "rows of the epilogue in LDS");
  uint8_t* part = lds + wave * PART;
  auto store = [&](auto jn, int j0) __attribute__((always_inline)) {
    constexpr int J = decltype(jn)::value, CH = J * 32 * Y::ES / 16;
    const int cw = (wn * WN + j0) * 32, nw = n0 + cw;
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      const int rw = (wm * WM + i) * 32, mb = tl.m0 + rw;
      if (mb >= tl.m1) break;
      const float s = row_scale[rw + fr];
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int c = j * 32 + 8 * b + 4 * fh;
          const f32x4 cs = *(const f32x4*)(col_scale + cw + c), cb = *(const f32x4*)(col_bias + cw + c);
          f32x4 v;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = scaled(acc[j0 + j][i][4 * b + k], s, cs[k], cb[k]);
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
  __syncthreads();  // every wave has read its last stage
#pragma unroll
  for (int j0 = 0; j0 + JB <= WN; j0 += JB) store(std::integral_constant<int, JB>(), j0);
  if constexpr (WN % JB) store(std::integral_constant<int, WN % JB>(), WN - WN % JB);
}

template <int YT, int BM, int BN, int WVM, int WVN, bool GROUPED>
int launch_gemm(const I8Args& a, hipStream_t s, const char* who) {
  constexpr int LDS = 2 * (BM + BN) * kStep + (BM + 2 * BN) * 4;
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static std::atomic<uint64_t> done{0};
  auto* fn = i8_gemm_kernel<YT, BM, BN, WVM, WVN, GROUPED>;
  const int st = lds_attr_once(done, (const void*)fn, LDS, who);
  if (st != TIERMM_OK) return st;
  const long long ntn = (a.N + BN - 1) / BN;
  // grouped: every group may end in a partly filled tile
  const long long ntm = GROUPED ? a.M / BM + std::min(a.E, a.M) + 1 : (a.M + BM - 1) / BM;
  const long long grid = (ntm * ntn + 7) / 8 * 8;
  if (grid > (1ll << 22)) return set_error(TIERMM_UNSUPPORTED, "%s: %lld tiles", who, ntm * ntn);
  fn<<<(unsigned)grid, 64 * WVM * WVN, LDS, s>>>(a);
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

// Few rows: the product is bound by the bytes of W, each read once.  A workgroup takes 16 * NF
// rows of W and up to 16 * MT rows of X; its NW waves share K, wave w taking the 128-byte chunks
// w, w + NW, .. of every row.  Both operands go straight to registers (an MFMA 16x16x64 operand
// is 16 rows of 64 bytes), so nothing is staged and no wave waits for another until the end,
// where the waves' sums meet in LDS.
//
// XT >= 0: x comes as M <= 16 * MT rows of that type and the workgroup quantizes them into
// LDS itself, the weight's first chunks already on their way.
template <int YT, int XT, int MT, int NF, int NW, bool GROUPED>
__global__ __launch_bounds__(64 * NW) void i8_rows_kernel(const I8Args a) {
  constexpr bool FUSED = XT >= 0;
  constexpr int BN = 16 * NF, BM = 16 * MT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ntn = (a.N + BN - 1) / BN;
  Tile tl;
  if constexpr (GROUPED) {
    if (!grouped_tile<BM>(a, ntn, blockIdx.x, tl)) return;
  } else {
    tl = {0, a.M, (int)blockIdx.x, 0};
  }
  const int n0 = tl.tn * BN;
  using Y = Rows<YT>;
  if (GROUPED && tl.e == a.E) {  // rows of no expert
    const int cols = min(BN, a.N - n0);
    for (int m = tl.m0; m < tl.m1; ++m)
      for (int c = tid * Y::EPU; c < cols; c += 64 * NW * Y::EPU)
        Y::set(a.Y + (size_t)m * a.ldy + (size_t)n0 * Y::ES, c, cols, u32x4{0u, 0u, 0u, 0u});
    return;
  }
  const uint8_t* W = a.W + (GROUPED ? (size_t)tl.e * a.N * a.rbw : 0);
  const float* sw = a.sw + (GROUPED ? (size_t)tl.e * a.N : 0);

  const uint8_t* wp[NF];
  const uint8_t* xp[MT];
#pragma unroll
  for (int f = 0; f < NF; ++f) wp[f] = W + (size_t)min(n0 + 16 * f + r, a.N - 1) * a.rbw + 16 * g;
  if constexpr (!FUSED) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int m = min(tl.m0 + 16 * t + r, tl.m1 - 1);
      xp[t] = a.X + (size_t)(GROUPED ? max(source_row(a, m), 0) : m) * a.rbx + 16 * g;
    }
  }
  // operands of one chunk: two steps of 64 bytes
  struct Chunk {
    i32x4 w[2][NF], x[2][FUSED ? 1 : MT];
  };
  auto load = [&](Chunk& q, int c) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int f = 0; f < NF; ++f) q.w[h][f] = *(const i32x4*)(wp[f] + (size_t)c * kStep + 64 * h);
      if constexpr (!FUSED) {
#pragma unroll
        for (int t = 0; t < MT; ++t) q.x[h][t] = *(const i32x4*)(xp[t] + (size_t)c * kStep + 64 * h);
      }
    }
  };
  i32x4 acc[NF][MT] = {};
  uint8_t* codes = lds + NW * NF * MT * 1024;  // FUSED: [M][nk * 128]
  auto mul = [&](const Chunk& q, int c) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        i32x4 x;
        if constexpr (FUSED)
          x = *(const i32x4*)(codes + (size_t)min(16 * t + r, a.M - 1) * a.nk * kStep + c * kStep + 64 * h + 16 * g);
        else
          x = q.x[h][t];
#pragma unroll
        for (int f = 0; f < NF; ++f) acc[f][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.w[h][f], x, acc[f][t], 0, 0, 0);
      }
  };
  constexpr int U = MT + NF <= 2 ? 3 : MT + NF <= 3 ? 2 : 1;  // chunks in flight
  Chunk q[U];
  int c = wave;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c + u * NW < a.nk) load(q[u], c + u * NW);

  __shared__ float row_scale[BM];
  if constexpr (FUSED) {
    using X = Rows<XT < 0 ? QT_F32 : XT>;
    __shared__ uint32_t red[NW];
    const int K = a.K, Kp = a.nk * kStep;
    for (int m = 0; m < a.M; ++m) {
      const uint8_t* row = a.X + (size_t)m * a.rbx;
      uint32_t top = 0;
      for (int k = tid * X::EPU; k < K; k += 64 * NW * X::EPU) {
        float v[X::EPU];
        X::widen(X::get(row, k, K), v);
        top = top_bits(v, top);
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
      if (lane == 0) red[wave] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) top = max(top, red[w]);
      const RowScale s = row_scale_of(top);
      for (int k = tid * X::EPU; k < Kp; k += 64 * NW * X::EPU) {
        float v[X::EPU] = {};
        if (k < K) X::widen(X::get(row, k, K), v);
#pragma unroll
        for (int i = 0; i < X::EPU; i += 4) *(uint32_t*)(codes + (size_t)m * Kp + k + i) = codes4(v + i, s);
      }
      if (tid == 0) row_scale[m] = s.sc;
      __syncthreads();
    }
  } else {
    if (tid < BM) {
      const int m = min(tl.m0 + tid, tl.m1 - 1), xr = GROUPED ? source_row(a, m) : m;
      row_scale[tid] = xr < 0 ? 0.f : a.sx[xr];
    }
  }

  while (c < a.nk) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c >= a.nk) break;
      mul(q[u], c);
      if (c + U * NW < a.nk) load(q[u], c + U * NW);
      c += NW;
    }
  }

  // element i of a sum is column 4 * g + i of row r
  i32x4* sums = (i32x4*)lds;
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) sums[(wave * NF * MT + f * MT + t) * 64 + lane] = acc[f][t];
  __syncthreads();
  for (int i = tid; i < NF * MT * 64; i += 64 * NW) {
    const int f = i / (MT * 64), t = i / 64 % MT, m = tl.m0 + 16 * t + r, n = n0 + 16 * f + 4 * g;
    if (m >= tl.m1 || n >= a.N) continue;
    i32x4 v = sums[i];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += sums[w * NF * MT * 64 + i];
    const float s = row_scale[16 * t + r];
    uint8_t* y = a.Y + (size_t)m * a.ldy + (size_t)n * Y::ES;
    float o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int nn = min(n + k, a.N - 1);
      o[k] = scaled(v[k], s, sw[nn], a.bias ? a.bias[nn] : 0.f);
    }
    Y::put4(y, o, min(4, a.N - n));
  }
}

template <int YT, int XT, int MT, int NF, int NW, bool GROUPED>
int launch_rows(const I8Args& a, hipStream_t s, const char* who) {
  const int LDS = NW * NF * MT * 1024 + (XT >= 0 ? a.M * a.nk * kStep : 0);
  static std::atomic<uint64_t> done{0};
  auto* fn = i8_rows_kernel<YT, XT, MT, NF, NW, GROUPED>;
  const int st = lds_attr_once(done, (const void*)fn, 160 * 1024 - 1024, who);
  if (st != TIERMM_OK) return st;
  const long long ntn = (a.N + 16 * NF - 1) / (16 * NF);
  const long long ntm = GROUPED ? a.M / (16 * MT) + std::min(a.E, a.M) + 1 : 1;
  const long long grid = GROUPED ? (ntm * ntn + 7) / 8 * 8 : ntn;
  if (grid > (1ll << 22)) return set_error(TIERMM_UNSUPPORTED, "%s: %lld tiles", who, ntm * ntn);
  fn<<<(unsigned)grid, 64 * NW, LDS, s>>>(a);
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

// Up to kRows rows the few-row kernel, above it 256 x 320 tiles.
constexpr int kRows = 64, kFused = 4, kFusedLds = 64 * 1024;

int gemm(const I8Args& a, int ytype, bool grouped, hipStream_t s, const char* who) {
  int st = TIERMM_OK;
  with_rows(ytype, [&](auto yt) {
    constexpr int YT = decltype(yt)::value;
    if (grouped) {
      const int avg = a.M / a.E;
      if (avg <= 8) st = launch_rows<YT, -1, 1, 2, 4, true>(a, s, who);
      else if (avg <= 32) st = launch_rows<YT, -1, 2, 2, 4, true>(a, s, who);
      else st = launch_gemm<YT, 128, 128, 2, 2, true>(a, s, who);
    } else if (a.M <= kRows) {
      if (a.M <= 16) st = launch_rows<YT, -1, 1, 2, 8, false>(a, s, who);
      else if (a.M <= 32) st = launch_rows<YT, -1, 2, 2, 8, false>(a, s, who);
      else if (a.M <= 48) st = launch_rows<YT, -1, 3, 2, 8, false>(a, s, who);
      else st = launch_rows<YT, -1, 4, 2, 8, false>(a, s, who);
    } else {
      st = launch_gemm<YT, 256, 320, 4, 2, false>(a, s, who);
    }
  });
  return st;
}

// x of a few rows is quantized by the product's own workgroups.
bool fuses(int M, int K) { return M <= kFused && M * padded(K) <= kFusedLds; }
int fused(const I8Args& a, int xtype, int ytype, hipStream_t s, const char* who) {
  int st = TIERMM_OK;
  with_rows(ytype, [&](auto yt) {
    with_rows(xtype, [&](auto xt) {
      st = launch_rows<decltype(yt)::value, decltype(xt)::value, 1, 2, 8, false>(a, s, who);
    });
  });
  return st;
}

int quant(const void* x, int xtype, size_t ldx, int8_t* q, size_t rb, float* scale, int M, int K, hipStream_t s,
          const char* who) {
  const size_t es = row_elem_bytes(xtype);
  with_rows(xtype, [&](auto xt) {
    i8_quant_kernel<decltype(xt)::value>
        <<<M, 256, 0, s>>>((const uint8_t*)x, ldx * es, q, rb, scale, K, padded(K));
  });
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

bool misaligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

// Checks of the sizes, and of one side's rows.
int check_size(const char* who, int M, int N, int K) {
  if (M < 0 || N < 0 || K < 1) return set_error(TIERMM_EINVAL, "%s: bad size %d x %d x %d", who, M, N, K);
  if (K > kMaxK) return set_error(TIERMM_UNSUPPORTED, "%s: K = %d, at most %d", who, K, kMaxK);
  if (M > (1 << 23)) return set_error(TIERMM_UNSUPPORTED, "%s: %d rows, at most %d", who, M, 1 << 23);
  return TIERMM_OK;
}
int check_i8_rows(const char* who, const char* what, const void* p, size_t rb, int K) {
  if (!p) return set_error(TIERMM_EINVAL, "%s: null %s", who, what);
  if (rb < (size_t)padded(K) || rb % 16 || misaligned(p, 16))
    return set_error(TIERMM_EINVAL, "%s: %s rows of %zu bytes (whole 16-byte units from %d up, 16-byte aligned)", who,
                     what, rb, padded(K));
  return TIERMM_OK;
}
int check_out(const char* who, const void* Y, int ytype, size_t ldy, int N) {
  const int es = row_elem_bytes(ytype);
  if (!es) return set_error(TIERMM_UNSUPPORTED, "%s: output of type %d", who, ytype);
  if (ldy < (size_t)N) return set_error(TIERMM_EINVAL, "%s: row stride below %d", who, N);
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
  if (ldx < (size_t)K) return set_error(TIERMM_EINVAL, "%s: row stride below %d", who, K);
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
                    ldy * row_elem_bytes(ytype), M, N, K, padded(K) / kStep, nullptr, nullptr, 0, 1, M};
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
  if (ldx < (size_t)K) return set_error(TIERMM_EINVAL, "%s: row stride below %d", who, K);
  if (M == 0 || N == 0) return TIERMM_OK;
  if (!x || misaligned(x, es)) return set_error(TIERMM_EINVAL, "%s: null or misaligned x", who);
  if ((st = check_out(who, Y, ytype, ldy, N)) != TIERMM_OK) return st;
  if ((st = check_i8_rows(who, "weight", W, rbw, K)) != TIERMM_OK) return st;
  if (!sw || misaligned(sw, 4) || misaligned(bias, 4))
    return set_error(TIERMM_EINVAL, "%s: null or misaligned scales", who);
  I8Args a = {(const uint8_t*)x, nullptr, (const uint8_t*)W, sw, bias, (uint8_t*)Y, ldx * es, rbw,
              ldy * row_elem_bytes(ytype), M, N, K, padded(K) / kStep, nullptr, nullptr, 0, 1, M};
  if (fuses(M, K)) return fused(a, xtype, ytype, (hipStream_t)stream, who);
  void* w = nullptr;
  if (misaligned(ws, 16)) return set_error(TIERMM_EINVAL, "%s: workspace not 16-byte aligned", who);
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
                    ldy * row_elem_bytes(ytype), P, N, K, padded(K) / kStep, expert_offsets, rows, n_experts, topk, n_rows};
  return gemm(a, ytype, true, (hipStream_t)stream, who);
}

}  // extern "C"
