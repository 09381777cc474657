// mx.hip -- microscaled products: Y[m][n] = sum over blocks b of 32 of 2^(ex + ew - 254)
// sum_{k in b} cx[m][k] cw[n][k] (+ bias[n]), with W in E2M1, x in E2M1 or E4M3, and the quantizer
// that makes such rows.  No reference function (the reference expands its MXFP4 blocks to fp16).
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes the scales with the operands: lane l holds row l % 16, and
// of a step of 128 elements block l / 16 (E2M1: its 16 bytes; E4M3: 16 bytes of each half of the
// step) and that block's scale.
#include "tm_mx.h"
#include "tm_tiles.h"

#include <algorithm>
#include <cmath>

namespace tiermm {
int device_cus(int* cus);
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// ------------------------------------------------------------------- quantizer
// A thread takes R units of 16 bytes of a row; the lanes of a block are neighbours.  Bound by memory: 4096 rows of
// 5120 bfloat16 11.1 us to E2M1 (4.8 TB/s, 53 MB) and 12.7 to E4M3 with two units a thread, 12.9 and 14.3 with one.
template <int XT, int FMT, int R>
__global__ __launch_bounds__(1024) void mx_quant_kernel(const uint8_t* __restrict__ x, size_t ldx, uint8_t* __restrict__ q,
                                                        size_t rb, uint8_t* __restrict__ scales, size_t sb, int K, int Kp) {
  using X = Rows<XT>;
  const int m = blockIdx.x, step = blockDim.x * X::EPU, k = blockIdx.y * R * step + threadIdx.x * X::EPU;
  uint8_t* sc = scales + (size_t)m * sb;
  const int b = Kp / 32 + threadIdx.x;  // scales of blocks behind the padded row
  if (blockIdx.y == 0 && b < mx_scales(K)) sc[b] = 0;
  u32x4 u[R];
#pragma unroll
  for (int i = 0; i < R; ++i) u[i] = k + i * step < K ? X::get_nt(x + (size_t)m * ldx, k + i * step, K) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (k + i * step >= Kp) break;
    float v[X::EPU];
    X::widen(u[i], v);
    mx_store<FMT>(q + (size_t)m * rb, sc, k + i * step, v);
  }
}

// Few rows wait for their latency and take a unit a thread, many two.  bfloat16 to E2M1, us with one and two: 2048
// columns 512 rows 2.2 / 2.3, 2048 rows 3.1 / 3.1, 4096 rows 5.5 / 4.8; 5120 columns 256 rows 2.4 / 2.4, 512 3.0 /
// 3.0, 640 3.7 / 3.3; 14336 columns 128 rows 2.7 / 3.0, 256 3.4 / 3.4, 512 5.2 / 4.5.  (fp32 rows would change over
// at 200: 5120 columns 512 rows 4.2 / 3.3.)
int quant(const void* x, int xtype, size_t ldx, int fmt, void* q, size_t rb, uint8_t* scales, size_t sb, int M, int K,
          hipStream_t s, const char* who) {
  with_rows(xtype, [&](auto xt) {
    with_mx(fmt, [&](auto f) {
      constexpr int XT = decltype(xt)::value, FMT = decltype(f)::value, EPU = Rows<XT>::EPU;
      auto run = [&](auto rc) {
        constexpr int R = decltype(rc)::value;
        const int units = mx_padded(K) / EPU, threads = std::min(1024, (units + 64 * R - 1) / (64 * R) * 64);
        mx_quant_kernel<XT, FMT, R><<<dim3(M, (units + R * threads - 1) / (R * threads)), threads, 0, s>>>(
            (const uint8_t*)x, ldx * Rows<XT>::ES, (uint8_t*)q, rb, scales, sb, K, mx_padded(K));
      };
      if (M <= 512) run(std::integral_constant<int, 1>());
      else run(std::integral_constant<int, 2>());
    });
  });
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

// Rows of MXFP4 blocks (a scale and 16 bytes: element i in the low bits of byte i, element 16 + i in
// the high ones) as E2M1 rows and their scales.  A thread takes a block, or one of padding.
__global__ __launch_bounds__(256) void mx_from_mxfp4_kernel(const uint8_t* __restrict__ w, size_t rb,
                                                            uint8_t* __restrict__ q, size_t rbq,
                                                            uint8_t* __restrict__ scales, size_t sb, int blocks,
                                                            int padded_blocks, int scale_bytes) {
  const int n = blockIdx.x, b = blockIdx.y * 256 + threadIdx.x;
  if (b >= scale_bytes) return;
  u32x4 out = {0u, 0u, 0u, 0u};
  uint8_t scale = 0;
  if (b < blocks) {
    const uint8_t* p = w + (size_t)n * rb + (size_t)b * 17;
    scale = p[0];
    uint32_t lo[2] = {0u, 0u}, hi[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      lo[i >> 3] |= (uint32_t)(p[1 + i] & 15) << (4 * (i & 7));
      hi[i >> 3] |= (uint32_t)(p[1 + i] >> 4) << (4 * (i & 7));
    }
    out = u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
  if (b < padded_blocks) *(u32x4*)(q + (size_t)n * rbq + (size_t)b * 16) = out;
  scales[(size_t)n * sb + b] = scale;
}

// --------------------------------------------------------------------- product
struct MxArgs {
  const uint8_t *X, *sx;  // M rows of rbx bytes, their scales sbx a row
  const uint8_t *W, *sw;  // N rows of rbw bytes, their scales sbw a row
  const float* bias;      // or null
  uint8_t* Y;
  size_t rbx, sbx, rbw, sbw, ldy;  // bytes
  int M, N, K, nk;        // nk steps of 256 elements
};

// The MFMA of an E4M3 operand aligns the products of eight neighbouring k to the largest sum of
// exponents among them and keeps 13 bits below it (measured; E2M1's own products, of 2^-2 to 36, all fit).
// An element of E4M3 spans 2^-9 to 448, so small ones next to large ones would lose bits: up to 7 * 2^-13 of
// the largest product of each eight, 1e-5 of the result on normal rows and more than any output's rounding where large
// neighbours cancel.  x is therefore multiplied in two parts, magnitudes from 2 up and those
// below: with W's exponents of 0 to 2 the first has sums of exponents of 10 at most and lowest bits of 2^-3
// (2^-2 of x, half of it by W), the second 2 and 2^-10, so every product keeps its bits.
template <int XF>
constexpr int kParts = XF == MX_E4M3 ? 2 : 1;

// The codes of magnitude 2 and more, whose bit 6 is set, and zeros.
__device__ __forceinline__ uint32_t mx_large(uint32_t c) {
  const uint32_t one = (c & 0x40404040u) >> 6;
  return c & ((one << 8) - one);
}
__device__ __forceinline__ i32x8 mx_large(const i32x8& x) {
  i32x8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (int)mx_large((uint32_t)x[i]);
  return y;
}

// What a workgroup computes: rows [m0, m1) of Y, column tile tn.
struct Tile {
  int m0, m1, tn;
  bool once;  // no other tile reads these rows of W
};
// The tile of this workgroup; false past the last.  XCD x takes the x-th contiguous share of a walk in groups
// of 4 tile rows, column by column.
template <int BM, int BN>
__device__ __forceinline__ bool find_tile(const MxArgs& a, Tile& tl) {
  const int ntn = (a.N + BN - 1) / BN, ntm = (a.M + BM - 1) / BM, t = xcd_share(blockIdx.x, ntm * ntn);
  if (t < 0) return false;
  constexpr int GM = 4;
  const int grp = t / (GM * ntn), first = grp * GM, gm = min(GM, ntm - first), in = t - grp * GM * ntn;
  tl.m0 = (first + in % gm) * BM;
  tl.m1 = min(tl.m0 + BM, a.M);
  tl.tn = in / gm;
  tl.once = ntm == 1;
  return true;
}

// v_mfma_scale_f32_32x32x64_f8f6f4 / _16x16x128_ of W (E2M1) and x, with the scales in byte SEL of each word.
template <int XF, int SEL>
__device__ __forceinline__ f32x16 mx_mfma32(const i32x8& w, const i32x8& x, const f32x16& c, int sw, int sx) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, 4, XF == MX_E2M1 ? 4 : 0, SEL, sw, SEL, sx);
}
template <int XF>
__device__ __forceinline__ f32x4 mx_mfma16(const i32x8& w, const i32x8& x, const f32x4& c, int sw, int sx) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, XF == MX_E2M1 ? 4 : 0, 0, sw, 0, sx);
}
__device__ __forceinline__ i32x8 e2m1(const i32x4& v) { return i32x8{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }
__device__ __forceinline__ i32x8 e4m3(const i32x4& lo, const i32x4& hi) {
  return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// LDS of a workgroup: S stages of codes, then scales of two stages at a time.  With two stages in the ring a wave has
// x's scales of both in registers before the next two stages' are asked for; W's have two places.
template <int XF, int BM, int BN, int S>
struct GemmLds {
  static constexpr int STAGE = (BM * (XF == MX_E4M3 ? 2 : 1) + BN) * 128, XP = S == 2 ? 1 : 2;
  static constexpr int XSC = S * STAGE, WSC = XSC + XP * BM * 16, BIAS = WSC + 2 * BN * 16, AHEAD = BIAS + BN * 4, BYTES = AHEAD + 256;
  static __device__ __forceinline__ int xscales(int kt) { return XSC + (XP == 2 ? (kt >> 1 & 1) * BM * 16 : 0); }
  static __device__ __forceinline__ int wscales(int kt) { return WSC + (kt >> 1 & 1) * BN * 16; }
};
constexpr int kAhead = 1;  // stages behind the last one asked for

// BM rows of x times BN rows of W by WVM x WVN waves of WM x WN blocks of 32 x 32.
//
// A stage is 256 elements: 128 bytes of every row of W and of E2M1 x, two times 128 of E4M3 x (blocks 0-3
// of a row, then 4-7), and 8 scales of every row; S stages take turns, brought to LDS by global_load_lds.  The
// scales come 16 of a row at a time, with every other stage: each row is a cache line of its own for them, and
// as words of one stage they took as many lines as the codes (4096 x 5120 x 14336: 168 us).
// A row's 16-byte chunk c lies at slot c ^ ((row >> 1) & 7), which spreads the 16 rows that one cycle of a
// fragment read touches over the banks.  A stage is four MFMA steps of two blocks, one for each half of the wave; a
// lane's four scales of a row in a stage become one word, of which step kk uses byte kk.  While the products of one
// step run, the fragments of the next come in, one read between two MFMAs, and the loads of stage kt + S go
// out, from the step after the barrier that frees their place on.
//
// W is the MFMA's first operand, so a lane holds four neighbouring columns of one row of Y; rows leave
// through LDS in 16-byte units.
//
// 4096 x 14336 x 5120, bfloat16 Y: E2M1 170 us on random codes (256 x 320 tiles, 3.5 PFLOP/s) and 138 on zeros, E4M3
// 398 (128 x 320, 1.5) and 362; the MFMAs alone, at their rates on random codes, 98 and 300.  The cycles are the same
// on zeros (E2M1 330000 to 340000, E4M3 880000), so power takes what the clock falls by, from 2.4 to 1.9 and 2.1 GHz.
// Of the cycles MFMAs are busy in 44 and 66 %.  A stage takes 5500 and 7300, its MFMAs 2560 and 5120, and its 224 KB
// of fragment reads and 74 KB of loads into LDS 2400 at 128 bytes a cycle: the two hardly overlap, which is what is
// left to gain here.  With four waves of 128 x 128 (E2M1) 225 us against 208 with eight, before scales came in units
// and lines ahead.
template <int YT, int XF, int BM, int BN, int WVM, int WVN, int S>
__global__ __launch_bounds__(64 * WVM * WVN) void mx_gemm_kernel(const MxArgs a) {
  constexpr int NW = WVM * WVN, WM = BM / WVM / 32, WN = BN / WVN / 32, XS = XF == MX_E4M3 ? 2 : 1, NF = WN + WM * XS;
  constexpr int PARTS = kParts<XF>;
  constexpr int ROWS = BM * XS + BN, STAGE = ROWS * 128;
  constexpr int IC = STAGE / 1024 / NW, IS = (BM + BN + 64 * NW - 1) / (64 * NW), INST = IC + IS;
  static_assert(WM * WVM * 32 == BM && WN * WVN * 32 == BN && IC * NW * 1024 == STAGE, "whole blocks and loads a wave");
  static_assert(BM * XS % (8 * NW) == 0 && BM % 64 == 0 && BN % 64 == 0, "a load is of x or of W");
  using Lds = GemmLds<XF, BM, BN, S>;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  float* col_bias = (float*)(lds + Lds::BIAS);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Tile tl;
  if (!find_tile<BM, BN>(a, tl)) return;
  const int n0 = tl.tn * BN;
  using Y = Rows<YT>;

  // load u of this wave: rows 8 * (wave + NW * u) .. + 7 of the stage (x's, its second halves, then W's); from IC on
  // the scales of 64 rows for two stages.  Offsets from the tile's own first row: launch_gemm() sees that they
  // fit 32 bits.
  const uint8_t *X = a.X + (size_t)tl.m0 * a.rbx, *W = a.W + (size_t)n0 * a.rbw;
  const uint8_t *sx = a.sx + (size_t)tl.m0 * a.sbx, *sw = a.sw + (size_t)n0 * a.sbw;
  auto xr = [&](int r) { return (uint32_t)min(r, a.M - 1 - tl.m0); };
  auto wr = [&](int r) { return (uint32_t)min(r, a.N - 1 - n0); };
  const uint32_t rbx = (uint32_t)a.rbx, rbw = (uint32_t)a.rbw;
  uint32_t off[INST];
#pragma unroll
  for (int u = 0; u < IC; ++u) {
    const int r = 8 * (wave + NW * u) + (lane >> 3);
    off[u] = (u * NW * 8 < BM * XS ? xr(r % BM) * rbx + r / BM * 128 : wr(r - BM * XS) * rbw) + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
  }
  // (groups of 64 rows past the end: the last one again)
  auto group = [&](int u) { return min(wave + NW * u, (BM + BN) / 64 - 1); };
#pragma unroll
  for (int u = 0; u < IS; ++u) {
    const int r = 64 * group(u) + lane;
    off[IC + u] = 64 * group(u) < BM ? xr(r) * (uint32_t)a.sbx : wr(r - BM) * (uint32_t)a.sbw;
  }
  const uint32_t lds0 = lds_addr(lds);
  auto ring = [](int kt) { return S == 2 ? kt & 1 : kt % S; };
  auto issue = [&](int kt, int u) __attribute__((always_inline)) {
    if (u < IC) {
      const uint8_t* from = u * NW * 8 < BM * XS ? X + (size_t)kt * 128 * XS : W + (size_t)kt * 128;
      dma16(from, off[u], lds0 + ring(kt) * STAGE + (wave + NW * u) * 1024);
    } else if (!(kt & 1)) {
      const int g = group(u - IC);
      const uint8_t* from = (64 * g < BM ? sx : sw) + (size_t)kt * 8;
      dma16(from, off[u], lds0 + (64 * g < BM ? Lds::xscales(kt) : Lds::wscales(kt) - BM * 16) + g * 1024);
    }
  };
  // Lines of a later stage into the L2: this workgroup's share of those that its neighbours read too (an eighth of x's,
  // a fourth of W's), by a load of one word of each to where nothing is read.
  constexpr int AX = BM * XS / 8, AW = BN / 4, WX = (AX + 63) / 64;
  static_assert(WX + (AW + 63) / 64 <= NW, "a line a lane");
  const bool ahead_x = wave < WX;
  const int al = ahead_x ? min(tid, AX - 1) * 8 + tl.tn % 8 : min(tid - 64 * WX, AW - 1) * 4 + tl.m0 / BM % 4;
  const uint32_t ahead_off = ahead_x ? xr(al % BM) * rbx + al / BM * 128 : wr(al) * rbw;
  auto ahead = [&](int kt) __attribute__((always_inline)) {
    const size_t k = (size_t)min(kt, a.nk - 1) * 128;
    dma4(ahead_x ? X + k * XS : W + k, ahead_off, lds0 + Lds::AHEAD);
  };
#pragma unroll
  for (int t = 0; t < S - 1; ++t)
    if (t < a.nk) {
#pragma unroll
      for (int u = 0; u < INST; ++u) issue(t, u);
    }
#pragma unroll
  for (int t = 0; t <= kAhead; ++t) ahead(S - 1 + t);
  for (int i = tid; i < BN; i += 64 * NW) col_bias[i] = a.bias ? a.bias[min(n0 + i, a.N - 1)] : 0.f;

  f32x16 acc[WN][WM];
#pragma unroll
  for (int j = 0; j < WN; ++j)
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0.f;

  const int wm = wave % WVM, wn = wave / WVM, fr = lane & 31, fh = lane >> 5, turn = (fr >> 1) & 7;
  const uint32_t xrow = (uint32_t)(wm * WM * 32 + fr) * 128, wrow = (uint32_t)(BM * XS + wn * WN * 32 + fr) * 128;
  i32x4 xf[2][WM][XS], wf[2][WN];
  int xs[WM], ws[WN], xs1[WM] = {};  // scales of this stage, and of x in an odd one behind it
  // fragment v of step kk of stage kt into set f: W's first, those of x, W's others
  auto fragment = [&](int kt, int kk, int f, int v) __attribute__((always_inline)) {
    const uint8_t* s = lds + ring(kt) * STAGE;
    const int wc = ((2 * kk + fh) ^ turn) * 16;
    if (v >= 1 && v <= WM * XS) {
      const int i = (v - 1) / XS, h = (v - 1) % XS;
      // (E4M3: half a block of the step's first one, and of its second)
      const int xc = XS == 1 ? wc : ((4 * (kk & 1) + 2 * h + fh) ^ turn) * 16;
      xf[f][i][h] = *(const i32x4*)(s + xc + xrow + ((XS == 1 ? 0 : (kk >> 1) * BM) + i * 32) * 128);
    } else {
      const int j = v == 0 ? 0 : v - WM * XS;
      wf[f][j] = *(const i32x4*)(s + wc + wrow + j * 32 * 128);
    }
  };
  // (every other byte of two words: the blocks of this half of the wave)
  const uint32_t mine = fh ? 0x07050301u : 0x06040200u;
  auto scales = [&](int kt, int (&x)[WM], int (&w)[WN]) __attribute__((always_inline)) {
    const uint8_t* px = lds + Lds::xscales(kt) + (wm * WM * 32 + fr) * 16;
    const uint8_t* pw = lds + Lds::wscales(kt) + (wn * WN * 32 + fr) * 16 + 8 * (kt & 1);
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      int even = xs1[i], odd = 0;
      if (!(kt & 1)) {
        const u32x4 v = *(const u32x4*)(px + i * 512);
        even = (int)__builtin_amdgcn_perm(v[1], v[0], mine);
        odd = (int)__builtin_amdgcn_perm(v[3], v[2], mine);
      }
      x[i] = even;
      xs1[i] = odd;
    }
#pragma unroll
    for (int j = 0; j < WN; ++j) {
      const u32x2 v = *(const u32x2*)(pw + j * 512);
      w[j] = (int)__builtin_amdgcn_perm(v[1], v[0], mine);
    }
  };
  // The products of step KK of fragments f, with the fragments (kt, kk) into the other set and n loads of stage
  // `dt` between them.
  auto step = [&](auto kc, int f, int kt, int kk, int dt, int n) __attribute__((always_inline)) {
    constexpr int KK = decltype(kc)::value, nm = WM * WN;
    i32x8 x[WM][PARTS];
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      if constexpr (XS == 1) x[i][0] = e2m1(xf[f][i][0]);
      else x[i][0] = e4m3(xf[f][i][0], xf[f][i][1]);
      if constexpr (PARTS == 2) {
        x[i][1] = mx_large(x[i][0]);
        x[i][0] ^= x[i][1];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < nm; ++q) {
#pragma unroll
      for (int v = 0; v < NF; ++v)
        if (std::max(v * (nm - 2) / NF, 0) == q) fragment(kt, kk, f ^ 1, v);
#pragma unroll
      for (int d = 0; d < n; ++d)
        if (std::min(1 + d * (nm - 1) / n, nm - 1) == q && dt < a.nk) issue(dt, d);
      const int j = q / WM, i = q % WM;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) acc[j][i] = mx_mfma32<XF, KK>(e2m1(wf[f][j]), x[i][p], acc[j][i], ws[j], xs[i]);
      // the compiler would sink these products past the loads' branches, all to the end of the loop (no
      // instruction: nothing reads the sum here)
      asm volatile("" : "+v"(acc[j][i]));
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // waits until stage kt has landed, those up to kt + S - 2 being on their way too
  auto landed = [&](int kt) __attribute__((always_inline)) {
    static_assert(S <= 3, "stages that one wait may leave on their way");
    // (each stage's loads are followed by one of a line ahead)
    if (S == 2) vm_wait<1>();
    else if (kt + 1 >= a.nk) vm_wait<2>();
    else if (kt & 1) vm_wait<INST + 2>();  // an even stage brings scales
    else vm_wait<IC + 2>();
  };
  vm_wait<0>();
  __syncthreads();
  if (S - 1 < a.nk) {
#pragma unroll
    for (int u = 0; u < INST; ++u) issue(S - 1, u);
  }
  scales(0, xs, ws);
  __builtin_amdgcn_sched_barrier(0);  // the first fragments in the loop's own order, one wait for each
#pragma unroll
  for (int v = 0; v < NF; ++v) {
    fragment(0, 0, 0, v);
    __builtin_amdgcn_sched_barrier(0);
  }
  for (int kt = 0; kt < a.nk; ++kt) {
    step(std::integral_constant<int, 0>(), 0, kt, 1, 0, 0);
    step(std::integral_constant<int, 1>(), 1, kt, 2, 0, 0);
    ahead(kt + S + kAhead);
    step(std::integral_constant<int, 2>(), 0, kt, 3, 0, 0);
    landed(kt + 1);
    __syncthreads();  // stage kt + 1 has landed for every wave, and stage kt is read
    // (past the end: the fragments of what the place holds, which nothing uses)
    int nx[WM], nw[WN];
    scales(kt + 1, nx, nw);
    step(std::integral_constant<int, 3>(), 1, kt + 1, 0, kt + S, INST);
#pragma unroll
    for (int i = 0; i < WM; ++i) xs[i] = nx[i];
#pragma unroll
    for (int j = 0; j < WN; ++j) ws[j] = nw[j];
  }

  // Element r of a block is column 8 * (r / 4) + 4 * fh + r % 4 of row fr.  Each wave passes 32 rows of one or
  // two blocks at a time through its part of LDS and stores whole 16-byte units, 8 of them a row.
  constexpr int JB = Y::ES == 2 ? 2 : 1, PART = 4096;
  static_assert(NW * PART <= S * STAGE, "rows of the epilogue in LDS");
  uint8_t* part = lds + wave * PART;
  auto store = [&](auto jn, int j0) __attribute__((always_inline)) {
    constexpr int J = decltype(jn)::value, CH = J * 32 * Y::ES / 16;
    const int cw = (wn * WN + j0) * 32, nw = n0 + cw;
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      const int mb = tl.m0 + (wm * WM + i) * 32;
      if (mb >= tl.m1) break;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int c = j * 32 + 8 * b + 4 * fh;
          f32x4 v = *(const f32x4*)(col_bias + cw + c);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] += acc[j0 + j][i][4 * b + k];
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

template <class Fn>
int launch(Fn* fn, std::atomic<uint64_t>& done, const MxArgs& a, int bm, int bn, int threads, int lds, hipStream_t s,
           const char* who) {
  const int st = lds_attr_once(done, (const void*)fn, lds, who);
  if (st != TIERMM_OK) return st;
  const long long tiles = ((a.N + bn - 1ll) / bn) * ((a.M + bm - 1ll) / bm), grid = (tiles + 7) / 8 * 8;
  if (grid * threads >= (1ll << 32)) return set_error(TIERMM_UNSUPPORTED, "%s: %lld tiles", who, tiles);
  fn<<<(unsigned)grid, threads, lds, s>>>(a);
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

template <int YT, int XF, int BM, int BN, int WVM, int WVN, int S>
int launch_gemm(const MxArgs& a, hipStream_t s, const char* who) {
  constexpr int LDS = GemmLds<XF, BM, BN, S>::BYTES;
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static std::atomic<uint64_t> done{0};
  return launch(mx_gemm_kernel<YT, XF, BM, BN, WVM, WVN, S>, done, a, BM, BN, 64 * WVM * WVN, LDS, s, who);
}

// Few rows: the product is bound by the bytes of W.  A workgroup takes a BM x BN tile; its WVN x WVK waves
// share the columns and the steps of 128 elements of a stage, which holds KS * 256 elements of every row and
// their scales.  A ring of S stages keeps S - 1 on their way by global_load_lds; one barrier a stage.
//
// Of a 128-byte piece of a row lane group g takes blocks g and 4 + g, one a step (E4M3: what the MFMA wants, half a
// block of each half of the step).
//
// 14336 x 5120: E2M1 and bfloat16 Y 9.7 us for 8 rows (4.0 TB/s), 13.2 for 37, E4M3 and fp32 Y 10.5 and 16.1; 37 rows
// in two tiles of 32 of each column took 14.3 and 19.4, one of 48 by four waves 13.0 and 19.4.  With both operands
// straight from memory into registers 8 rows of E4M3 took 13.9 us, 37 21.7.
template <int YT, int XF, int BM, int BN, int WVN, int WVK, int KS, int S>
__global__ __launch_bounds__(64 * WVN * WVK) void mx_tile_kernel(const MxArgs a) {
  constexpr int NW = WVN * WVK, MB = BM / 16, NB = BN / WVN / 16, KK = 2 * KS / WVK, XS = XF == MX_E4M3 ? 2 : 1;
  constexpr int PARTS = kParts<XF>;
  constexpr int ROWS = BM * XS + BN, SUB = ROWS * 128, CODES = KS * SUB, IC = CODES / 1024 / NW;
  constexpr int CH = KS / 2, UNITS = CH * (BM + BN), IS = (UNITS + 64 * NW - 1) / (64 * NW), INST = IC + IS;
  constexpr int STAGE = CODES + UNITS * 16;
  static_assert(UNITS >= 64, "a load of scales fills its place");
  static_assert(IC * NW * 1024 == CODES && KK * WVK == 2 * KS && NB * WVN * 16 == BN && KS % 2 == 0, "whole loads, steps and blocks a wave");
  constexpr int LDO = BN + 4;  // words of a row of sums
  static_assert(WVK * BM * LDO * 4 <= S * STAGE, "sums in LDS");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Tile tl;
  if (!find_tile<BM, BN>(a, tl)) return;
  const int n0 = tl.tn * BN;
  using Y = Rows<YT>;

  // load u of this wave: eight rows of a sub-stage (x's, its second halves, then W's); from IC on 16 scales of
  // 64 rows (units past the end: the last 64 again)
  const uint8_t* src[INST];
#pragma unroll
  for (int u = 0; u < IC; ++u) {
    const int r = (8 * (wave + NW * u) + (lane >> 3)) % ROWS;
    const uint8_t* row = r < BM * XS ? a.X + (size_t)min(tl.m0 + r % BM, a.M - 1) * a.rbx + r / BM * 128
                                     : a.W + (size_t)min(n0 + r - BM * XS, a.N - 1) * a.rbw;
    src[u] = row + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
  }
  int unit[IS], place[IS];  // which 16 of a row's scales in the stage, and the load's first unit
#pragma unroll
  for (int u = 0; u < IS; ++u) {
    place[u] = min(64 * (wave + NW * u), UNITS - 64);
    const int i = place[u] + lane, r = i % (BM + BN);
    unit[u] = i / (BM + BN);
    src[IC + u] = r < BM ? a.sx + (size_t)min(tl.m0 + r, a.M - 1) * a.sbx : a.sw + (size_t)min(n0 + r - BM, a.N - 1) * a.sbw;
  }
  const uint32_t lds0 = lds_addr(lds);
  const int ns = (a.nk + KS - 1) / KS, last_unit = (a.nk - 1) / 2;
  int put = 0;
  auto issue = [&](int st) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < IC; ++u) {
      const int i = 8 * (wave + NW * u), r = i % ROWS;
      // sub-stages past the end load the last one again, and are not multiplied
      const size_t k = (size_t)min(st * KS + i / ROWS, a.nk - 1);
      const uint32_t to = lds0 + put * STAGE + (wave + NW * u) * 1024;
      if (r < BM * XS) dma16(src[u] + k * 128 * XS, to);
      else if (tl.once) dma16_nt(src[u] + k * 128, to);
      else dma16(src[u] + k * 128, to);
    }
#pragma unroll
    for (int u = 0; u < IS; ++u)
      dma16(src[IC + u] + (size_t)min(st * CH + unit[u], last_unit) * 16, lds0 + put * STAGE + CODES + 16 * place[u]);
    put = put + 1 == S ? 0 : put + 1;
  };
  static_assert(BM * XS % 8 == 0 && BN % 8 == 0, "a load is of x or of W");
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < ns) issue(i);

  f32x4 acc[NB][MB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
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
      const int step = wk * KK + k, sub = step >> 1, h = step & 1;
      if (st * KS + sub >= a.nk) break;
      const int wc = ((4 * h + fg) ^ turn) * 16;
      const uint8_t* p = s + sub * SUB + fr * 128;
      const uint8_t* sc = s + CODES + ((sub >> 1) * (BM + BN) + fr) * 16 + (sub & 1) * 8 + 4 * h + fg;
      i32x8 xf[MB][PARTS], wf[NB];
      int xs[MB], ws[NB];
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const uint8_t* x = p + ((XS == 1 ? 0 : h * BM) + i * 16) * 128;
        if constexpr (XS == 1) xf[i][0] = e2m1(*(const i32x4*)(x + wc));
        else xf[i][0] = e4m3(*(const i32x4*)(x + (fg ^ turn) * 16), *(const i32x4*)(x + ((4 + fg) ^ turn) * 16));
        xs[i] = sc[i * 256];
        if constexpr (PARTS == 2) {
          xf[i][1] = mx_large(xf[i][0]);
          xf[i][0] ^= xf[i][1];
        }
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        wf[j] = e2m1(*(const i32x4*)(p + wc + (BM * XS + (wn * NB + j) * 16) * 128));
        ws[j] = sc[(BM + (wn * NB + j) * 16) * 16];
      }
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int q = 0; q < PARTS; ++q) acc[j][i] = mx_mfma16<XF>(wf[j], xf[i][q], acc[j][i], ws[j], xs[i]);
    }
  }
  __syncthreads();
  // a lane's sum is columns 4 * fg .. + 3 of row fr of each block
  float* sums = (float*)lds;
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i)
      *(f32x4*)(sums + (wk * BM + i * 16 + fr) * LDO + (wn * NB + j) * 16 + 4 * fg) = acc[j][i];
  __syncthreads();
  for (int q = tid; q < BM * BN / 4; q += 64 * NW) {
    const int r = q / (BN / 4), c = q % (BN / 4) * 4, m = tl.m0 + r, n = n0 + c;
    if (m >= tl.m1 || n >= a.N) continue;
    f32x4 v = *(const f32x4*)(sums + r * LDO + c);
#pragma unroll
    for (int w = 1; w < WVK; ++w) {
      const f32x4 t = *(const f32x4*)(sums + (w * BM + r) * LDO + c);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += t[k];
    }
    float o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = v[k] + (a.bias ? a.bias[min(n + k, a.N - 1)] : 0.f);
    Y::put4(a.Y + (size_t)m * a.ldy + (size_t)n * Y::ES, o, min(4, a.N - n));
  }
}

template <int YT, int XF, int BM, int BN, int WVN, int WVK, int KS, int S>
int launch_tile(const MxArgs& a, hipStream_t s, const char* who) {
  constexpr int XS = XF == MX_E4M3 ? 2 : 1;
  constexpr int LDS = S * (KS * (BM * XS + BN) * 128 + KS / 2 * (BM + BN) * 16);
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static std::atomic<uint64_t> done{0};
  return launch(mx_tile_kernel<YT, XF, BM, BN, WVN, WVK, KS, S>, done, a, BM, BN, 64 * WVN * WVK, LDS, s, who);
}

// ----------------------------------------------------------------- single tokens
template <int CTRL>
__device__ __forceinline__ float add_ror(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// Up to MX rows of x, quantized by each workgroup into LDS while its first weights are on the way.  A wave
// takes R rows of W in 1 KiB pieces, 16 bytes (a block) a lane, so each load is eight whole lines of one row.
//
// The piece is the MFMA's first operand as it comes: lane l = 16 g + i holds "row" i's block of group g, which
// stands for block 16 g + i of the one row of W.  With x's blocks laid out alike as the second, the diagonal of the
// 16 x 16 result holds sum_g <W block 16 g + i, x block 16 g + i>, and its trace over all pieces is the product.  The
// other 240 sums are waste, but the matrix cores have a tenth of the bytes' time to spend, and nothing is unpacked.
// 1 x 14336 x 5120, E2M1 and bfloat16: 8.0 us, 4.9 TB/s (a large copy reaches 4.8), E4M3 11.7, for its MFMAs take
// four times as long; 1 x 1024 x 5120, E4M3 and fp32: 3.5 us, of which the launch and one latency are most.
template <int YT, int XT, int XF, int MX, int R, int NW>
__global__ __launch_bounds__(64 * NW) void mx_gemv_kernel(const MxArgs a) {
  // [MX][pieces][XB KiB] codes in the order that lanes read them, then [MX][pieces][64] scales
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  constexpr int XB = XF == MX_E4M3 ? 2048 : 1024, PARTS = kParts<XF>;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = a.nk * 8, nc = (blocks + 63) >> 6;
  uint8_t* xsc = lds + MX * nc * XB;
  const int n0 = (blockIdx.x * NW + wave) * R;
  const uint8_t *wp[R], *sp[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    wp[r] = a.W + (size_t)min(n0 + r, a.N - 1) * a.rbw + 16 * lane;
    sp[r] = a.sw + (size_t)min(n0 + r, a.N - 1) * a.sbw + lane;
  }
  constexpr int U = 3;  // pieces in flight
  i32x4 q[U][R];
  int qs[U][R];
  auto load = [&](int u, int c) __attribute__((always_inline)) {
    const bool in = c * 64 + lane < blocks;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      q[u][r] = in ? __builtin_nontemporal_load((const i32x4*)(wp[r] + ((size_t)c << 10))) : i32x4{0, 0, 0, 0};
      qs[u][r] = in ? sp[r][(size_t)c << 6] : 0;
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < nc) load(u, u);

  using X = Rows<XT>;
  constexpr int EPU = X::EPU, STEP = 64 * NW * EPU;
  // (whole pieces: blocks past the row become zeros)
  for (int k = tid * EPU; k < nc * 2048; k += STEP) {
    u32x4 xu[MX];
#pragma unroll
    for (int m = 0; m < MX; ++m)
      xu[m] = k < a.K ? X::get(a.X + (size_t)min(m, a.M - 1) * a.rbx, k, a.K) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int m = 0; m < MX; ++m) {
      float v[EPU];
      X::widen(xu[m], v);
      uint32_t top = 0, w[2];
#pragma unroll
      for (int i = 0; i < EPU; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      const int byte = mx_scale_of<XF>(mx_block_top<32 / EPU>(top));
      mx_codes<XF>(v, mx_inverse(byte), w);
      const int piece = k >> 11, b = (k >> 5) & 63, in = k & 31;
      uint8_t* to = lds + (m * nc + piece) * XB;
      if constexpr (XF == MX_E2M1) mx_put<XF, EPU>(to + b * 16, in, w);
      else mx_put<XF, EPU>(to + (b >> 5) * 1024 + (2 * ((b >> 4) & 1) + (in >> 4)) * 256 + (b & 15) * 16, in & 15, w);
      if (in == 0) xsc[(m * nc + piece) * 64 + b] = (uint8_t)byte;
    }
  }
  __syncthreads();

  f32x4 acc[MX][R];
#pragma unroll
  for (int m = 0; m < MX; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[m][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c0 = 0; c0 < nc; c0 += U)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u;
      if (c >= nc) break;
#pragma unroll
      for (int m = 0; m < MX; ++m) {
        const uint8_t* xp = lds + (m * nc + c) * XB + 16 * lane;
        const int xs = xsc[(m * nc + c) * 64 + lane];
        i32x8 x[PARTS];
        if constexpr (XF == MX_E2M1) x[0] = e2m1(*(const i32x4*)xp);
        else x[0] = e4m3(*(const i32x4*)xp, *(const i32x4*)(xp + 1024));
        if constexpr (PARTS == 2) {
          x[1] = mx_large(x[0]);
          x[0] ^= x[1];
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int p = 0; p < PARTS; ++p) acc[m][r] = mx_mfma16<XF>(e2m1(q[u][r]), x[p], acc[m][r], qs[u][r], xs);
      }
      if (c + U < nc) load(u, c + U);
    }
  using Y = Rows<YT>;
  const int col = lane & 15, g = lane >> 4;
#pragma unroll
  for (int m = 0; m < MX; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      // the diagonal: row 4 g + i, column `col`
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) v = col == 4 * g + i ? acc[m][r][i] : v;
      v = add_ror<0x121>(add_ror<0x122>(add_ror<0x124>(add_ror<0x128>(v))));  // row_ror 8, 4, 2, 1
      v = row_sum4(v);
      const int n = n0 + r;
      if (lane == 0 && m < a.M && n < a.N) {
        const float o[4] = {v + (a.bias ? a.bias[n] : 0.f), 0.f, 0.f, 0.f};
        Y::put4(a.Y + (size_t)m * a.ldy + (size_t)n * Y::ES, o, 1);
      }
    }
}

template <int YT, int XT, int XF, int MX, int R, int NW>
int launch_gemv(const MxArgs& a, hipStream_t s, const char* who) {
  const int nc = (a.nk * 8 + 63) / 64;
  mx_gemv_kernel<YT, XT, XF, MX, R, NW><<<(a.N + NW * R - 1) / (NW * R), 64 * NW, MX * nc * (XF == MX_E4M3 ? 2112 : 1088), s>>>(a);
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

// One or two rows of x are quantized by the product's own workgroups: a launch less, and each byte of W in whole
// lines.  Two tokens of 4096 x 4096, us, against the quantizer (2.2) and the tiles: E2M1 4.2 and 6.5, E4M3 5.5 and
// 7.2; of 14336 x 5120 E2M1 11.4 and 11.4, E4M3 15.8 and 12.0, whose MFMAs for two rows take longer than W's bytes.
// (That one stays here all the same: a call of one or two rows needs no workspace.)
constexpr int kGemvLds = 60 * 1024;
bool fuses(int xfmt, int M, int K) {
  return M <= 2 && M * (long long)((mx_padded(K) + 2047) / 2048) * (xfmt == MX_E4M3 ? 2112 : 1088) <= kGemvLds;
}

int fused(const MxArgs& a, int xtype, int xfmt, int ytype, hipStream_t s, const char* who) {
  int st = TIERMM_OK;
  with_rows(ytype, [&](auto yt) {
    with_rows(xtype, [&](auto xt) {
      with_mx(xfmt, [&](auto f) {
        constexpr int YT = decltype(yt)::value, XT = decltype(xt)::value, XF = decltype(f)::value;
        auto rows = [&](auto mx) {
          constexpr int MX = decltype(mx)::value;
          // Short products take workgroups of 8 rows, so that every CU has some; long ones of 32, which prepare x
          // fewer times.  us with 8 and 32 rows, 1 token of K = 5120: E2M1 1024 columns 3.3 / 4.7, 4096 4.2 / 5.1,
          // 5120 5.0 / 5.2, 8192 5.9 / 5.9, 14336 9.2 / 8.2; E4M3 4096 5.2 / 6.1, 5120 6.4 / 6.3, 8192 7.7 / 7.0.  K
          // = 14336 crosses between 4096 and 5120 columns too, K = 2048 at 5120 (E4M3) or past 8192 (E2M1: 3.5 / 3.8
          // there, 14336 5.5 / 4.5).
          if (a.N < 5120) st = launch_gemv<YT, XT, XF, MX, 1, 8>(a, s, who);
          else st = launch_gemv<YT, XT, XF, MX, 2, 16>(a, s, who);
        };
        if (a.M == 1) rows(std::integral_constant<int, 1>());
        else rows(std::integral_constant<int, 2>());
      });
    });
  });
  return st;
}

// The tiles, and what one costs: a call takes about t0 + n * (fix + K / 1024 * each) us, n the tiles that the fullest
// CU runs.  Fitted to measured times of 192 sizes (4 to 4096 rows, 512 to 28672 columns, K of 1024 to 14336), on
// weights that the last-level cache holds where they fit; the tile with the least such time is within 0.9 % of the
// best of its list in the mean up to 256 rows and within 0.4 % over all, 26 % at worst.  E4M3 x, in its two parts,
// has a list of its own (fitted on fp32 Y).  Example, 5120 columns and rows of 5120, E2M1, us: 16 rows 16 x 32 tiles
// 6.3, 64 x 128 12.4, 128 x 128 16.0; 256 rows 64 x 128 14.1, 128 x 128 18.7, 32 x 64 20.4; 4096 rows 256 x 320 59.6,
// 256 x 192 70.3, 128 x 128 95.8.
struct TileCost {
  int bm, bn;
  float t0, fix, each;
};
constexpr TileCost kE2m1Tiles[] = {
    {16, 16, 2.64f, 0.60f, 0.26f}, {16, 32, 1.65f, 1.70f, 0.43f}, {16, 64, 1.36f, 2.10f, 0.65f}, {32, 32, 1.59f, 1.65f, 0.54f},
    {32, 64, 1.18f, 2.49f, 0.79f}, {48, 64, 1.09f, 2.61f, 1.08f}, {64, 128, 2.09f, 0.81f, 2.04f}, {128, 128, 0.f, 3.22f, 2.91f},
    {256, 128, 0.f, 4.51f, 3.96f}, {256, 192, 0.f, 4.90f, 4.87f}, {256, 256, 0.f, 5.89f, 5.41f}, {256, 320, 0.f, 6.88f, 6.62f},
};
constexpr TileCost kE4m3Tiles[] = {
    {16, 16, 1.51f, 1.67f, 0.52f}, {16, 32, 1.63f, 1.53f, 0.66f}, {16, 64, 1.36f, 2.30f, 0.91f}, {32, 32, 1.22f, 2.32f, 0.97f},
    {32, 64, 1.10f, 2.53f, 1.34f}, {48, 64, 1.15f, 2.65f, 2.11f}, {64, 128, 0.19f, 3.28f, 4.70f}, {128, 128, 0.f, 4.54f, 8.01f},
    {128, 192, 0.f, 5.50f, 7.41f}, {128, 256, 0.f, 6.44f, 9.32f}, {128, 320, 0.f, 7.33f, 10.8f},
};
constexpr int kTileKernels = 6;  // the first ones, of mx_tile_kernel

template <int N>
int pick_of(const TileCost (&tiles)[N], const MxArgs& a, int cus) {
  int best = 0;
  float least = 1e30f;
  for (int i = 0; i < N; ++i) {
    const TileCost& c = tiles[i];
    // mx_gemm_kernel's offsets from a tile's first row have 32 bits
    if (i >= kTileKernels && std::max(a.rbx * c.bm, a.rbw * c.bn) + std::max(a.sbx * c.bm, a.sbw * c.bn) >= (1ull << 32)) continue;
    const float n = std::ceil(std::ceil((float)a.M / c.bm) * ((a.N + c.bn - 1) / c.bn) / cus);
    const float t = c.t0 + n * (c.fix + a.nk * (kMxStep / 1024.f) * c.each);
    if (t < least) least = t, best = i;
  }
  return best;
}

template <int YT, int XF>
int launch_picked(const MxArgs& a, int cus, hipStream_t s, const char* who) {
  constexpr bool E4 = XF == MX_E4M3;
  switch (E4 ? pick_of(kE4m3Tiles, a, cus) : pick_of(kE2m1Tiles, a, cus)) {
    case 0: return launch_tile<YT, XF, 16, 16, 1, 8, 4, 4>(a, s, who);
    case 1: return launch_tile<YT, XF, 16, 32, 1, 8, 4, 4>(a, s, who);
    case 2: return launch_tile<YT, XF, 16, 64, 1, 8, 4, 3>(a, s, who);
    case 3: return launch_tile<YT, XF, 32, 32, 1, 8, 4, 3>(a, s, who);
    case 4: return launch_tile<YT, XF, 32, 64, 1, 8, 4, E4 ? 2 : 3>(a, s, who);
    case 5: return launch_tile<YT, XF, 48, 64, 2, 4, E4 ? 2 : 4, E4 ? 3 : 2>(a, s, who);
    case 6: return launch_gemm<YT, XF, 64, 128, 2, 4, 3>(a, s, who);
    case 7: return launch_gemm<YT, XF, 128, 128, 2, 4, 3>(a, s, who);
    case 8: return launch_gemm<YT, XF, E4 ? 128 : 256, E4 ? 192 : 128, 4, 2, E4 ? 2 : 3>(a, s, who);
    case 9: return launch_gemm<YT, XF, E4 ? 128 : 256, E4 ? 256 : 192, 4, 2, 2>(a, s, who);
    case 10: return launch_gemm<YT, XF, E4 ? 128 : 256, E4 ? 320 : 256, 4, 2, 2>(a, s, who);
    default: return launch_gemm<YT, XF, E4 ? 128 : 256, 320, 4, 2, 2>(a, s, who);  // (E2M1)
  }
}

int gemm(const MxArgs& a, int xfmt, int ytype, hipStream_t s, const char* who) {
  int cus = 0, st = device_cus(&cus);
  if (st != TIERMM_OK) return st;
  with_rows(ytype, [&](auto yt) {
    with_mx(xfmt, [&](auto f) { st = launch_picked<decltype(yt)::value, decltype(f)::value>(a, cus, s, who); });
  });
  return st;
}

bool misaligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

int check_size(const char* who, int M, int N, int K) {
  if (M < 0 || N < 0 || K < 1) return set_error(TIERMM_EINVAL, "%s: bad size %d x %d x %d", who, M, N, K);
  if (K > kMxMaxK) return set_error(TIERMM_UNSUPPORTED, "%s: K = %d, at most %d", who, K, kMxMaxK);
  if (M > (1 << 20)) return set_error(TIERMM_UNSUPPORTED, "%s: %d rows, at most %d", who, M, 1 << 20);
  // (a launch has less than 2^32 threads, of which a row of W may have 256)
  if (N >= (1 << 24)) return set_error(TIERMM_UNSUPPORTED, "%s: %d columns, at most %d", who, N, (1 << 24) - 1);
  return TIERMM_OK;
}
int check_fmt(const char* who, int fmt) {
  if (fmt == MX_E2M1 || fmt == MX_E4M3) return TIERMM_OK;
  return set_error(TIERMM_UNSUPPORTED, "%s: format %d", who, fmt);
}
int check_out(const char* who, const void* Y, int ytype, size_t ldy, const float* bias, int N) {
  const int es = row_elem_bytes(ytype);
  if (!es) return set_error(TIERMM_UNSUPPORTED, "%s: output of type %d", who, ytype);
  if (bad_stride(ldy, N)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, N);
  if (!Y || misaligned(Y, es)) return set_error(TIERMM_EINVAL, "%s: null or misaligned output", who);
  if (misaligned(bias, 4)) return set_error(TIERMM_EINVAL, "%s: misaligned bias", who);
  return TIERMM_OK;
}

}  // namespace
}  // namespace tiermm

using namespace tiermm;

extern "C" {

size_t tiermm_mx_row_bytes(int fmt, int K) { return mx_row_bytes(fmt, K); }
size_t tiermm_mx_scale_bytes(int K) { return K < 1 || K > kMxMaxK ? 0 : (size_t)mx_scales(K); }

int tiermm_mx_quant(const void* x, int xtype, size_t ldx, int fmt, void* q, size_t rb, uint8_t* scales, size_t sb,
                    int M, int K, tiermm_stream_t stream) {
  const char* who = "tiermm_mx_quant";
  int st = check_size(who, M, 0, K);
  if (st != TIERMM_OK || (st = check_fmt(who, fmt)) != TIERMM_OK) return st;
  const int es = row_elem_bytes(xtype);
  if (!es) return set_error(TIERMM_UNSUPPORTED, "%s: rows of type %d", who, xtype);
  if (bad_stride(ldx, K)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, K);
  if (M == 0) return TIERMM_OK;
  if (!x || misaligned(x, es)) return set_error(TIERMM_EINVAL, "%s: null or misaligned x", who);
  if ((st = check_mx_rows(who, "output", fmt, q, rb, scales, sb, K)) != TIERMM_OK) return st;
  return quant(x, xtype, ldx, fmt, q, rb, scales, sb, M, K, (hipStream_t)stream, who);
}

int tiermm_mx_from_mxfp4(const void* W, size_t rb, void* q, size_t rbq, uint8_t* scales, size_t sb, int N, int K,
                         tiermm_stream_t stream) {
  const char* who = "tiermm_mx_from_mxfp4";
  int st = check_size(who, 0, N, K);
  if (st != TIERMM_OK) return st;
  if (K % 32) return set_error(TIERMM_UNSUPPORTED, "%s: %d columns are not whole blocks", who, K);
  if (bad_stride(rb, (size_t)K / 32 * 17)) return set_error(TIERMM_EINVAL, "%s: rows of %zu bytes", who, rb);
  if (N == 0) return TIERMM_OK;
  if (!W) return set_error(TIERMM_EINVAL, "%s: null W", who);
  if ((st = check_mx_rows(who, "output", MX_E2M1, q, rbq, scales, sb, K)) != TIERMM_OK) return st;
  const dim3 grid(N, (mx_scales(K) + 255) / 256);
  mx_from_mxfp4_kernel<<<grid, 256, 0, (hipStream_t)stream>>>((const uint8_t*)W, rb, (uint8_t*)q, rbq, scales, sb, K / 32,
                                                              mx_padded(K) / 32, mx_scales(K));
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

int tiermm_mx_gemm(const void* Xq, int xfmt, size_t rbx, const uint8_t* sx, size_t sbx, const void* W, size_t rbw,
                   const uint8_t* sw, size_t sbw, const float* bias, void* Y, int ytype, size_t ldy, int M, int N, int K,
                   tiermm_stream_t stream) {
  const char* who = "tiermm_mx_gemm";
  int st = check_size(who, M, N, K);
  if (st != TIERMM_OK || (st = check_fmt(who, xfmt)) != TIERMM_OK || M == 0 || N == 0) return st;
  if ((st = check_out(who, Y, ytype, ldy, bias, N)) != TIERMM_OK) return st;
  if ((st = check_mx_rows(who, "x", xfmt, Xq, rbx, sx, sbx, K)) != TIERMM_OK) return st;
  if ((st = check_mx_rows(who, "weight", MX_E2M1, W, rbw, sw, sbw, K)) != TIERMM_OK) return st;
  const MxArgs a = {(const uint8_t*)Xq, sx, (const uint8_t*)W, sw, bias, (uint8_t*)Y, rbx, sbx, rbw, sbw,
                    ldy * row_elem_bytes(ytype), M, N, K, mx_padded(K) / kMxStep};
  return gemm(a, xfmt, ytype, (hipStream_t)stream, who);
}

size_t tiermm_mx_linear_ws_bytes(int xfmt, int M, int N, int K) {
  if (M < 1 || N < 1 || M > (1 << 20)) return 0;
  const size_t rb = mx_row_bytes(xfmt, K);
  return rb ? M * (rb + mx_scales(K)) : 0;
}

int tiermm_mx_linear(const void* x, int xtype, size_t ldx, int xfmt, const void* W, size_t rbw, const uint8_t* sw,
                     size_t sbw, const float* bias, void* Y, int ytype, size_t ldy, int M, int N, int K, void* ws,
                     size_t ws_bytes, tiermm_stream_t stream) {
  const char* who = "tiermm_mx_linear";
  int st = check_size(who, M, N, K);
  if (st != TIERMM_OK || (st = check_fmt(who, xfmt)) != TIERMM_OK) return st;
  const int es = row_elem_bytes(xtype);
  if (!es) return set_error(TIERMM_UNSUPPORTED, "%s: x of type %d", who, xtype);
  if (bad_stride(ldx, K)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, K);
  if (M == 0 || N == 0) return TIERMM_OK;
  if (!x || misaligned(x, es)) return set_error(TIERMM_EINVAL, "%s: null or misaligned x", who);
  if ((st = check_out(who, Y, ytype, ldy, bias, N)) != TIERMM_OK) return st;
  if ((st = check_mx_rows(who, "weight", MX_E2M1, W, rbw, sw, sbw, K)) != TIERMM_OK) return st;
  if (misaligned(ws, 16)) return set_error(TIERMM_EINVAL, "%s: workspace not 16-byte aligned", who);
  if (fuses(xfmt, M, K)) {
    const MxArgs a = {(const uint8_t*)x, nullptr, (const uint8_t*)W, sw, bias, (uint8_t*)Y, ldx * es, 0, rbw, sbw,
                      ldy * row_elem_bytes(ytype), M, N, K, mx_padded(K) / kMxStep};
    return fused(a, xtype, xfmt, ytype, (hipStream_t)stream, who);
  }
  void* w = nullptr;
  if ((st = get_workspace(ws, ws_bytes, tiermm_mx_linear_ws_bytes(xfmt, M, N, K), &w, who)) != TIERMM_OK) return st;
  const size_t rbx = mx_row_bytes(xfmt, K), sbx = mx_scales(K);
  uint8_t *q = (uint8_t*)w, *sx = q + M * rbx;
  if ((st = quant(x, xtype, ldx, xfmt, q, rbx, sx, sbx, M, K, (hipStream_t)stream, who)) != TIERMM_OK) return st;
  const MxArgs a = {q, sx, (const uint8_t*)W, sw, bias, (uint8_t*)Y, rbx, sbx, rbw, sbw, ldy * row_elem_bytes(ytype), M, N,
                    K, mx_padded(K) / kMxStep};
  return gemm(a, xfmt, ytype, (hipStream_t)stream, who);
}

}  // extern "C"
