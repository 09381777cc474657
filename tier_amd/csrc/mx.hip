// mx.hip -- microscaled products: Y[m][n] = sum over blocks b of 32 of 2^(ex + ew - 254)
// sum_{k in b} cx[m][k] cw[n][k] (+ bias[n]), with W in E2M1, x in E2M1 or E4M3, and the quantizer
// that makes such rows.  No reference function (the reference expands its MXFP4 blocks to fp16).
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes the scales with the operands: lane l holds row l % 16, and
// of a step of 128 elements block l / 16 (E2M1: its 16 bytes; E4M3: 16 bytes of each half of the
// step) and that block's scale.
#include "tm_mx.h"

namespace tiermm {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------- quantizer
// A thread takes one unit of 16 bytes of a row; the lanes of a block are neighbours.
template <int XT, int FMT>
__global__ __launch_bounds__(256) void mx_quant_kernel(const uint8_t* __restrict__ x, size_t ldx, uint8_t* __restrict__ q,
                                                       size_t rb, uint8_t* __restrict__ scales, size_t sb, int K, int Kp) {
  using X = Rows<XT>;
  const int m = blockIdx.x, k = (blockIdx.y * 256 + threadIdx.x) * X::EPU;
  uint8_t* sc = scales + (size_t)m * sb;
  const int b = Kp / 32 + threadIdx.x;  // scales of blocks behind the padded row
  if (blockIdx.y == 0 && b < mx_scales(K)) sc[b] = 0;
  if (k >= Kp) return;
  float v[X::EPU];
  X::widen(k < K ? X::get(x + (size_t)m * ldx, k, K) : u32x4{0u, 0u, 0u, 0u}, v);
  mx_store<FMT>(q + (size_t)m * rb, sc, k, v);
}

int quant(const void* x, int xtype, size_t ldx, int fmt, void* q, size_t rb, uint8_t* scales, size_t sb, int M, int K,
          hipStream_t s, const char* who) {
  with_rows(xtype, [&](auto xt) {
    with_mx(fmt, [&](auto f) {
      constexpr int XT = decltype(xt)::value, FMT = decltype(f)::value, EPU = Rows<XT>::EPU;
      const dim3 grid(M, (mx_padded(K) / EPU + 255) / 256);
      mx_quant_kernel<XT, FMT><<<grid, 256, 0, s>>>((const uint8_t*)x, ldx * Rows<XT>::ES, (uint8_t*)q, rb, scales, sb, K,
                                                    mx_padded(K));
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
// An element of E4M3 spans 2^-9 to 448, so small ones next to large ones lose bits: 1e-5 of the result
// on normal rows.  Where Y is fp32 x is therefore multiplied in two parts, magnitudes from 2 up and those
// below: with W's exponents of 0 to 2 the first has sums of exponents of 10 at most and lowest bits of 2^-3
// (2^-2 of x, half of it by W), the second 2 and 2^-10, so every product keeps its bits.  16-bit outputs, which
// round to 2^-9 or 2^-12, take x as it is: half the products of a large batch.
template <int XF, int YT>
constexpr int kParts = XF == MX_E4M3 && YT == QT_F32 ? 2 : 1;

// The codes of magnitude 2 and more, whose bit 6 is set, and zeros.
__device__ __forceinline__ uint32_t mx_large(uint32_t c) {
  const uint32_t bit = c & 0x40404040u, top = bit << 1;
  return c & (top | (top - (bit >> 6)));
}
__device__ __forceinline__ i32x8 mx_large(const i32x8& x) {
  i32x8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (int)mx_large((uint32_t)x[i]);
  return y;
}

// One wave a tile of 16 x 16, operands straight from memory.
template <int YT, int XF>
__global__ __launch_bounds__(64) void mx_simple_kernel(const MxArgs a) {
  using Y = Rows<YT>;
  const int lane = threadIdx.x, r = lane & 15, g = lane >> 4, m = blockIdx.y * 16 + r, n0 = blockIdx.x * 16;
  const int mr = min(m, a.M - 1), nr = min(n0 + r, a.N - 1);
  const uint8_t *x = a.X + (size_t)mr * a.rbx, *w = a.W + (size_t)nr * a.rbw;
  const uint8_t *sx = a.sx + (size_t)mr * a.sbx, *sw = a.sw + (size_t)nr * a.sbw;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int t = 0; t < 2 * a.nk; ++t) {
    const i32x4 wf = *(const i32x4*)(w + (size_t)t * 64 + g * 16);
    i32x8 A = {wf[0], wf[1], wf[2], wf[3], 0, 0, 0, 0}, B;
    if constexpr (XF == MX_E2M1) {
      const i32x4 xf = *(const i32x4*)(x + (size_t)t * 64 + g * 16);
      B = i32x8{xf[0], xf[1], xf[2], xf[3], 0, 0, 0, 0};
    } else {
      const i32x4 lo = *(const i32x4*)(x + (size_t)t * 128 + g * 16), hi = *(const i32x4*)(x + (size_t)t * 128 + 64 + g * 16);
      B = i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
    const int ws = sw[t * 4 + g], xs = sx[t * 4 + g];
    auto product = [&](const i32x8& b) __attribute__((always_inline)) {
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, b, acc, 4, XF == MX_E2M1 ? 4 : 0, 0, ws, 0, xs);
    };
    if constexpr (kParts<XF, YT> == 1) {
      product(B);
    } else {
      const i32x8 large = mx_large(B);
      product(large);
      product(B ^ large);
    }
  }
  if (m >= a.M) return;
  const int n = n0 + 4 * g;
  float o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = acc[i] + (a.bias ? a.bias[min(n + i, a.N - 1)] : 0.f);
  if (n < a.N) Y::put4(a.Y + (size_t)m * a.ldy + (size_t)n * Y::ES, o, min(4, a.N - n));
}

int gemm(const MxArgs& a, int xfmt, int ytype, hipStream_t s, const char* who) {
  with_rows(ytype, [&](auto yt) {
    with_mx(xfmt, [&](auto f) {
      mx_simple_kernel<decltype(yt)::value, decltype(f)::value>
          <<<dim3((a.N + 15) / 16, (a.M + 15) / 16), 64, 0, s>>>(a);
    });
  });
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

bool misaligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

int check_size(const char* who, int M, int N, int K) {
  if (M < 0 || N < 0 || K < 1) return set_error(TIERMM_EINVAL, "%s: bad size %d x %d x %d", who, M, N, K);
  if (K > kMxMaxK) return set_error(TIERMM_UNSUPPORTED, "%s: K = %d, at most %d", who, K, kMxMaxK);
  if (M > (1 << 20)) return set_error(TIERMM_UNSUPPORTED, "%s: %d rows, at most %d", who, M, 1 << 20);
  if (N > (1 << 26)) return set_error(TIERMM_UNSUPPORTED, "%s: %d columns, at most %d", who, N, 1 << 26);
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
