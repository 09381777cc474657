// norm.hip -- RMS norm with the residual's addition, its output as rows, as int8 codes or as
// microscaled codes, and its gradient.  No reference entry points (its own norms are kernels of
// the engine, fp32 in and out); here it stands in front of the int8 and microscaled products,
// whose quantizer it spares.
//
//   h = T(x + residual)         T: the rows' type; without a residual h = x
//   r = fp32((mean(h^2) + eps)^-1/2)
//   y = (h r) gain              two fp32 products
//
// The mean and r's root are held in 64 bits, and the squares of a row are added in one order whatever the number of rows:
// 16 bytes by a lane (in rows of more than 4096 such units what one of 1024 threads takes), the sums of 64 lanes in
// pairs, and those of up to 64 such groups in pairs.  r and every code behind it is then the same in any call.  (Another
// order gives another r where it falls next to a border between two fp32 numbers, one row in some 2^25.)
#include "tm_i8.h"
#include "tm_mx.h"

#include <cmath>

namespace tiermm {
namespace {

struct NormArgs {
  const uint8_t *x, *res;  // res or null
  const float* gain;
  uint8_t *h, *y;          // or null
  uint8_t* q;
  void* scale;             // int8: float[M]; microscaled: bytes, sb a row
  float* rstd;             // or null
  size_t ldx, ldr, ldh, ldy, rb, sb;  // bytes
  float eps;
  int K, Kp;               // Kp: elements that q's row holds (K without q)
};

// What q holds.
enum : int { Q_NONE = 0, Q_I8 = 1, Q_E4M3 = 2, Q_E2M1 = 3 };

typedef f32x4 f32x4_a4 __attribute__((aligned(4)));

template <int N>
__device__ __forceinline__ void load_gain(const float* gain, int c, int K, float (&g)[N]) {
  if (c + N <= K) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4 v = *(const f32x4_a4*)(gain + c + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) g[i + j] = v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = c + i < K ? gain[c + i] : 0.f;
  }
}

// What f makes of a value of all lanes (f commutes), in every lane: in a row of 16 with lanes 1, 2, 7 and 15 away, which
// by then hold what lanes 4 and 8 away do, then the rows.  Moves within the registers: shuffles go through LDS.
template <class T, class F>
__device__ __forceinline__ T wave_join(T v, F f) {
  constexpr int N = sizeof(T) / 4;
  struct Words {
    uint32_t w[N];
  };
  auto lanes = [&](auto ctrl) __attribute__((always_inline)) {
    Words t = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < N; ++i)
      t.w[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)t.w[i], decltype(ctrl)::value, 0xf, 0xf, true);
    v = f(v, __builtin_bit_cast(T, t));
  };
  lanes(std::integral_constant<int, 0xB1>());   // quad_perm [1, 0, 3, 2]
  lanes(std::integral_constant<int, 0x4E>());   // quad_perm [2, 3, 0, 1]
  lanes(std::integral_constant<int, 0x141>());  // row_half_mirror
  lanes(std::integral_constant<int, 0x140>());  // row_mirror
  auto rows = [&](auto swap) __attribute__((always_inline)) {
    Words a = __builtin_bit_cast(Words, v), b = a;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const auto t = swap(a.w[i]);
      a.w[i] = t[0], b.w[i] = t[1];
    }
    v = f(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
  };
  rows([](uint32_t a) { return __builtin_amdgcn_permlane16_swap(a, a, false, false); });
  rows([](uint32_t a) { return __builtin_amdgcn_permlane32_swap(a, a, false, false); });
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
  return wave_join(v, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One row a workgroup.  R > 0: the row has at most R units of 16 bytes a thread and stays in
// registers, all its loads on their way at once; R = 0: any row, read again from h (or x and
// the residual) for each pass.  STREAM: rows come from past the caches, and h goes there.
//
// Bound by memory: 4096 x 5120 bf16 with a residual, int8 out, 28.5 us (5.2 TB/s, where a large copy moves 4.8),
// through the caches 32.6, and 38.3 with one unit a thread.  8 rows of 5120 fp32 4.7 us.
template <int XT, int Q, int R, bool STREAM>
__global__ __launch_bounds__(1024) void norm_kernel(const NormArgs a) {
  using X = Rows<XT>;
  constexpr int EPU = X::EPU, NU = R > 0 ? R : 1;
  __shared__ double sums[NU * 16];
  __shared__ uint32_t tops[16];
  const int m = blockIdx.x, tid = threadIdx.x, k0 = tid * EPU, step = blockDim.x * EPU, K = a.K, nw = blockDim.x / 64;
  auto get = [](const uint8_t* row, int k, int n) __attribute__((always_inline)) {
    if constexpr (STREAM) return X::get_nt(row, k, n);
    else return X::get(row, k, n);
  };
  const uint8_t* xr = a.x + (size_t)m * a.ldx;
  const uint8_t* rr = a.res ? a.res + (size_t)m * a.ldr : nullptr;
  uint8_t* hr = a.h ? a.h + (size_t)m * a.ldh : nullptr;
  const u32x4 none = {0u, 0u, 0u, 0u};
  auto add = [](u32x4 x, u32x4 r) __attribute__((always_inline)) {
    float v[EPU], w[EPU];
    X::widen(x, v);
    X::widen(r, w);
#pragma unroll
    for (int i = 0; i < EPU; ++i) v[i] += w[i];
    return X::narrow(v);
  };
  auto squares = [&](u32x4 u, double s) __attribute__((always_inline)) {
    float v[EPU];
    X::widen(u, v);
#pragma unroll
    for (int i = 0; i < EPU; ++i) s = fma((double)v[i], (double)v[i], s);
    return s;
  };
  double part[NU];  // of this lane's units, one by one (R = 0: of all)
#pragma unroll
  for (int i = 0; i < NU; ++i) part[i] = 0.;
  u32x4 u[NU];
  float g[NU][EPU];
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) u[i] = k0 + i * step < K ? get(xr, k0 + i * step, K) : none;
    if (rr) {
      u32x4 w[NU];
#pragma unroll
      for (int i = 0; i < R; ++i) w[i] = k0 + i * step < K ? get(rr, k0 + i * step, K) : none;
#pragma unroll
      for (int i = 0; i < R; ++i) u[i] = add(u[i], w[i]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (k0 + i * step < K) load_gain(a.gain, k0 + i * step, K, g[i]);
      else
#pragma unroll
        for (int j = 0; j < EPU; ++j) g[i][j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (hr && k0 + i * step < K) {
        if constexpr (STREAM) X::set_nt(hr, k0 + i * step, K, u[i]);
        else X::set(hr, k0 + i * step, K, u[i]);
      }
      part[i] = squares(u[i], 0.);
    }
  } else {
    for (int k = k0; k < K; k += step) {
      u32x4 v = X::get(xr, k, K);
      if (rr) v = add(v, X::get(rr, k, K));
      if (hr) X::set(hr, k, K, v);
      part[0] = squares(v, part[0]);
    }
  }
#pragma unroll
  for (int i = 0; i < NU; ++i) part[i] = wave_sum(part[i]);
  if ((tid & 63) == 0)  // group i * nw + wave of 64 units
#pragma unroll
    for (int i = 0; i < NU; ++i) sums[i * nw + (tid >> 6)] = part[i];
  __syncthreads();
  const int lane = tid & 63;
  const double s = wave_sum(lane < NU * nw ? sums[lane] : 0.);
  const float r = (float)(1. / sqrt(s / K + (double)a.eps));
  if (a.rstd && tid == 0) a.rstd[m] = r;

  // elements k .. of y, in fp32
  auto values = [&](u32x4 h, const float (&gain)[EPU], float (&v)[EPU]) __attribute__((always_inline)) {
    X::widen(h, v);
#pragma unroll
    for (int j = 0; j < EPU; ++j) v[j] = (v[j] * r) * gain[j];
  };
  auto value_at = [&](int k, float (&v)[EPU]) __attribute__((always_inline)) {  // R = 0
    float gain[EPU];
    if (k >= K) {
#pragma unroll
      for (int j = 0; j < EPU; ++j) v[j] = 0.f;
      return;
    }
    u32x4 h;
    if (hr) h = X::get(hr, k, K);
    else {
      h = X::get(xr, k, K);
      if (rr) h = add(h, X::get(rr, k, K));
    }
    load_gain(a.gain, k, K, gain);
    values(h, gain, v);
  };
  uint8_t* yr = a.y ? a.y + (size_t)m * a.ldy : nullptr;
  uint8_t* q = Q != Q_NONE ? a.q + (size_t)m * a.rb : nullptr;
  uint8_t* sc = Q >= Q_E4M3 ? (uint8_t*)a.scale + (size_t)m * a.sb : nullptr;
  constexpr int FMT = Q == Q_E4M3 ? MX_E4M3 : MX_E2M1;
  uint32_t top = 0;
  // rows and microscaled codes need nothing of the rest of the row
  auto finish = [&](int k, const float (&v)[EPU]) __attribute__((always_inline)) {
    if (yr && k < K) X::set(yr, k, K, X::narrow(v));
    if constexpr (Q == Q_I8) top = top_bits(v, top);
    if constexpr (Q >= Q_E4M3)
      if (k < a.Kp) mx_store<FMT>(q, sc, k, v);
  };
  float v[NU][EPU];
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      values(u[i], g[i], v[i]);
      if (k0 + i * step >= K)  // (0 times an infinite r)
#pragma unroll
        for (int j = 0; j < EPU; ++j) v[i][j] = 0.f;
      else if (k0 + i * step + EPU > K)
#pragma unroll
        for (int j = 0; j < EPU; ++j) v[i][j] = k0 + i * step + j < K ? v[i][j] : 0.f;
      finish(k0 + i * step, v[i]);
    }
  } else {
    for (int k = k0; k < (Q == Q_NONE ? K : a.Kp); k += step) {
      value_at(k, v[0]);
      if (k < K && k + EPU > K)
#pragma unroll
        for (int j = 0; j < EPU; ++j) v[0][j] = k + j < K ? v[0][j] : 0.f;
      finish(k, v[0]);
    }
  }
  if constexpr (Q >= Q_E4M3) {  // scales of blocks behind the padded row
    const int b = a.Kp / 32 + tid;
    if (b < mx_scales(K)) sc[b] = 0;
  }
  if constexpr (Q == Q_I8) {
    top = wave_join(top, [](uint32_t a, uint32_t b) { return max(a, b); });
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    for (int w = 0; w < nw; ++w) top = max(top, tops[w]);
    const RowScale rs = row_scale_of(top);
    auto put = [&](int k, const float (&t)[EPU]) __attribute__((always_inline)) {
      if constexpr (EPU == 8) *(u32x2*)(q + k) = u32x2{codes4(t, rs), codes4(t + 4, rs)};
      else *(uint32_t*)(q + k) = codes4(t, rs);
    };
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (k0 + i * step < a.Kp) put(k0 + i * step, v[i]);
    } else {
      for (int k = k0; k < a.Kp; k += step) {
        value_at(k, v[0]);
        if (k < K && k + EPU > K)
#pragma unroll
          for (int j = 0; j < EPU; ++j) v[0][j] = k + j < K ? v[0][j] : 0.f;
        put(k, v[0]);
      }
    }
    if (tid == 0) ((float*)a.scale)[m] = rs.sc;
  }
}

// -------------------------------------------------------------------- gradient
// With xh = h r and d = dy gain: dx = r (d - xh mean(d xh)) + dh, dgain = sum over rows of dy xh.
struct GradArgs {
  const uint8_t *dy, *h, *dh;  // dh or null
  const float *gain, *rstd;
  uint8_t* dx;
  float* part;                 // [grid][K] sums of dy xh, or null
  size_t ldy, ldh, lddh, lddx;  // bytes
  int M, K;
};

// A workgroup takes rows blockIdx.x, + gridDim.x, ...; a thread keeps its columns of dgain in
// registers (R = 0: in its row of `part`).  STREAM: rows come from past the caches.
template <int XT, int R, bool STREAM>
__global__ __launch_bounds__(1024) void norm_grad_kernel(const GradArgs a) {
  using X = Rows<XT>;
  constexpr int EPU = X::EPU, NU = R > 0 ? R : 1;
  __shared__ float sums[2][16];
  const int tid = threadIdx.x, k0 = tid * EPU, step = blockDim.x * EPU, K = a.K, nw = blockDim.x / 64;
  auto get = [](const uint8_t* row, int k, int n) __attribute__((always_inline)) {
    if constexpr (STREAM) return X::get_nt(row, k, n);
    else return X::get(row, k, n);
  };
  const u32x4 none = {0u, 0u, 0u, 0u};
  float* part = a.part ? a.part + (size_t)blockIdx.x * K : nullptr;
  float g[NU][EPU], dg[NU][EPU];
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int j = 0; j < EPU; ++j) dg[i][j] = g[i][j] = 0.f;
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (k0 + i * step < K) load_gain(a.gain, k0 + i * step, K, g[i]);
  }
  int turn = 0;
  auto row_sum = [&](float s) __attribute__((always_inline)) {
    s = wave_sum(s);
    if ((tid & 63) == 0) sums[turn][tid >> 6] = s;
    __syncthreads();
    s = sums[turn][0];
    for (int w = 1; w < nw; ++w) s += sums[turn][w];
    turn ^= 1;  // the next row's sums do not meet slow readers of this one's
    return s;
  };
  auto products = [&](u32x4 dyu, u32x4 hu, const float (&gain)[EPU], float r, float (&d)[EPU], float (&xh)[EPU],
                      float (&acc)[EPU], float s) __attribute__((always_inline)) {
    X::widen(dyu, d);
    X::widen(hu, xh);
#pragma unroll
    for (int j = 0; j < EPU; ++j) {
      xh[j] *= r;
      acc[j] = fmaf(d[j], xh[j], acc[j]);
      d[j] *= gain[j];
      s = fmaf(d[j], xh[j], s);
    }
    return s;
  };
  auto grad = [&](const float (&d)[EPU], const float (&xh)[EPU], float r, float mean, u32x4 dhu) __attribute__((always_inline)) {
    float v[EPU], e[EPU];
    X::widen(dhu, e);
#pragma unroll
    for (int j = 0; j < EPU; ++j) v[j] = fmaf(r, fmaf(-xh[j], mean, d[j]), e[j]);
    return X::narrow(v);
  };
  for (int m = blockIdx.x; m < a.M; m += gridDim.x) {
    const uint8_t *dyr = a.dy + (size_t)m * a.ldy, *hr = a.h + (size_t)m * a.ldh;
    const uint8_t* dhr = a.dh ? a.dh + (size_t)m * a.lddh : nullptr;
    uint8_t* dxr = a.dx + (size_t)m * a.lddx;
    const float r = a.rstd[m];
    float s = 0.f;
    if constexpr (R > 0) {
      u32x4 dyu[NU], hu[NU], dhu[NU];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int k = k0 + i * step;
        dyu[i] = k < K ? get(dyr, k, K) : none;
        hu[i] = k < K ? get(hr, k, K) : none;
        dhu[i] = dhr && k < K ? get(dhr, k, K) : none;
      }
      float d[NU][EPU], xh[NU][EPU];
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (k0 + i * step < K) s = products(dyu[i], hu[i], g[i], r, d[i], xh[i], dg[i], s);
      const float mean = row_sum(s) / K;
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (k0 + i * step < K) X::set(dxr, k0 + i * step, K, grad(d[i], xh[i], r, mean, dhu[i]));
    } else {
      float d[EPU], xh[EPU];
      for (int k = k0; k < K; k += step) {
        load_gain(a.gain, k, K, g[0]);
#pragma unroll
        for (int j = 0; j < EPU; ++j) dg[0][j] = 0.f;
        s = products(X::get(dyr, k, K), X::get(hr, k, K), g[0], r, d, xh, dg[0], s);
        if (part)
#pragma unroll
          for (int j = 0; j < EPU; ++j)
            if (k + j < K) part[k + j] = m == (int)blockIdx.x ? dg[0][j] : part[k + j] + dg[0][j];
      }
      const float mean = row_sum(s) / K;
      for (int k = k0; k < K; k += step) {
        load_gain(a.gain, k, K, g[0]);
        products(X::get(dyr, k, K), X::get(hr, k, K), g[0], r, d, xh, dg[0], 0.f);
        X::set(dxr, k, K, grad(d, xh, r, mean, dhr ? X::get(dhr, k, K) : none));
      }
    }
  }
  if (R > 0 && part)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < EPU; ++j)
        if (k0 + i * step + j < K) part[k0 + i * step + j] = dg[i][j];
}

// dgain[k] = sum of n partial rows, in a fixed order.
constexpr int kSumCols = 32, kSumParts = 32;
__global__ __launch_bounds__(kSumCols * kSumParts) void norm_gain_kernel(const float* __restrict__ part, int n, int K,
                                                                         float* __restrict__ dgain) {
  __shared__ float s[kSumParts][kSumCols];
  const int c = threadIdx.x % kSumCols, p = threadIdx.x / kSumCols, k = blockIdx.x * kSumCols + c;
  float v = 0.f;
  if (k < K)
    for (int i = p; i < n; i += kSumParts) v += part[(size_t)i * K + k];
  s[p][c] = v;
  __syncthreads();
  if (p == 0 && k < K) {
#pragma unroll
    for (int i = 1; i < kSumParts; ++i) v += s[i][c];
    dgain[k] = v;
  }
}

// Rows up to which a thread takes one unit where that is enough: few rows wait for their latency, many for memory, and
// take two.  int8 out of bf16 rows and a residual, us with one and two units: 2048 columns 64 rows 3.4 / 3.7, 512 4.0
// / 4.4, 768 4.7 / 4.7, 1024 5.8 / 5.3, 4096 15.2 / 12.6; 5120 columns 64 rows 4.1 / 4.3, 256 4.7 / 4.7, 512 7.1 /
// 6.5, 1024 12.0 / 10.5, 4096 38 / 28.5.  (Long rows would change over at fewer rows: 8192 columns 64 rows 4.7 /
// 4.2.)
constexpr int kNormWide = 512;
// Bytes read by a call from which on its rows are streamed: what the last-level cache does not keep for the next
// call. Streamed / through the caches, us, bf16 rows of 5120 columns: with a residual 32 MiB read 14.3 / 13.7, 48
// 19.4 / 19.1, 64 24.1 / 27.2, 80 28.6 / 32.6, 192 60 / 66; without 32 MiB 16.2 / 13.8, 64 26.7 / 27.6, 80 31.8 /
// 34.1, 128 51.1 / 50.5; the gradient with dh 48 MiB 25.2 / 22.0, 64 28.9 / 27.9, 80 31.4 / 33.3, 192 54 / 61.
constexpr size_t kNormStream = (size_t)72 << 20;

// Units a thread (0: any number) and threads for rows of so many units.
struct Shape {
  int r, threads;
};
Shape shape_of(int units, bool one, int most) {
  for (int r = one || units <= 128 ? 1 : 2; r <= most; r *= 2) {
    const int threads = (units + 64 * r - 1) / (64 * r) * 64;
    if (threads <= 1024) return {r, threads};
  }
  return {0, 1024};
}
template <class F>
void with_shape(Shape h, F f) {
  if (h.r == 1) f(std::integral_constant<int, 1>());
  else if (h.r == 2) f(std::integral_constant<int, 2>());
  else if (h.r == 4) f(std::integral_constant<int, 4>());
  else f(std::integral_constant<int, 0>());
}

template <int Q>
int norm(const NormArgs& a, int xtype, int M, hipStream_t s, const char* who) {
  with_rows(xtype, [&](auto xt) {
    constexpr int XT = decltype(xt)::value, EPU = Rows<XT>::EPU;
    const Shape h = shape_of(((Q == Q_NONE ? a.K : a.Kp) + EPU - 1) / EPU, M <= kNormWide, 4);
    const bool stream = (size_t)M * a.K * Rows<XT>::ES * (a.res ? 2 : 1) >= kNormStream;
    with_shape(h, [&](auto r) {
      constexpr int R = decltype(r)::value;
      if (R && stream) norm_kernel<XT, Q, R, R != 0><<<M, h.threads, 0, s>>>(a);
      else norm_kernel<XT, Q, R, false><<<M, h.threads, 0, s>>>(a);
    });
  });
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

// Workgroups of the gradient, each with its rows' part of dgain: more of them read the rows faster, and leave more parts
// to add.  Rows of 5120 bf16 with dh, us with 64 / 128 / 256 / 512 workgroups: 128 rows 9.0 / 9.1, 256 rows 11.6 / 10.4 /
// 12.3, 512 rows 17.6 / 13.5 / 14.6 / 20.7, 1024 rows 27.1 / 19.3 / 17.5 / 21.1, 2048 rows 53 / 30 / 25.2 / 27.2, 4096 rows
// 256 44, 512 39.3 (4.3 TB/s), 768 50 (their rows are no whole rounds).  8 us more there where 16 columns of all parts
// were a workgroup's.
int grad_grid(int M) { return M > 2048 ? 512 : M > 384 ? 256 : std::min(M, 128); }

constexpr int kRows = (1 << 22) - 1;  // a launch has less than 2^32 threads

// Checks of what the forward entry points share; *es = bytes of an element.
int check_norm(const char* who, const void* x, int xtype, size_t ldx, const void* res, size_t ldr, const float* gain,
               float eps, const void* h, size_t ldh, const void* y, size_t ldy, const float* rstd, int M, int K, int* es) {
  *es = row_elem_bytes(xtype);
  if (!*es) return set_error(TIERMM_UNSUPPORTED, "%s: rows of type %d", who, xtype);
  if (M < 0 || K < 1) return set_error(TIERMM_EINVAL, "%s: bad size %d x %d", who, M, K);
  if (M > kRows || K > kMxMaxK) return set_error(TIERMM_UNSUPPORTED, "%s: %d x %d, at most %d x %d", who, M, K, kRows, kMxMaxK);
  if (!(eps >= 0.f) || std::isinf(eps)) return set_error(TIERMM_EINVAL, "%s: eps = %g", who, eps);
  if (bad_stride(ldx, K) || (res && bad_stride(ldr, K)) || (h && bad_stride(ldh, K)) || (y && bad_stride(ldy, K)))
    return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, K);
  if (M == 0) return TIERMM_OK;
  if (!x || !gain) return set_error(TIERMM_EINVAL, "%s: null buffer", who);
  if (misaligned(x, *es) || misaligned(res, *es) || misaligned(h, *es) || misaligned(y, *es) || misaligned(gain, 4) ||
      misaligned(rstd, 4))
    return set_error(TIERMM_EINVAL, "%s: misaligned buffer", who);
  return TIERMM_OK;
}

}  // namespace
}  // namespace tiermm

using namespace tiermm;

extern "C" {

int tiermm_rms_norm(const void* x, int xtype, size_t ldx, const void* residual, size_t ldr, const float* gain,
                    float eps, void* h, size_t ldh, void* y, size_t ldy, int8_t* q, size_t rb, float* scale,
                    float* rstd, int M, int K, tiermm_stream_t stream) {
  const char* who = "tiermm_rms_norm";
  int es;
  const int st = check_norm(who, x, xtype, ldx, residual, ldr, gain, eps, h, ldh, y, ldy, rstd, M, K, &es);
  if (st != TIERMM_OK) return st;
  if (q) {
    if (K > kMaxK) return set_error(TIERMM_UNSUPPORTED, "%s: int8 rows of K = %d, at most %d", who, K, kMaxK);
    if (bad_stride(rb, padded(K)) || rb % 16 || misaligned(q, 16))
      return set_error(TIERMM_EINVAL, "%s: int8 rows of %zu bytes (whole 16-byte units from %d up, 16-byte aligned)", who,
                       rb, padded(K));
    if (!scale || misaligned(scale, 4)) return set_error(TIERMM_EINVAL, "%s: null or misaligned scales", who);
  }
  if (M == 0) return TIERMM_OK;
  const NormArgs a = {(const uint8_t*)x, (const uint8_t*)residual, gain, (uint8_t*)h, (uint8_t*)y, (uint8_t*)q, scale,
                      rstd, ldx * es, ldr * es, ldh * es, ldy * es, rb, 0, eps, K, q ? padded(K) : K};
  return q ? norm<Q_I8>(a, xtype, M, (hipStream_t)stream, who) : norm<Q_NONE>(a, xtype, M, (hipStream_t)stream, who);
}

int tiermm_rms_norm_mx(const void* x, int xtype, size_t ldx, const void* residual, size_t ldr, const float* gain,
                       float eps, void* h, size_t ldh, void* y, size_t ldy, int fmt, void* q, size_t rb,
                       uint8_t* scales, size_t sb, float* rstd, int M, int K, tiermm_stream_t stream) {
  const char* who = "tiermm_rms_norm_mx";
  int es;
  int st = check_norm(who, x, xtype, ldx, residual, ldr, gain, eps, h, ldh, y, ldy, rstd, M, K, &es);
  if (st != TIERMM_OK) return st;
  if (!mx_row_bytes(fmt, K)) return set_error(TIERMM_UNSUPPORTED, "%s: format %d", who, fmt);
  if (M == 0) return TIERMM_OK;
  if ((st = check_mx_rows(who, "output", fmt, q, rb, scales, sb, K)) != TIERMM_OK) return st;
  const NormArgs a = {(const uint8_t*)x, (const uint8_t*)residual, gain, (uint8_t*)h, (uint8_t*)y, (uint8_t*)q, scales,
                      rstd, ldx * es, ldr * es, ldh * es, ldy * es, rb, sb, eps, K, mx_padded(K)};
  return fmt == MX_E4M3 ? norm<Q_E4M3>(a, xtype, M, (hipStream_t)stream, who)
                        : norm<Q_E2M1>(a, xtype, M, (hipStream_t)stream, who);
}

size_t tiermm_rms_norm_grad_ws_bytes(int M, int K) {
  if (M < 1 || K < 1 || M > kRows || K > kMxMaxK) return 0;
  return (size_t)grad_grid(M) * K * sizeof(float);
}

int tiermm_rms_norm_grad(const void* dy, int type, size_t ldy, const void* h, size_t ldh, const float* gain,
                         const float* rstd, const void* dh, size_t lddh, void* dx, size_t lddx, float* dgain, int M,
                         int K, void* ws, size_t ws_bytes, tiermm_stream_t stream) {
  const char* who = "tiermm_rms_norm_grad";
  const int es = row_elem_bytes(type);
  if (!es) return set_error(TIERMM_UNSUPPORTED, "%s: rows of type %d", who, type);
  if (M < 0 || K < 1) return set_error(TIERMM_EINVAL, "%s: bad size %d x %d", who, M, K);
  if (M > kRows || K > kMxMaxK) return set_error(TIERMM_UNSUPPORTED, "%s: %d x %d, at most %d x %d", who, M, K, kRows, kMxMaxK);
  if (bad_stride(ldy, K) || bad_stride(ldh, K) || (dh && bad_stride(lddh, K)) || bad_stride(lddx, K))
    return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, K);
  if (M && (!dy || !h || !gain || !rstd || !dx)) return set_error(TIERMM_EINVAL, "%s: null buffer", who);
  if (misaligned(dy, es) || misaligned(h, es) || misaligned(dh, es) || misaligned(dx, es) || misaligned(gain, 4) ||
      misaligned(rstd, 4) || misaligned(dgain, 4) || misaligned(ws, 4))
    return set_error(TIERMM_EINVAL, "%s: misaligned buffer", who);
  hipStream_t s = (hipStream_t)stream;
  const int grid = grad_grid(M);
  void* part = nullptr;
  if (dgain && M) {
    const int st = get_workspace(ws, ws_bytes, tiermm_rms_norm_grad_ws_bytes(M, K), &part, who);
    if (st != TIERMM_OK) return st;
  }
  if (M) {
    const GradArgs a = {(const uint8_t*)dy, (const uint8_t*)h, (const uint8_t*)dh, gain, rstd, (uint8_t*)dx, (float*)part,
                        ldy * es, ldh * es, lddh * es, lddx * es, M, K};
    with_rows(type, [&](auto xt) {
      constexpr int XT = decltype(xt)::value;
      // (four units of 16 bits do not fit the registers of 1024 threads)
      const Shape shape = shape_of((K + Rows<XT>::EPU - 1) / Rows<XT>::EPU, true, XT == QT_F32 ? 4 : 2);
      const bool stream = (size_t)M * K * es * (dh ? 3 : 2) >= kNormStream;
      with_shape(shape, [&](auto r) {
        constexpr int R = decltype(r)::value;
        if constexpr (R < 4 || XT == QT_F32) {
          if (R && stream) norm_grad_kernel<XT, R, R != 0><<<grid, shape.threads, 0, s>>>(a);
          else norm_grad_kernel<XT, R, false><<<grid, shape.threads, 0, s>>>(a);
        }
      });
    });
    TM_LAUNCH_CHECK(who);
  }
  if (dgain) {
    norm_gain_kernel<<<(K + kSumCols - 1) / kSumCols, kSumCols * kSumParts, 0, s>>>((const float*)part, M ? grid : 0, K, dgain);
    TM_LAUNCH_CHECK(who);
  }
  return TIERMM_OK;
}

}  // extern "C"
