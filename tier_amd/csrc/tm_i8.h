// tm_i8.h -- rows of int8 codes with a scale each, as the int8 products, the norm and the routed
// layer of a few tokens share them: padding, scales and codes of a row, and what a product's
// element is.
#pragma once

#include "tm_rows.h"

namespace tiermm {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 128;          // bytes of K a row holds a step
constexpr int kMaxK = 133120;       // whole steps up to 2^31 / 127^2

constexpr int padded(int K) { return (K + kStep - 1) / kStep * kStep; }

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
  // a scale of 0 or NaN has inv = 0: codes 0, whatever the element
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = (uint32_t)(int)(r.inv == 0.f ? 0.f : __builtin_rintf((v[i] * r.pre) * r.inv));
  // byte 0 of each
  const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
  return lo | hi;
}

template <int N>
__device__ __forceinline__ uint32_t top_bits(const float (&v)[N], uint32_t top) {
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  return top;
}

// One element of Y: the sum rounded to fp32, times sx * sw, plus the bias (0: none).  Where sx * sw
// is not a normal fp32 number the sum takes the smaller scale first: a product of a whole number that
// falls below the normal numbers is exact, and it overflows only if the element does.
__device__ __forceinline__ bool normal(float v) { return __builtin_amdgcn_classf(v, 0x108); }
__device__ __forceinline__ float scaled(int sum, float sx, float sw, float bias) {
  const float s = sx * sw;
  if (__builtin_expect(normal(s), 1)) return fmaf((float)sum, s, bias);
  const bool x_first = fabsf(sx) < fabsf(sw);  // (NaN: stays in the second product)
  return fmaf((float)sum * (x_first ? sx : sw), x_first ? sw : sx, bias);
}
// The same, bit for bit, for scales of which neither is far: their products are normal, 0 or NaN.
__device__ __forceinline__ float scaled_near(int sum, float sx, float sw, float bias) {
  return fmaf((float)sum, sx * sw, bias);
}
inline bool misaligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

}  // namespace tiermm
