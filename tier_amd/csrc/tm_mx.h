// tm_mx.h -- microscaled rows: E2M1 (4-bit) or E4M3 (8-bit) elements with an E8M0 scale (the
// byte b stands for 2^(b - 127), 255 for NaN) for every 32 of them, after the OCP formats of these
// names.  A row's elements are padded with zeros to whole 256 and its scales to whole 16 bytes.
#pragma once

#include "tm_rows.h"

namespace tiermm {

enum : int { MX_E2M1 = TIERMM_MX_E2M1, MX_E4M3 = TIERMM_MX_E4M3 };  // bits of an element

constexpr int kMxStep = 256;        // elements of whole steps
constexpr int kMxMaxK = 1 << 20;
constexpr int mx_padded(int K) { return (K + kMxStep - 1) / kMxStep * kMxStep; }
constexpr int mx_scales(int K) { return (K + 511) / 512 * 16; }

// Scale byte of a block whose largest magnitude has the fp32 bits `top`: floor(log2 max) less the
// exponent of the format's largest number (6, 448), not below 2^-127.  A block that holds a NaN or an
// infinity has the scale NaN.
template <int FMT>
__device__ __forceinline__ int mx_scale_of(uint32_t top) {
  return top >= 0x7f800000u ? 255 : max((int)(top >> 23) - (FMT == MX_E2M1 ? 2 : 8), 0);
}
// What a block's elements are multiplied with: 2^(127 - byte), exactly (0 under the scale NaN).
__device__ __forceinline__ float mx_inverse(int byte) {
  return byte == 255 ? 0.f : __uint_as_float((uint32_t)(254 - byte) << 23);
}

// N (4 or 8) elements under their block's inverse as codes, packed from the low bits up: to nearest even,
// magnitudes past the format's largest number become it.  (An infinity or a NaN: 0, of a block
// whose scale says so.)
template <int FMT, int N>
__device__ __forceinline__ void mx_codes(const float (&v)[N], float inverse, uint32_t* out) {
  float s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = inverse == 0.f ? 0.f : v[i] * inverse;
    if constexpr (FMT == MX_E4M3) s[i] = __builtin_amdgcn_fmed3f(s[i], -448.f, 448.f);
  }
  if constexpr (FMT == MX_E2M1) {
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, s[0], s[1], 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[2], s[3], 1.f, 1);
    if constexpr (N == 8) {
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[4], s[5], 1.f, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[6], s[7], 1.f, 3);
    }
    out[0] = w;
  } else {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(s[4 * j], s[4 * j + 1], 0, false);
      out[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[4 * j + 2], s[4 * j + 3], w, true);
    }
  }
}

// The codes of N elements to the place of element c of a row.
template <int FMT, int N>
__device__ __forceinline__ void mx_put(uint8_t* row, int c, const uint32_t* w) {
  uint8_t* p = row + (FMT == MX_E2M1 ? c / 2 : c);
  if constexpr (N * FMT == 64) *(u32x2*)p = u32x2{w[0], w[1]};
  else if constexpr (N * FMT == 32) *(uint32_t*)p = w[0];
  else *(uint16_t*)p = (uint16_t)w[0];
}

// The largest of `top` over the neighbouring lanes that hold one block, L (4 or 8) of them.
template <int L>
__device__ __forceinline__ uint32_t mx_block_top(uint32_t top) {
  auto other = [&](auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, decltype(ctrl)::value, 0xf, 0xf, true);
  };
  top = max(top, other(std::integral_constant<int, 0xB1>()));  // quad_perm [1, 0, 3, 2]
  top = max(top, other(std::integral_constant<int, 0x4E>()));  // quad_perm [2, 3, 0, 1]
  if constexpr (L == 8) top = max(top, other(std::integral_constant<int, 0x141>()));  // row_half_mirror
  return top;
}

// Elements c .. c + N - 1 of a row, the lanes of a block side by side, as codes; one of the lanes
// stores the block's scale.
template <int FMT, int N>
__device__ __forceinline__ void mx_store(uint8_t* q, uint8_t* scales, int c, const float (&v)[N]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  const int byte = mx_scale_of<FMT>(mx_block_top<32 / N>(top));
  uint32_t w[2];
  mx_codes<FMT>(v, mx_inverse(byte), w);
  mx_put<FMT, N>(q, c, w);
  if (c % 32 == 0) scales[c / 32] = (uint8_t)byte;
}

// Bytes of a row of K elements of a format, 0 for a format that is none or a K that is not supported.
inline size_t mx_row_bytes(int fmt, int K) {
  if ((fmt != MX_E2M1 && fmt != MX_E4M3) || K < 1 || K > kMxMaxK) return 0;
  return (size_t)mx_padded(K) / 8 * fmt;
}

// f(std::integral_constant<int, FMT>) for a format already checked.
template <class F>
inline void with_mx(int fmt, F f) {
  if (fmt == MX_E2M1) f(std::integral_constant<int, MX_E2M1>());
  else f(std::integral_constant<int, MX_E4M3>());
}

// Checks of a side's rows and of their scales.
inline int check_mx_rows(const char* who, const char* what, int fmt, const void* q, size_t rb, const void* scales,
                         size_t sb, int K) {
  if (!q || !scales) return set_error(TIERMM_EINVAL, "%s: null %s", who, what);
  if (bad_stride(rb, mx_row_bytes(fmt, K)) || rb % 16 || (uintptr_t)q % 16)
    return set_error(TIERMM_EINVAL, "%s: %s rows of %zu bytes (whole 16-byte units from %zu up, 16-byte aligned)", who,
                     what, rb, mx_row_bytes(fmt, K));
  if (bad_stride(sb, mx_scales(K)) || sb % 16 || (uintptr_t)scales % 16)
    return set_error(TIERMM_EINVAL, "%s: %s scales of %zu bytes a row (whole 16-byte units from %d up, 16-byte aligned)",
                     who, what, sb, mx_scales(K));
  return TIERMM_OK;
}

}  // namespace tiermm
