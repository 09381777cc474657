// tm_rows.h -- rows of fp32, fp16 or bf16 elements, read and written in units of 16
// bytes as fp32 values.  Rows start wherever their elements may (a stride of any
// number of elements): the unit types promise no more than the element's alignment,
// and global memory takes dwordx4 accesses at any address.
#pragma once

#include "tm_device.h"

namespace tiermm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));

// Rows of type XT (QT_F32, QT_F16, QT_BF16): ES bytes an element, EPU elements a unit.
template <int XT>
struct Rows {
  static_assert(XT == QT_F32 || XT == QT_F16 || XT == QT_BF16, "row types");
  static constexpr int ES = XT == QT_F32 ? 4 : 2, EPU = 16 / ES;

  static __device__ __forceinline__ void widen(u32x4 u, float (&v)[EPU]) {
    if constexpr (XT == QT_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = one((uint16_t)(u[i] & 0xffffu));
        v[2 * i + 1] = one((uint16_t)(u[i] >> 16));
      }
    }
  }
  // Rounds to nearest even.
  static __device__ __forceinline__ u32x4 narrow(const float (&v)[EPU]) {
    u32x4 u;
    if constexpr (XT == QT_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = pair(v[2 * i], v[2 * i + 1]);
    }
    return u;
  }
  static __device__ __forceinline__ u32x4 raw(const uint8_t* p) { return *(const u32x4_a2*)p; }
  static __device__ __forceinline__ void put(uint8_t* p, u32x4 u) { *(u32x4_a2*)p = u; }
  // A store past the caches, of what is not read again soon.
  static __device__ __forceinline__ void set_nt(uint8_t* row, int c, int cols, u32x4 u) {
    uint8_t* p = row + (size_t)c * ES;
    if (c + EPU <= cols) __builtin_nontemporal_store(u, (u32x4_a2*)p);
    else put_part(p, u, cols - c);
  }
  // The first n elements at p as a unit (0 behind them), and the first n of a unit to p: bits as they are.
  static __device__ __forceinline__ u32x4 raw_part(const uint8_t* p, int n) {
    u32x4 u = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < EPU; ++i) {
      if (i >= n) break;
      if constexpr (XT == QT_F32) u[i] = *(const uint32_t*)(p + 4 * i);
      else u[i >> 1] |= (uint32_t)*(const uint16_t*)(p + 2 * i) << (16 * (i & 1));
    }
    return u;
  }
  static __device__ __forceinline__ void put_part(uint8_t* p, u32x4 u, int n) {
#pragma unroll
    for (int i = 0; i < EPU; ++i) {
      if (i >= n) break;
      if constexpr (XT == QT_F32) *(uint32_t*)(p + 4 * i) = u[i];
      else *(uint16_t*)(p + 2 * i) = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
    }
  }
  // Unit starting at element c of a row of `cols` elements (c < cols).
  static __device__ __forceinline__ u32x4 get(const uint8_t* row, int c, int cols) {
    const uint8_t* p = row + (size_t)c * ES;
    return c + EPU <= cols ? raw(p) : raw_part(p, cols - c);
  }
  // The same for rows that are read once.
  static __device__ __forceinline__ u32x4 get_nt(const uint8_t* row, int c, int cols) {
    const uint8_t* p = row + (size_t)c * ES;
    return c + EPU <= cols ? __builtin_nontemporal_load((const u32x4_a2*)p) : raw_part(p, cols - c);
  }
  static __device__ __forceinline__ void set(uint8_t* row, int c, int cols, u32x4 u) {
    uint8_t* p = row + (size_t)c * ES;
    if (c + EPU <= cols) put(p, u);
    else put_part(p, u, cols - c);
  }
  // Four elements at p (aligned to them).
  static __device__ __forceinline__ void set4(uint8_t* p, const f32x4& v) {
    if constexpr (XT == QT_F32) *(f32x4*)p = v;
    else *(u32x2*)p = u32x2{pair(v[0], v[1]), pair(v[2], v[3])};
  }
  // The first n of four elements to p, which is aligned to one.
  static __device__ __forceinline__ void put4(uint8_t* p, const float (&v)[4], int n) {
    if (n == 4) {
      if constexpr (XT == QT_F32) *(u32x4_a2*)p = u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]),
                                                        __float_as_uint(v[2]), __float_as_uint(v[3])};
      else *(u32x2_a2*)p = u32x2{pair(v[0], v[1]), pair(v[2], v[3])};
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= n) break;
      if constexpr (XT == QT_F32) *(float*)(p + 4 * i) = v[i];
      else *(uint16_t*)(p + 2 * i) = (uint16_t)pair(v[i], 0.f);
    }
  }

 private:
  static __device__ __forceinline__ float one(uint16_t h) {
    if constexpr (XT == QT_F16) return h2f(h);
    else return __uint_as_float((uint32_t)h << 16);
  }
  // v_cvt_pk_bf16_f32 rounds to nearest even, two at a time, and keeps NaN.
  static __device__ __forceinline__ uint32_t pair(float a, float b) {
    if constexpr (XT == QT_F16) return (uint32_t)f2h(a) | ((uint32_t)f2h(b) << 16);
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
  }
};

// Bytes of one element of row type `xtype`, 0 for a type that is none.
inline int row_elem_bytes(int xtype) {
  return xtype == QT_F32 ? 4 : xtype == QT_F16 || xtype == QT_BF16 ? 2 : 0;
}

// Whether rows of `cols` elements (bytes) cannot lie `ld` apart: too close, or as far as only a negative
// number taken for a size is (2^40 is past the end of any memory).
inline bool bad_stride(size_t ld, size_t cols) { return ld < cols || ld > (size_t)1 << 40; }

// f(std::integral_constant<int, XT>) for a row type already checked.
template <class F>
inline void with_rows(int xtype, F f) {
  if (xtype == QT_F32) f(std::integral_constant<int, QT_F32>());
  else if (xtype == QT_F16) f(std::integral_constant<int, QT_F16>());
  else f(std::integral_constant<int, QT_BF16>());
}

}  // namespace tiermm
