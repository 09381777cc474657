// tm_tiles.h -- what the tiled products of int8 and microscaled rows share: the order of tiles, waits for
// stages on their way to LDS, and the way of a tile's rows out through LDS.
#pragma once

#include "tm_device.h"

namespace tiermm {

// Tile `t` of the workgroups' sequence in which XCD x (blockIdx % 8) walks the x-th
// contiguous share, or -1 past the end.
__device__ __forceinline__ int xcd_share(int bid, int total) {
  const int x = bid & 7, i = bid >> 3, each = total >> 3, more = total & 7;
  return i < each + (x < more) ? x * each + min(x, more) + i : -1;
}

// dma16 from a wave-uniform base and each lane's offset of 32 bits, and 4 bytes a lane in the same way.
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base),
               "s"(__builtin_amdgcn_readfirstlane(lds_addr))
               : "memory");
}
__device__ __forceinline__ void dma4(const void* base, uint32_t off, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base),
               "s"(__builtin_amdgcn_readfirstlane(lds_addr))
               : "memory");
}

// Waits until no more than n (at most N) stages of INST loads are on their way.
template <int N, int INST>
__device__ __forceinline__ void wait_stages(int n) {
  if constexpr (N > 0) {
    if (n >= N) vm_wait<N * INST>();
    else wait_stages<N - 1, INST>(n);
  } else {
    vm_wait<0>();
  }
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

}  // namespace tiermm
