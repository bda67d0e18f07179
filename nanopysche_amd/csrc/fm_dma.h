// Loads from memory straight into LDS, their descriptors, and the waits and barrier
// that order them.
#pragma once

#include "fm_common.h"

namespace fm {

typedef int v4i __attribute__((ext_vector_type(4)));

// LDS-DMA: the 64 lanes' loads land at consecutive LDS addresses starting at
// `lds` (wave-uniform).  Issued from inline assembly so the compiler's wait
// insertion does not treat them as pending LDS writes (it would wait for every
// prefetch in flight before each LDS read); the kernels order them with explicit
// vmcnt waits instead.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return uint32_t(size_t((__attribute__((address_space(3))) const void*)(p)));
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is written here and nowhere else
// A raw-buffer descriptor of a wave-uniform base (the wave's first row of the
// tile), a 32-bit per-lane offset and a 32-bit uniform offset (group + K
// position), so no 64-bit address arithmetic is spent per load.  Measured on
// gfx950 it moves the tile's 64 KiB per K step at the same rate as the flat form.
// byte address = base + voff + soff.
__device__ __forceinline__ void bdma16(v4i rsrc, uint32_t voff, uint32_t soff, uint32_t lds) {
  const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %3\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff),
               "s"(m)
               : "memory", "m0");
}
__device__ __forceinline__ void bdma4(v4i rsrc, uint32_t voff, uint32_t soff, uint32_t lds) {
  const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %3\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff),
               "s"(m)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// Raw-buffer descriptor (stride 0, no range clipping) of a wave-uniform base.
__device__ __forceinline__ v4i make_rsrc(const void* base) {
  const uint64_t a = uint64_t(size_t(base));
  v4i r;
  r[0] = __builtin_amdgcn_readfirstlane(int(uint32_t(a)));
  r[1] = __builtin_amdgcn_readfirstlane(int(uint32_t(a >> 32) & 0xffffu));
  r[2] = -1;
  r[3] = 0x00020000;   // gfx9 raw buffer: 32-bit data format, no swizzle
  return r;
}

// s_waitcnt vmcnt(n) lgkmcnt(0) (gfx9 encoding: vmcnt bits [3:0] and [15:14],
// expcnt [6:4] left at its maximum, lgkmcnt [11:8]).  Draining lgkmcnt too
// means this wave's LDS reads of a stage have returned before the barrier that
// allows the stage to be refilled.
#define FM_WAIT_VMCNT(n) __builtin_amdgcn_s_waitcnt(((n) & 0xF) | (((n) >> 4) << 14) | (0x7 << 4))

// A barrier the compiler moves nothing across.  It carries no memory fence,
// which would wait for the prefetches still in flight.
__device__ __forceinline__ void block_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// The lane id read from the hardware (v_mbcnt) at each use.  Volatile, so the
// compiler neither hoists nor shares it: values derived from the lane between
// tiles are rebuilt from it instead of being kept live across the K loops,
// where the register budget is spent (a spilled value's reload waits for
// every load in flight, the operand prefetch included).
__device__ __forceinline__ int fresh_lane() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}

}  // namespace fm
