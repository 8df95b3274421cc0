// lds_dma.hpp — copies from global memory straight into LDS (gfx950).
#pragma once
#include "common.hpp"

namespace memopt {

// LDS-DMA copy (buffer_load ... lds): lane i's 16 bytes at buffer offset
// voff + soff land at LDS byte m0v + 16 i. Written as inline assembly so the
// compiler does not track it: with the builtin, its wait-count pass cannot
// tell the LDS buffers apart (it waits for the next tiles' copies before
// operand reads of the current one) and the barrier's release fence turns
// the counted wait below into vmcnt(0). Callers wait for completion
// themselves (s_waitcnt vmcnt before the barrier that publishes a tile).
// m0 is an input operand ("{m0}"), so the compiler sets it and knows it is
// read; nothing is clobbered behind its back. The s_nop are the wait states
// that the hardware needs behind a write of the operands: one between an SALU
// write of m0 and an LDS DMA that reads it, five between a vector
// instruction's write of a scalar register (v_readfirstlane, or a spilled one
// that v_readlane brings back) and a buffer instruction that reads it. The
// compiler keeps them for its own instructions, not for those in inline
// assembly, and may bring a register back right before; so they stand here and
// not where a descriptor is made. (Their cost: nothing that shows but in
// latent_kernel, 2 % where each copy had its own and nothing in pairs.)
//
// lds_dma<C0, N> issues copies C0 .. C0 + N - 1 (N = 1 or 2) of one group
// that shares m0 and the scalar offset: copy c carries the immediate offset
// c * 1024, which the hardware adds to both the global and the LDS address
// (measured on MI355X), and the lane offset vo[c] holds the rest of its
// global address minus that immediate. So a group of copies needs one m0
// write and one wait instead of one of each per copy.
template <int C0, int N>
__device__ __forceinline__ void lds_dma(__amdgpu_buffer_rsrc_t r, uint32_t m0v, const uint32_t *vo, uint32_t soff) {
  static_assert(N == 1 || N == 2, "one or two copies per group");
  static_assert((C0 + N) * 1024 <= 4096, "immediate offsets are 12 bits");
  if constexpr (N == 1) {
    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen offset:%4 lds"
                 :
                 : "v"(vo[C0]), "s"(r), "s"(soff), "{m0}"(m0v), "i"(C0 * 1024)
                 : "memory");
  } else {
    asm volatile(
        "s_nop 4\n\tbuffer_load_dwordx4 %0, %2, %3 offen offset:%5 lds\n\t"
        "buffer_load_dwordx4 %1, %2, %3 offen offset:%6 lds"
        :
        : "v"(vo[C0]), "v"(vo[C0 + 1]), "s"(r), "s"(soff), "{m0}"(m0v), "i"(C0 * 1024), "i"(C0 * 1024 + 1024)
        : "memory");
  }
}

// Copies [C0, C1) of a group, two per m0 write.
template <int C0, int C1>
__device__ __forceinline__ void lds_dma_range(__amdgpu_buffer_rsrc_t r, uint32_t m0v, const uint32_t *vo,
                                              uint32_t soff) {
  if constexpr (C1 - C0 == 1) {
    lds_dma<C0, 1>(r, m0v, vo, soff);
  } else if constexpr (C1 - C0 >= 2) {
    lds_dma<C0, 2>(r, m0v, vo, soff);
    lds_dma_range<C0 + 2, C1>(r, m0v, vo, soff);
  }
}

// The descriptor of `range` bytes from a wave-uniform address, in scalar
// registers from here on (left to the compiler, scores.hip's selection of a
// page or none is moved to vector instructions that it cannot encode).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t uniform_rsrc(const void *base, int range) {
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)uniform_ptr((const uint8_t *)base), (short)0,
                                                               __builtin_amdgcn_readfirstlane(range), 0x00020000);
  asm volatile("" : "+s"(r));
  return r;
}

// LDS byte address of a __shared__ object, wave-uniform.
__device__ __forceinline__ uint32_t lds_u32(const void *p) {
  return __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}

}  // namespace memopt
