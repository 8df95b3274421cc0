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
// read; nothing is clobbered behind its back. The s_nop is the one wait
// state the hardware needs between an SALU write of m0 and an LDS DMA that
// reads it.
//
// lds_dma<C0, N> issues copies C0 .. C0 + N - 1 (N = 1 or 2) of one group
// that shares m0 and the scalar offset: copy c carries the immediate offset
// c * 1024, which the hardware adds to both the global and the LDS address
// (measured on MI355X), and the lane offset vo[c] holds the rest of its
// global address minus that immediate. So a group of copies needs one m0
// write and one wait state instead of one of each per copy.
template <int C0, int N>
__device__ __forceinline__ void lds_dma(__amdgpu_buffer_rsrc_t r, uint32_t m0v, const uint32_t *vo, uint32_t soff) {
  static_assert(N == 1 || N == 2, "one or two copies per group");
  static_assert((C0 + N) * 1024 <= 4096, "immediate offsets are 12 bits");
  if constexpr (N == 1) {
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen offset:%4 lds"
                 :
                 : "v"(vo[C0]), "s"(r), "s"(soff), "{m0}"(m0v), "i"(C0 * 1024)
                 : "memory");
  } else {
    asm volatile(
        "s_nop 0\n\tbuffer_load_dwordx4 %0, %2, %3 offen offset:%5 lds\n\t"
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

// LDS byte address of a __shared__ object, wave-uniform.
__device__ __forceinline__ uint32_t lds_u32(const void *p) {
  return __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}

}  // namespace memopt
