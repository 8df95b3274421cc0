// tiles.hpp — what the matrix-core attention kernels over packed rows share:
// the 16-bit operand types, transposed LDS reads, and the order in which
// workgroups take the tiles of sequences of different lengths.
#pragma once
#include <atomic>

#include "packed.hpp"

namespace memopt {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4p_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2p_t __attribute__((ext_vector_type(2)));
typedef float f32x4p_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// 16-bit operand types. Products of two elements are exact in the 32-bit
// accumulators; what is rounded to 16 bits are the probabilities, which enter
// the second product as operands, and the outputs. The row sum adds the
// rounded probabilities, so that the weights of a row sum to one.
struct Fp16 {
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16_t mfma(u32x4p_t a, u32x4p_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return as_u32(half2_t{(half_t)a, (half_t)b}); }
  static __device__ __forceinline__ float dot2(uint32_t w, uint32_t y, float s) {
    return __builtin_amdgcn_fdot2(as_half2(w), as_half2(y), s, false);
  }
  static __device__ __forceinline__ float value(uint16_t x) { return (float)__builtin_bit_cast(half_t, x); }
  static constexpr uint32_t kOnes = 0x3C003C00u;
  static constexpr uint32_t kExponent = 0x7C00u;
  // Where a row's maximum lands, as a power of two: weights reach 2^15 before the next rescale, and those down to 2^-21
  // of the largest are normal numbers.
  static constexpr float kTop = 7.0f;
};
struct Bf16 {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16_t mfma(u32x4p_t a, u32x4p_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, x2{(__bf16)a, (__bf16)b});
  }
  static __device__ __forceinline__ float dot2(uint32_t w, uint32_t y, float s) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(x2, w), __builtin_bit_cast(x2, y), s, false);
  }
  static __device__ __forceinline__ float value(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
  static constexpr uint32_t kOnes = 0x3F803F80u;
  static constexpr uint32_t kExponent = 0x7F80u;
  // The type has 32 bits' range: weights stay under 2^-20, so that 2^20 of them times the largest value do not overflow
  // the 32-bit sums (nor underflow with values down to 2^-98).
  static constexpr float kTop = -28.0f;
};

__device__ __forceinline__ float both_halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Sum of a wave's lanes, wave-uniform (lane exchanges in registers).
__device__ __forceinline__ int32_t wave_sum(int32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);   // quad_perm: lane ^ 1
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);   // quad_perm: lane ^ 2
  v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true);  // row_half_mirror
  v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true);  // row_mirror
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
         __builtin_amdgcn_readlane(v, 48);
}

// The tile (R rows of one sequence) that comes rank-th when the tiles of all
// sequences are ordered by their place in their sequence, last places first:
// under the causal mask those see the most keys, and a grid that ends with its
// longest workgroups leaves the GPU idle behind them. Each lane holds the
// tile counts of up to four sequences; the tiles at place >= x are counted
// with one sum over the wave, x found by bisection. More than 256 sequences
// are taken in order instead. Returns false past the last tile. Over a cache
// only staged sequences have tiles; slot is their rank.
struct Tile {
  int32_t b, t, slot;
};
template <int R, bool PAGED, class Params>
__device__ __forceinline__ bool find_tile(const Params &p, int32_t rank, Tile &out) {
  const int lane = threadIdx.x & 63;
  out = {0, 0, 0};
  auto tiles_of = [&](int32_t b) {
    if (b >= p.B) return 0;
    const int32_t n = rows_of(p.starts, p.T, b).n;
    if constexpr (PAGED)
      if (!is_staged(p.st, n, p.G)) return 0;
    return (n * p.G + R - 1) / R;
  };
  if (p.B == 1) {
    const int32_t n = tiles_of(0);
    out.t = n - 1 - rank;
    return rank < n;
  }
  const uint64_t below = (1ull << lane) - 1;
  if (p.B <= 256) {
    int32_t n[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) n[k] = 64 * k < p.B ? tiles_of(64 * k + lane) : 0;
    auto at_or_past = [&](int32_t x) {
      int32_t s = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) s += max(0, n[k] - x);
      return wave_sum(s);
    };
    if (rank >= at_or_past(0)) return false;
    int32_t lo = 0, hi = (p.T * p.G + R - 1) / R;  // at_or_past(lo) > rank >= at_or_past(hi)
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (at_or_past(mid) > rank) lo = mid;
      else hi = mid;
    }
    int32_t r = rank - at_or_past(hi);  // among the sequences with more than lo tiles
    out.t = lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t m = __ballot(n[k] > lo), staged = PAGED ? __ballot(n[k] > 0) : 0;
      const int32_t c = __popcll(m);
      if (r < c) {
        const int src = __builtin_ctzll(__ballot(n[k] > lo && (int32_t)__popcll(m & below) == r));
        out.b = 64 * k + src;
        out.slot += (int32_t)__popcll(staged & ((1ull << src) - 1));
        return true;
      }
      r -= c;
      out.slot += (int32_t)__popcll(staged);
    }
    return false;
  }
  int32_t before = 0;
  for (int32_t b0 = 0; b0 < p.B; b0 += 64) {
    const int32_t n = tiles_of(b0 + lane);
    const uint64_t staged = PAGED ? __ballot(n > 0) : 0;
    int32_t incl = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int32_t u = __shfl_up(incl, off, 64);
      if (lane >= off) incl += u;
    }
    const int32_t total = __builtin_amdgcn_readlane(incl, 63);
    if (rank < before + total) {
      const int src = __builtin_ctzll(__ballot(rank < before + incl));
      out.b = b0 + src;
      const int32_t count = __builtin_amdgcn_readlane(n, src), end = __builtin_amdgcn_readlane(incl, src);
      out.t = count - 1 - (rank - (before + end - count));
      out.slot += (int32_t)__popcll(staged & ((1ull << src) - 1));
      return true;
    }
    before += total;
    out.slot += (int32_t)__popcll(staged);
  }
  return false;
}

// Four 16-bit elements of one column of V from four LDS rows (the load
// transposes among 16 lanes: lane i gives the address of row i / 4, columns
// 4 (i % 4) .. + 3, and gets column i of the four rows).
__device__ __forceinline__ u32x2p_t v_read(const uint8_t *tile, uint32_t off) {
  typedef __attribute__((address_space(3))) s16x4_t lds_t;
  return __builtin_bit_cast(u32x2p_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t *)(tile + off)));
}

// A pair of elements with inf and NaN replaced by the largest finite value of
// their sign; `odd` collects a nonzero bit wherever that changed one.
template <class E>
__device__ __forceinline__ uint32_t tame(uint32_t w, uint32_t &odd) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  constexpr unsigned short most = (unsigned short)(E::kExponent - 1);
  const u16x2 m = __builtin_elementwise_min(__builtin_bit_cast(u16x2, w & 0x7FFF7FFFu), u16x2{most, most});
  const uint32_t y = (w & 0x80008000u) | __builtin_bit_cast(uint32_t, m);
  odd |= y ^ w;
  return y;
}

// A block-table entry (or another uniform word that no kernel of the launch
// writes) through the scalar cache: a vector load would be waited for together
// with every load and copy before it.
__device__ __forceinline__ int32_t uniform_entry(const int32_t *x) {
  return *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)uniform_ptr(x);
}

// More than 64 KiB of LDS is allowed per kernel and device: once for each.
template <auto Kernel>
static hipError_t allow_lds(int bytes) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (e != hipSuccess || (done.load(std::memory_order_relaxed) & bit)) return e;
  e = hipFuncSetAttribute(reinterpret_cast<const void *>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <int N>
struct IntConst {
  static constexpr int value = N;
};

}  // namespace memopt
