// packed.hpp — what the kernels over packed batches share: the division that
// turns rows into tokens, and the staged form of long query chunks.
#pragma once
#include "attention.hpp"

namespace memopt {

// x / d for 0 <= x < 2^31 by a product: with 2^l >= d and m = floor(2^(31 + l)
// / d) + 1, floor(m x / 2^(31 + l)) = floor(x / d) (the classic round-up
// multiplier; a division takes some 25 vector instructions, and a workgroup
// that takes ten steps per wave felt them).
struct Divisor {
  uint32_t d, mul, shift;
  static Divisor of(uint32_t d) {
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    return {d, d > 1 ? (uint32_t)((1ull << (31 + l)) / d + 1) : 0, l > 0 ? l - 1 : 0};
  }
  __device__ __forceinline__ int32_t operator()(int32_t x) const {
    return d == 1 ? x : (int32_t)(__umulhi((uint32_t)x, mul) >> shift);
  }
};

// Inclusive prefix sum over the wave (DPP row shifts, then row broadcasts),
// saturating: neither query starts that do not ascend nor counts that a user
// asks for can wrap it.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t scan_step(uint32_t v) {
  return __builtin_elementwise_add_sat(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, ROWS == 0xF));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = scan_step<0x111, 0xF>(v);
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);
  return scan_step<0x143, 0xC>(v);
}

// Rows of sequence b: G query heads per key head make each token G rows.
struct Rows {
  int32_t start, n;  // first token row, tokens
};
__device__ __forceinline__ Rows rows_of(const int32_t *starts, int32_t T, int32_t b) {
  Rows r;
  r.start = min(max(starts[b], 0), T);
  r.n = min(max(starts[b + 1], r.start), T) - r.start;
  return r;
}

// Sequences whose chunk is long enough to attend from a staged copy of the
// keys and values they can see (prompt.hip), instead of from the cache: their
// K and V as fp16 [slot][cap tokens][Hk][D], slot = the sequence's rank among
// them. Tokens [0, sinks) and the window lie one behind the other, each from a
// multiple of 64; links has one byte per 16 tokens, 1 where their page is there.
// From INT4 pages, K are the codes less 8, which fp16 holds exactly; factors
// [slot][Hk][2][cap] make scores of their sums: the scale of a key's first
// group over that of its last (D = 64 has one group: not used), and the last
// one's scale times qk_scale_log2. (Rounding K to fp16 instead was the largest
// error of the operator, 6.7e-4 of the output's norm; 3.0e-4 is left.)
struct Staged {
  int32_t min_rows, max_query;  // rows from which a sequence is staged; queries a slot has room for
  int32_t slots, cap;           // sequences, tokens per slot (a multiple of 64)
  half_t *k, *v;
  uint8_t *links;
  float *factors;  // null: K holds values
};
__device__ __forceinline__ bool is_staged(const Staged &s, int32_t n, int32_t G) {
  return s.slots > 0 && (int64_t)n * G >= s.min_rows && n <= s.max_query;
}
// First position of the window of a sequence's chunk that is staged, the
// sinks' end, and what a window position loses on its way to its staged row.
struct StagedMap {
  int32_t sink_end, lo, skip;
};
__device__ __forceinline__ StagedMap staged_map(int32_t kv_lim, int32_t pos0, int32_t W, int32_t sinks) {
  StagedMap m;
  m.sink_end = (min(sinks, max(kv_lim, 0)) + 63) / 64 * 64;
  m.lo = max(0, pos0 - W + 1) / 64 * 64;
  m.skip = max(0, m.lo - m.sink_end);
  return m;
}

struct PagedTiles {
  const half_t *q;
  half_t *out;
  int64_t q_ts, q_hs, o_ts, o_hs;
  const int32_t *starts, *ctx;
  int32_t T, B, Hk, G, D, max_tokens, W, sinks;
  float qk_scale_log2;
  Staged st;
};
// Attention of the staged sequences' rows (prompt.hip).
int launch_paged_tiles(const PagedTiles &p, hipStream_t stream);

}  // namespace memopt
