// prompt.hip — causal attention over whole prompts, packed one behind the
// other, straight from the projections' q, k and v (gfx950 matrix cores).
//
// For query row i of a sequence (positions count from its first row) and key
// head h / G of query head h (G = query heads per key head):
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(q_i . k_j / sqrt(D) - m_i),
//   j <= i and (j < sinks or j > i - W)
// which is the causal rule of the paged attention (attention.hpp key_range).
// One pass over the keys with a running maximum m and sum; a later, larger
// maximum scales what was summed before it.
//
// Bound by the matrix instructions and the softmax between them: 4 D flops per
// visible pair and query head. A workgroup takes 128 rows (32 per wave, as
// v_mfma_f32_32x32x16 has columns) against 64-key tiles: that reads K and V
// once per 128 rows, and two workgroups (64 KiB of LDS and 252 registers each)
// fit a CU. The softmax of one tile runs beside the products of the next, in
// one wave, since two waves per SIMD do not cover it by themselves (16384
// tokens, window 4096, 32 query over 8 key heads of 128: 1068 us one behind the
// other, 941 now, 1.02 PFLOP/s; a library product of 8192^3 reaches 1.24).
// Three prompts of up to 9000 tokens, 40 heads: 839 us, 1.03 PFLOP/s. 24 of 20
// to 2500 tokens: 195 us, 0.77: its 3376 workgroups have 11 key tiles each on
// average, and every one pays the search for its tile, its queries and first
// tiles with nothing beside them, and the plain form of its masked tiles (9 % of
// the iterations; the mask itself hides only 5 % of the products).
#include <algorithm>
#include <cmath>

#include "attention.hpp"
#include "lds_dma.hpp"
#include "packed.hpp"

namespace memopt {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4p_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2p_t __attribute__((ext_vector_type(2)));
typedef float f32x4p_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

struct PromptParams {
  const uint16_t *q, *k, *v;  // 16-bit elements; strides in elements
  uint16_t *out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
  const int32_t *starts;
  int32_t T, B, Hk, G, W, sinks;
  Divisor by_g;
  float qk_scale_log2;
  // chunks over a cache: k and v are the staged copies
  const int32_t *ctx;
  int32_t max_tokens;
  Staged st;
};

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
template <int R, bool PAGED>
__device__ __forceinline__ bool find_tile(const PromptParams &p, int32_t rank, Tile &out) {
  const int lane = threadIdx.x & 63;
  out = {0, 0, 0};
  auto tiles_of = [&](int32_t b) {
    if (b >= p.B) return 0;
    const int32_t n = rows_of(p.starts, p.T, b).n;
    if (PAGED && !is_staged(p.st, n, p.G)) return 0;
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

template <int N>
struct IntConst {
  static constexpr int value = N;
};

// `n` instructions of class `mask` here in the schedule (0x002 VALU, 0x008
// MFMA, 0x100 LDS read, 0x400 transcendental).
#define SCHED(mask, n) __builtin_amdgcn_sched_group_barrier(mask, n, 0)

// Where keys and values come from: the packed rows themselves, or for chunks
// over a cache their staged copies, of fp16 values or of codes and factors.
enum Source { kPacked, kStagedRows, kStagedCodes };

template <class E, int D, int NW, Source FROM>
__global__ __launch_bounds__(NW * 64, 2) void prompt_kernel(const PromptParams p) {
  constexpr bool PAGED = FROM != kPacked, CODES = FROM == kStagedCodes;
  constexpr int TK = 64, R = 32 * NW;             // keys per tile, query rows per workgroup
  constexpr int RB = 2 * D, CPR = RB / 16;         // bytes and 16-byte pieces of an LDS row
  constexpr int NCH = D / 16, NDB = D / 32;
  constexpr int RPC = 1024 / RB, NC = TK / RPC / NW;  // rows per copy; copies per wave of K (and of V)
  __shared__ __attribute__((aligned(16))) uint8_t lds_k0[TK * RB], lds_k1[TK * RB], lds_v0[TK * RB],
      lds_v1[TK * RB];
  // Codes: per key of a tile the factors' ratio, then the second factor (Staged::factors).
  constexpr int FB = 2 * TK * 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds_f[CODES ? 2 * FB : 16];

  const int lane = threadIdx.x & 63, n = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroup i runs on XCD i % 8: a key head's workgroups share an XCD and its
  // L2 where the heads deal out evenly.
  const int32_t kvh = (int32_t)(blockIdx.x % p.Hk);
  Tile tile;
  if (!find_tile<R, PAGED>(p, (int32_t)(blockIdx.x / p.Hk), tile)) return;
  const int32_t b = __builtin_amdgcn_readfirstlane(tile.b), slot = __builtin_amdgcn_readfirstlane(tile.slot);
  if (PAGED && slot >= p.st.slots) return;  // sequences overlap
  // The rows of a sequence and a key head: token i's G query heads are rows
  // G i .. G i + G - 1. (So a tile spans few positions, its waves end with the
  // same key tile, and short prompts fill tiles.) Positions: of the sequence,
  // or over a cache the last ones of the context.
  const Rows seq = rows_of(p.starts, p.T, b);
  const int32_t rows = seq.n * p.G, ctx = PAGED ? p.ctx[b] : seq.n, pos0 = ctx - seq.n;
  const int32_t len = PAGED ? min(ctx, p.max_tokens) : seq.n;  // keys
  const int32_t q0 = R * __builtin_amdgcn_readfirstlane(tile.t), qw0 = q0 + 32 * wave;
  auto pos_of = [&](int32_t row) { return pos0 + p.by_g(min(row, rows - 1)); };

  u32x4p_t qf[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) qf[c] = (u32x4p_t){};
  if (qw0 + n < rows) {
    const int32_t tok = p.by_g(qw0 + n);
    const uint16_t *src = p.q + (int64_t)(seq.start + tok) * p.q_ts +
                          ((int64_t)kvh * p.G + qw0 + n - tok * p.G) * p.q_hs + 8 * hl;
#pragma unroll
    for (int c = 0; c < NCH; ++c) qf[c] = *reinterpret_cast<const u32x4p_t *>(src + 16 * c);
  }

  // Tiles of the workgroup: sinks, then the window of its rows.
  const int32_t hi = max(0, min(len, pos_of(q0 + R - 1) + 1));
  const int32_t sink_tiles = (min(p.sinks, hi) + TK - 1) / TK;
  const int32_t t_first = max(max(0, pos_of(q0) - p.W + 1) / TK, sink_tiles), t_last = (hi + TK - 1) / TK;
  const int32_t n_tiles = sink_tiles + max(0, t_last - t_first);
  auto tile_base = [&](int32_t it) { return (it < sink_tiles ? it : t_first + (it - sink_tiles)) * TK; };

  // LDS rows are the 64 keys, their 16-byte pieces XOR-swizzled so that the
  // reads below meet no bank twice: a K operand reads one piece of 32 rows, a
  // V operand 32 dims of four rows at once (transposed by the load).
  auto k_swz = [](int row) { return CPR == 16 ? row & 15 : (row >> 1) & 7; };
  auto v_swz = [](int row) { return CPR == 16 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); };
  const uint32_t k_rb = 2 * (uint32_t)p.k_ts, v_rb = 2 * (uint32_t)p.v_ts;
  uint32_t k_off[NC], v_off[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int row = (wave * NC + c) * RPC + lane / CPR, j = lane % CPR;
    k_off[c] = row * k_rb + 16 * (j ^ k_swz(row)) - c * 1024;
    v_off[c] = row * v_rb + 16 * (j ^ v_swz(row)) - c * 1024;
  }
  const int64_t key_row = PAGED ? (int64_t)slot * p.st.cap : seq.start;
  const uint8_t *k_base = reinterpret_cast<const uint8_t *>(p.k + key_row * p.k_ts + kvh * p.k_hs);
  const uint8_t *v_base = reinterpret_cast<const uint8_t *>(p.v + key_row * p.v_ts + kvh * p.v_hs);
  // Row of a position: staged copies leave out what lies between sinks and window.
  const StagedMap sm = staged_map(len, pos0, p.W, p.sinks);
  auto key_at = [&](int32_t pos) { return PAGED && pos >= sm.sink_end ? pos - sm.skip : pos; };
  const uint32_t wave_lds = (uint32_t)wave * NC * 1024;
  const uint32_t mk[2] = {lds_u32(lds_k0) + wave_lds, lds_u32(lds_k1) + wave_lds};
  const uint32_t mv[2] = {lds_u32(lds_v0) + wave_lds, lds_u32(lds_v1) + wave_lds};
  // A tile's rows through a descriptor of their own: 64-bit bases, and rows
  // past the sequence lie outside its range and read as zeros.
  auto rows_at = [&](const uint8_t *base, uint32_t rb, int32_t key0) __attribute__((always_inline)) {
    const int32_t rows = min(TK, len - key0);
    return __builtin_amdgcn_make_buffer_rsrc((void *)(base + (int64_t)key_at(key0) * rb), (short)0,
                                             (int)((rows - 1) * rb + RB), 0x00020000);
  };
  auto load_k = [&](int32_t it, int buf) __attribute__((always_inline)) {
    lds_dma_range<0, NC>(rows_at(k_base, k_rb, tile_base(it)), mk[buf], k_off, 0);
    if constexpr (CODES) {
      if (wave == buf && lane < FB / 16) {  // (either buffer's by one wave; both lists of a tile in one copy)
        const float *f = p.st.factors + ((int64_t)slot * p.Hk + kvh) * 2 * p.st.cap + key_at(tile_base(it));
        const uint32_t off[1] = {(lane < FB / 32 ? 0u : 4u * p.st.cap - FB / 2) + 16u * lane};
        lds_dma<0, 1>(__builtin_amdgcn_make_buffer_rsrc((void *)f, (short)0, (int)(4 * p.st.cap + FB / 2), 0x00020000),
                      lds_u32(lds_f) + buf * FB, off, 0);
      }
    }
  };
  auto load_v = [&](int32_t it, int buf) __attribute__((always_inline)) {
    lds_dma_range<0, NC>(rows_at(v_base, v_rb, tile_base(it)), mv[buf], v_off, 0);
  };

  uint32_t ka[NCH], va[NDB];
#pragma unroll
  for (int c = 0; c < NCH; ++c) ka[c] = n * RB + 16 * ((2 * c + hl) ^ k_swz(n));
  const int i16 = lane & 15, vrow = 4 * hl + (i16 >> 2);
#pragma unroll
  for (int db = 0; db < NDB; ++db)
    va[db] = vrow * RB + 16 * ((4 * db + 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ v_swz(vrow)) + 8 * (i16 & 1);

  f32x16_t o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = (f32x16_t){};
  // x = qk_scale_log2 s + ncm is the exp2 argument; a new maximum lands at
  // kTop, and the next rescale comes once one passes kTop + 8, so that
  // probabilities lie in (0, 2^15] and fp16 holds those down to 2^-21 of the
  // largest as normal numbers.
  constexpr float kTop = 7.0f;
  float ncm = 0.0f, thr = -INFINITY, lsum = 0.0f, lsum1 = 0.0f;

  // What this wave sees: the sink tiles and window iterations [v0, v1); of
  // those, iterations [f0, f1) hold window tiles that all its rows see whole.
  const bool any = qw0 < rows;
  int32_t v0 = sink_tiles, v1 = sink_tiles, f0 = 0, f1 = 0;
  int32_t first_whole = 0;  // keys from here on are in every row's window, as far as it reaches
  if (any) {
    const int32_t off = sink_tiles - t_first;  // iteration of tile t: t + off
    const int32_t first = pos_of(qw0), last = pos_of(qw0 + 31);
    first_whole = max(0, last - p.W + 1);
    v0 = max(sink_tiles, max(0, first - p.W + 1) / TK + off);
    v1 = max(v0, max(0, min(last, len - 1) + TK) / TK + off);
    f0 = max(sink_tiles, (first_whole + TK - 1) / TK + off);
    f1 = max(f0, max(0, min(first + 1, len)) / TK + off);
  }
  // Over a cache: one byte per 16 tokens, 1 where their page is there. If one
  // in sight is not, every tile is masked.
  const uint32_t *links = nullptr;
  if constexpr (PAGED) {
    links = reinterpret_cast<const uint32_t *>(p.st.links + (int64_t)slot * (p.st.cap / 16));
    bool gap = false;
    for (int32_t it = lane; it < n_tiles; it += 64) gap |= links[key_at(tile_base(it)) / TK] != 0x01010101u;
    if (__any(gap)) f1 = f0;
  }
  auto sees = [&](int32_t it) { return it < sink_tiles ? any : it >= v0 && it < v1; };

  // Register r of block blk holds key tb + 32 blk + 8 (r / 4) + 4 hl + r % 4.
  // (The row is worked out again from the lane: held through the tiles it spills.)
  auto lane_row = [&]() __attribute__((always_inline)) {
    int32_t row = qw0 + (int32_t)(__lane_id() & 31);
    asm volatile("" : "+v"(row));
    return row;
  };
  auto apply_mask = [&](f32x16_t (&s)[2], int32_t tb) __attribute__((always_inline)) {
    const int32_t key0 = tb + 4 * hl, row = lane_row(), qp = pos_of(row);
    const bool q_ok = row < rows;
    const int32_t last = q_ok ? min(qp, len - 1) - key0 : -1;
    const uint32_t link = PAGED ? links[key_at(tb) / TK] : 0x01010101u;
    if (tb >= first_whole) {  // (wave-uniform) no row's window begins behind the tile's first key
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int32_t end = !PAGED || ((link >> (16 * blk + 8 * half)) & 1) ? last : -1;
#pragma unroll
          for (int r = 8 * half; r < 8 * half + 8; ++r)
            s[blk][r] = 32 * blk + 8 * (r >> 2) + (r & 3) <= end ? s[blk][r] : -INFINITY;
        }
      return;
    }
    const int32_t first = qp - p.W + 1 - key0, sink = p.sinks - key0;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int32_t end = !PAGED || ((link >> (16 * blk + 8 * half)) & 1) ? last : -1;
#pragma unroll
        for (int r = 8 * half; r < 8 * half + 8; ++r) {
          const int32_t c = 32 * blk + 8 * (r >> 2) + (r & 3);
          s[blk][r] = (c <= end) & ((c >= first) | (c < sink)) ? s[blk][r] : -INFINITY;
        }
      }
  };
  auto row_max = [&](const f32x16_t (&s)[2]) __attribute__((always_inline)) {
    float t = s[0][0];
#pragma unroll
    for (int r = 1; r < 16; ++r) t = fmaxf(t, s[0][r]);
#pragma unroll
    for (int r = 0; r < 16; ++r) t = fmaxf(t, s[1][r]);
    return both_halves_max(t);
  };
  // Four keys' factors: list 0 or 1 of buffer fb, registers 4 i .. 4 i + 3 of block blk.
  auto factors = [&](int fb, int list, int blk, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const f32x4p_t *>(lds_f + fb * FB + list * (FB / 2) + 4 * (32 * blk + 8 * i + 4 * hl));
  };
  auto to_x = [&](f32x16_t &s, int fb, int blk) __attribute__((always_inline)) {
    if constexpr (CODES) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4p_t f = factors(fb, 1, blk, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * i + j] = fmaf(s[4 * i + j], f[j], ncm);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], p.qk_scale_log2, ncm);
    }
  };
  // Codes of two scale groups (D = 128): the first group's sum is brought to
  // the second's factor before that group is added to it.
  constexpr bool SPLIT = CODES && D == 128;
  auto to_second = [&](f32x16_t &s, int fb, int blk) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4p_t f = factors(fb, 0, blk, i);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[4 * i + j] *= f[j];
    }
  };
  auto raise_max = [&](float t, f32x16_t (&s)[2]) __attribute__((always_inline)) {
    if (__any(t > thr)) {
      const bool start = thr == -INFINITY, found = t > -INFINITY;
      const float shift = start ? (found ? t - kTop : 0.0f) : fmaxf(t - kTop, 0.0f);
      const float alpha = start ? (found ? 0.0f : 1.0f) : (shift > 0.0f ? fast_exp2(-shift) : 1.0f);
      lsum *= alpha;
      lsum1 *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[blk][r] -= shift;
      ncm -= shift;
      thr = (start && !found) ? thr : kTop + 8.0f;
    }
  };
  // Probabilities of one block, which two register quads each make an operand
  // of the second product as they are; their sum, from the rounded pairs.
  auto probs = [&](f32x16_t &s, u32x4p_t (&pb)[2], float &sum) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[2 * i] = fast_exp2(s[2 * i]);
      s[2 * i + 1] = fast_exp2(s[2 * i + 1]);
      pb[i >> 2][i & 3] = E::pack(s[2 * i], s[2 * i + 1]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = E::dot2(pb[i >> 2][i & 3], E::kOnes, sum);
  };
  // Operands: K piece c of a 32-key block; V of 16 keys (half i % 2 of a
  // 32-key block) and dims 32 (i / 2) .. + 31, transposed from four-row reads.
  auto kfrag = [&](const uint8_t *kt, int blk, int c) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4p_t *>(kt + 32 * blk * RB + ka[c]);
  };
  auto vfrag = [&](const uint8_t *vt, int blk, int i) __attribute__((always_inline)) {
    const uint8_t *src = vt + (32 * blk + 16 * (i & 1)) * RB;
    const u32x2p_t a = v_read(src, va[i >> 1]), b8 = v_read(src + 8 * RB, va[i >> 1]);
    return u32x4p_t{a[0], a[1], b8[0], b8[1]};
  };
  auto qk_block = [&](const uint8_t *kt, int blk, f32x16_t &acc, auto prec, const u32x4p_t (&pre)[4])
                      __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      acc = E::mfma((decltype(prec)::value && c < 4) ? pre[c] : kfrag(kt, blk, c), qf[c], c == 0 ? (f32x16_t){} : acc);
  };
  // Half of both blocks' products: scale group G of both.
  auto qk_group = [&](const uint8_t *kt, auto group, f32x16_t (&acc)[2], const u32x4p_t (&pre)[4])
                      __attribute__((always_inline)) {
    constexpr int G = decltype(group)::value;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int blk = i / (NCH / 2), c = G * (NCH / 2) + i % (NCH / 2);
      acc[blk] = E::mfma(G == 1 && i < 4 ? pre[i] : kfrag(kt, blk, c), qf[c], c == 0 ? (f32x16_t){} : acc[blk]);
    }
  };
  auto scores = [&](const uint8_t *kt, int fb, f32x16_t (&s)[2]) __attribute__((always_inline)) {
    u32x4p_t pre[4] = {};
    if constexpr (SPLIT) {
      qk_group(kt, IntConst<0>{}, s, pre);
      to_second(s[0], fb, 0);
      to_second(s[1], fb, 1);
#pragma unroll
      for (int c = 0; c < 4; ++c) pre[c] = kfrag(kt, 0, NCH / 2 + c);
      qk_group(kt, IntConst<1>{}, s, pre);
    } else {
      qk_block(kt, 0, s[0], IntConst<0>{}, pre);
      qk_block(kt, 1, s[1], IntConst<0>{}, pre);
    }
    to_x(s[0], fb, 0);
    to_x(s[1], fb, 1);
  };
  auto pv_block = [&](const uint8_t *vt, int blk, const u32x4p_t (&pb)[2], const u32x4p_t (&pre)[4])
                      __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2 * NDB; ++i)
      o[i >> 1] = E::mfma(i < 4 ? pre[i] : vfrag(vt, blk, i), pb[i & 1], o[i >> 1]);
  };
  // End of an iteration: this wave's copies have arrived and its reads are
  // done; the barrier says so for all waves.
  auto publish = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
  };

  // Iteration `it` of parity P takes the exp2 arguments x(it) in sc and leaves
  // x(it + 1) in sn. K(it + 1) is read from buffer P ^ 1 while K(it + 2) is
  // copied into buffer P; V(it) is read from buffer P while V(it + 1) is
  // copied into buffer P ^ 1.
  // Pipelined form, for tiles seen whole: four segments of matrix
  // instructions, each with vector work of another tile or block beside it,
  // operands read ahead (a segment's first four under the segment before).
  auto iter_full = [&](int32_t it, f32x16_t (&sc)[2], f32x16_t (&sn)[2], auto pc) __attribute__((always_inline)) {
    constexpr int P = decltype(pc)::value;
    const uint8_t *const kt = P ? lds_k0 : lds_k1, *const vt = P ? lds_v1 : lds_v0;
    const u32x4p_t none[4] = {};
    u32x4p_t pre_k[4], pre_a[4], pre_b[4], pa[2], pb[2];
    if (it + 2 < n_tiles) load_k(it + 2, P);
    __builtin_amdgcn_s_setprio(1);
    // QK(it + 1) block 0 (or group 0) | maximum of x(it)
    if constexpr (SPLIT) qk_group(kt, IntConst<0>{}, sn, none);
    else qk_block(kt, 0, sn[0], IntConst<0>{}, none);
    const float t = row_max(sc);
#pragma unroll
    for (int c = 0; c < 4; ++c) pre_k[c] = SPLIT ? kfrag(kt, 0, NCH / 2 + c) : kfrag(kt, 1, c);
    SCHED(0x100, 4);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      SCHED(0x008, 1);
      SCHED(0x100, 1);
      SCHED(0x002, 2);
    }
    __builtin_amdgcn_sched_barrier(0);
    raise_max(t, sc);
    // QK(it + 1) block 1 (or group 1) | probabilities of block 0
    if constexpr (SPLIT) {
      to_second(sn[0], P ^ 1, 0);
      to_second(sn[1], P ^ 1, 1);
      __builtin_amdgcn_sched_barrier(0);
      qk_group(kt, IntConst<1>{}, sn, pre_k);
    } else {
      qk_block(kt, 1, sn[1], IntConst<1>{}, pre_k);
    }
    probs(sc[0], pa, lsum);
#pragma unroll
    for (int i = 0; i < 4; ++i) pre_a[i] = vfrag(vt, 0, i);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      SCHED(0x008, 1);
      if (NCH == 8 && c < 4) SCHED(0x100, 1);
      else SCHED(0x100, 2);
      SCHED(0x002, 16 / NCH);
      SCHED(0x400, 16 / NCH);
    }
    asm volatile("" ::"v"(pa[0]), "v"(pa[1]));  // (keeps the exp2s in this segment)
    __builtin_amdgcn_sched_barrier(0);
    if (it + 1 < n_tiles) load_v(it + 1, P ^ 1);
    // PV(it) block 0 | probabilities of block 1
    pv_block(vt, 0, pa, pre_a);
    probs(sc[1], pb, lsum1);
#pragma unroll
    for (int i = 0; i < 4; ++i) pre_b[i] = vfrag(vt, 1, i);
#pragma unroll
    for (int c = 0; c < 2 * NDB; ++c) {
      SCHED(0x008, 1);
      SCHED(0x100, 2);
      SCHED(0x002, 16 / (2 * NDB));
      SCHED(0x400, 16 / (2 * NDB));
    }
    asm volatile("" ::"v"(pb[0]), "v"(pb[1]));
    __builtin_amdgcn_sched_barrier(0);
    // PV(it) block 1 | x(it + 1)
    pv_block(vt, 1, pb, pre_b);
    to_x(sn[0], P ^ 1, 0);
    to_x(sn[1], P ^ 1, 1);
#pragma unroll
    for (int c = 0; c < 2 * NDB; ++c) {
      SCHED(0x008, 1);
      if (c < 2 * NDB - 4) SCHED(0x100, 2);
      if (CODES) SCHED(0x100, 8 / (2 * NDB));
      SCHED(0x002, 32 / (2 * NDB));
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    publish();
  };
  // Plain form, for tiles that are masked, not seen, or followed by one that
  // is not.
  uint32_t odd = 0;  // nonzero where a masked tile's V held inf or NaN
  auto iter_edge = [&](int32_t it, f32x16_t (&sc)[2], f32x16_t (&sn)[2], auto pc) __attribute__((always_inline)) {
    constexpr int P = decltype(pc)::value;
    const uint8_t *const kt = P ? lds_k0 : lds_k1, *const vt = P ? lds_v1 : lds_v0;
    if (it + 2 < n_tiles) load_k(it + 2, P);
    if (it + 1 < n_tiles) load_v(it + 1, P ^ 1);
    if (sees(it)) {
      const int32_t tb = tile_base(it);
      const bool full = it >= f0 && it < f1;
      if (!full) apply_mask(sc, tb);
      raise_max(row_max(sc), sc);
      u32x4p_t pf[2][2];
      probs(sc[0], pf[0], lsum);
      probs(sc[1], pf[1], lsum1);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        u32x4p_t vf[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) vf[c] = vfrag(vt, c >> 1, 2 * db + (c & 1));
        if (!full) {
          // A weight of 0 must not meet an inf or NaN. Few tiles hold one, and
          // a sum of zero times every element tells with a quarter of the work.
          float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) z[c] = E::dot2(vf[c][i], 0, z[c]);
          if (__any(!((z[0] + z[1]) + (z[2] + z[3]) == 0.0f))) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 4; ++i) vf[c][i] = tame<E>(vf[c][i], odd);
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) o[db] = E::mfma(vf[c], pf[c >> 1][c & 1], o[db]);
      }
    }
    if (it + 1 < n_tiles && sees(it + 1)) {
      scores(kt, P ^ 1, sn);
    } else {
      sn[0] = (f32x16_t){};
      sn[1] = (f32x16_t){};
    }
    publish();
  };

  f32x16_t sx[2], sy[2];
  if (n_tiles > 0) {
    load_k(0, 0);
    load_v(0, 0);
    if (n_tiles > 1) load_k(1, 1);
    publish();
    if (sees(0)) {
      scores(lds_k0, 0, sx);
    } else {
      sx[0] = (f32x16_t){};
      sx[1] = (f32x16_t){};
    }
    __syncthreads();  // K(0)'s buffer is refilled by the first iteration
  }
  // Iterations [m0, m1) are pipelined: this tile seen whole, the next seen (and
  // in the list: where the context passes the block table, a wave's positions
  // can lie behind its last tile). Two iterations per trip keep buffers and score registers constant. (One
  // loop for the plain iterations before and behind, with the buffer as a
  // variable, spilled operand addresses into the pipelined loop: twice as long.)
  const int32_t m0 = min(n_tiles, f0 + (f0 & 1)), m1 = max(m0, min(min(f1, v1 - 1), n_tiles - 1));
  int32_t it = 0;
  for (; it < m0; it += 2) {
    iter_edge(it, sx, sy, IntConst<0>{});
    if (it + 1 >= m0) {
      ++it;
      break;
    }
    iter_edge(it + 1, sy, sx, IntConst<1>{});
  }
  for (; it < m1; it += 2) {
    iter_full(it, sx, sy, IntConst<0>{});
    if (it + 1 >= m1) {
      ++it;
      break;
    }
    iter_full(it + 1, sy, sx, IntConst<1>{});
  }
  if (it < n_tiles && (it & 1)) {
    iter_edge(it, sy, sx, IntConst<1>{});
    ++it;
  }
  for (; it < n_tiles; it += 2) {
    iter_edge(it, sx, sy, IntConst<0>{});
    if (it + 1 >= n_tiles) break;
    iter_edge(it + 1, sy, sx, IntConst<1>{});
  }

  if (__any(odd != 0)) {
    // inf and NaN in V entered the masked tiles as finite values. Rows that do
    // see one have inf or NaN in that column whatever its weight.
    const int32_t qp = pos_of(lane_row());
    const bool q_ok = lane_row() < rows;
#pragma unroll 1
    for (int32_t i = 0; i < n_tiles; ++i) {
      if (!sees(i) || (i >= f0 && i < f1)) continue;
      const int32_t tb = tile_base(i);
#pragma unroll 1
      for (int32_t key = tb; key < min(tb + TK, len); ++key) {
        if (PAGED && p.st.links[(int64_t)slot * (p.st.cap / 16) + key_at(key) / 16] == 0) continue;
        const uint16_t *row = reinterpret_cast<const uint16_t *>(v_base + (int64_t)key_at(key) * v_rb) + 4 * hl;
        const bool see = q_ok && key <= qp && (key < p.sinks || key > qp - p.W);
#pragma unroll
        for (int r = 0; r < 16 * NDB; ++r) {
          const uint16_t bits = row[8 * (r >> 2) + (r & 3)];
          if (see && (bits & E::kExponent) == E::kExponent) o[r >> 4][r & 15] += E::value(bits);
        }
      }
    }
  }

  const float l = xor32_sum(lsum + lsum1);
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  const int32_t row = lane_row();
  if (row >= rows) return;
  const int32_t row_tok = p.by_g(row);
  uint16_t *dst = p.out + (int64_t)(seq.start + row_tok) * p.o_ts + ((int64_t)kvh * p.G + row - row_tok * p.G) * p.o_hs +
                  4 * hl;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<u32x2p_t *>(dst + 32 * db + 8 * g) =
          u32x2p_t{E::pack(o[db][4 * g] * inv, o[db][4 * g + 1] * inv),
                   E::pack(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv)};
}

// Tiles of T tokens in B sequences, at most.
static int64_t most_tiles(int64_t T, int64_t B, int64_t G) { return (T * G + 127 * std::min(B, T)) / 128; }

template <class E, int D>
static void launch_prompt(const PromptParams &p, hipStream_t stream) {
  hipLaunchKernelGGL((prompt_kernel<E, D, 4, kPacked>), dim3((unsigned)(most_tiles(p.T, p.B, p.G) * p.Hk)), dim3(256), 0,
                     stream, p);
}

int launch_paged_tiles(const PagedTiles &d, hipStream_t stream) {
  PromptParams p = {};
  p.q = (const uint16_t *)d.q;
  p.out = (uint16_t *)d.out;
  p.q_ts = d.q_ts;
  p.q_hs = d.q_hs;
  p.o_ts = d.o_ts;
  p.o_hs = d.o_hs;
  p.k = (const uint16_t *)d.st.k;
  p.v = (const uint16_t *)d.st.v;
  p.k_hs = p.v_hs = d.D;
  p.k_ts = p.v_ts = (int64_t)d.Hk * d.D;
  p.starts = d.starts;
  p.ctx = d.ctx;
  p.T = d.T;
  p.B = d.B;
  p.Hk = d.Hk;
  p.G = d.G;
  p.by_g = Divisor::of((uint32_t)d.G);
  p.W = d.W;
  p.sinks = d.sinks;
  p.max_tokens = d.max_tokens;
  p.qk_scale_log2 = d.qk_scale_log2;
  p.st = d.st;
  const dim3 grid((unsigned)(most_tiles(d.T, std::min(d.B, d.st.slots), d.G) * d.Hk));
  if (d.st.factors) {
    if (d.D == 128) hipLaunchKernelGGL((prompt_kernel<Fp16, 128, 4, kStagedCodes>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((prompt_kernel<Fp16, 64, 4, kStagedCodes>), grid, dim3(256), 0, stream, p);
  } else {
    if (d.D == 128) hipLaunchKernelGGL((prompt_kernel<Fp16, 128, 4, kStagedRows>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((prompt_kernel<Fp16, 64, 4, kStagedRows>), grid, dim3(256), 0, stream, p);
  }
  return check_launch("packed_attention(tiles)");
}

}  // namespace memopt

using namespace memopt;

extern "C" int memopt_prompt_attention(const memopt_prompt_desc *desc, void *stream) {
  MEMOPT_REQUIRE(desc, MEMOPT_ERR_INVALID, "prompt_attention: null descriptor");
  const memopt_prompt_desc &d = *desc;
  MEMOPT_REQUIRE(d.dtype == MEMOPT_FP16 || d.dtype == MEMOPT_BF16, MEMOPT_ERR_INVALID,
                 "prompt_attention: dtype must be fp16 or bf16");
  MEMOPT_REQUIRE(d.tokens >= 0 && d.batch >= 0, MEMOPT_ERR_INVALID, "prompt_attention: negative size");
  MEMOPT_REQUIRE(d.num_heads > 0 && d.num_kv_heads > 0 && d.num_heads % d.num_kv_heads == 0, MEMOPT_ERR_INVALID,
                 "prompt_attention: num_heads must be a positive multiple of num_kv_heads");
  MEMOPT_REQUIRE(d.head_dim == 64 || d.head_dim == 128, MEMOPT_ERR_UNSUPPORTED,
                 "prompt_attention: head_dim must be 64 or 128");
  if (d.tokens == 0 || d.batch == 0) return MEMOPT_OK;
  MEMOPT_REQUIRE(d.query && d.key && d.value && d.out && d.query_starts, MEMOPT_ERR_INVALID,
                 "prompt_attention: null pointer");
  auto aligned = [](const void *x, int64_t ts, int64_t hs) {
    return ((uintptr_t)x & 15) == 0 && ts % 8 == 0 && hs % 8 == 0;
  };
  MEMOPT_REQUIRE(aligned(d.query, d.q_token_stride, d.q_head_stride) &&
                     aligned(d.key, d.k_token_stride, d.k_head_stride) &&
                     aligned(d.value, d.v_token_stride, d.v_head_stride) &&
                     aligned(d.out, d.o_token_stride, d.o_head_stride),
                 MEMOPT_ERR_INVALID, "prompt_attention: rows must be 16-byte aligned");
  // (a tile of 64 rows lies in one 31-bit buffer range)
  auto in_range = [&](int64_t ts) { return ts >= d.head_dim && ts < (1LL << 23); };
  MEMOPT_REQUIRE(in_range(d.k_token_stride) && in_range(d.v_token_stride), MEMOPT_ERR_UNSUPPORTED,
                 "prompt_attention: key and value token strides must be head_dim to 2^23 - 1 elements");
  PromptParams p = {};
  p.q = (const uint16_t *)d.query;
  p.k = (const uint16_t *)d.key;
  p.v = (const uint16_t *)d.value;
  p.out = (uint16_t *)d.out;
  p.q_ts = d.q_token_stride;
  p.q_hs = d.q_head_stride;
  p.k_ts = d.k_token_stride;
  p.k_hs = d.k_head_stride;
  p.v_ts = d.v_token_stride;
  p.v_hs = d.v_head_stride;
  p.o_ts = d.o_token_stride;
  p.o_hs = d.o_head_stride;
  p.starts = d.query_starts;
  p.T = d.tokens;
  p.B = d.batch;
  p.Hk = d.num_kv_heads;
  p.G = d.num_heads / d.num_kv_heads;
  p.by_g = Divisor::of((uint32_t)p.G);
  p.W = d.window_size <= 0 ? 1 << 30 : std::min(d.window_size, 1 << 30);  // (position - W stays in 32 bits)
  p.sinks = std::max(0, d.num_sink_tokens);
  p.qk_scale_log2 = 1.4426950408889634f / sqrtf((float)d.head_dim);
  MEMOPT_REQUIRE(d.tokens <= 1 << 30 && (int64_t)d.tokens * d.num_heads <= INT32_MAX - 255 &&
                     most_tiles(d.tokens, d.batch, p.G) * d.num_kv_heads < (1LL << 24),
                 MEMOPT_ERR_UNSUPPORTED, "prompt_attention: too many query rows");  // (a launch holds 2^32 - 1 threads)
  hipStream_t s = (hipStream_t)stream;
  if (d.dtype == MEMOPT_FP16) {
    if (d.head_dim == 128) launch_prompt<Fp16, 128>(p, s);
    else launch_prompt<Fp16, 64>(p, s);
  } else {
    if (d.head_dim == 128) launch_prompt<Bf16, 128>(p, s);
    else launch_prompt<Bf16, 64>(p, s);
  }
  return check_launch("prompt_attention");
}
