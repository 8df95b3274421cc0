// scores.hip — attention weights added up per cached token, the scores that
// eviction goes by (gfx950 matrix cores).
//
// For sequence b, key head h and token j, over the sequence's query rows r and
// the G query heads g of the group:
//   out[b,h,j] = scores[b,h,j] + sum_{r,g} exp(q_rg . k_hj / sqrt(D) - lse_rg),
//   lse_rg = log sum_{j' visible} exp(q_rg . k_hj' / sqrt(D))
// with the masks of packed_attention. A weight needs its row's sum over all
// keys, so there are two passes with a sum between. In both, keys stay in
// registers (a wave's 64 as matrix operands, unpacked once) and query rows
// stream past, so that a key's total is one lane's sum, in a fixed order, and
// needs no atomics.
//
// INT4 keys enter the products as exact codes (code - 8, which fp16 holds) and
// the sums of each 64-dim group are scaled in 32 bits: nothing is rounded to
// fewer bits on the way from the cache to the result.
#include <algorithm>
#include <cmath>

#include "lds_dma.hpp"
#include "page_format.hpp"
#include "tiles.hpp"

namespace memopt {

typedef _Float16 f16x8s_t __attribute__((ext_vector_type(8)));

struct ScoresParams {
  const uint16_t *q;
  int64_t q_ts, q_hs;
  const uint8_t *k;
  int64_t k_ps, k_hs, k_ts;  // bytes: page, head, token (fp16)
  const int32_t *bt, *ctx, *starts;
  int64_t nb;
  const float *scores;  // null: zeros
  float *out;
  int32_t T, B, Hk, G, M, bs, W, sinks, L;
  int32_t max_keys, max_rows;  // tokens that are looked at; rows of a sequence and key head
  int32_t kts;                 // key tiles of kTileKeys
  Divisor by_g, by_chunks;     // by_chunks: 16-token chunks of a page
  float qk_scale_log2;
  float2 *ml;    // few rows: [B][Hk][kts][4][max_rows]; chunks: [Hk][kts][T G]
  float *probs;  // few rows: [B][Hk][max_rows][kts * kTileKeys]
  float *lse;    // chunks: [Hk][T G]
  int32_t parts;  // chunks: workgroups that share a key tile's rows
  float *sums;    // chunks, parts > 1: [parts][B][Hk][kts * kTileKeys]
};

static constexpr int kTileKeys = 256;  // keys of a workgroup: 64 per wave
static constexpr int kFewRows = 16;  // (the columns of one product)

// A sequence as one key head sees it.
struct ScoredSeq {
  int32_t start, rows, pos0, len;  // first token row; rows; position of the first; keys
};
__device__ __forceinline__ ScoredSeq scored_seq(const ScoresParams &p, int32_t b) {
  const Rows r = rows_of(p.starts, p.T, b);
  const int32_t ctx = p.ctx[b];
  return {r.start, min(r.n, p.max_rows / p.G) * p.G, ctx - r.n, max(0, min(ctx, p.max_keys))};
}
// Whether a query at position pos can see a key of [k0, k1).
__device__ __forceinline__ bool meets(const ScoresParams &p, int32_t pos, int32_t k0, int32_t k1) {
  return k0 <= pos && (k0 < p.sinks || k1 > pos - p.W + 1);
}
// Token range [lo, hi) of the sequence's queries that can see a key of [k0, k1).
__device__ __forceinline__ void queries_of(const ScoresParams &p, const ScoredSeq &s, int32_t n, int32_t k0, int32_t k1,
                                           int32_t &lo, int32_t &hi) {
  lo = min(max(k0 - s.pos0, 0), n);
  hi = k0 < p.sinks ? n : (int32_t)min(max((int64_t)k1 + p.W - 1 - s.pos0, (int64_t)0), (int64_t)n);
  if (k0 >= s.len) hi = lo;
}

__device__ __forceinline__ float max_over_quarters(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return both_halves_max(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
}
__device__ __forceinline__ float sum_over_quarters(float v) { return xor32_sum(xor16_sum(v)); }

// Eight codes less 8 as exact fp16 values, in the order 0 4 1 5 2 6 3 7 of
// their dims: a nibble beside the exponent of 1024 (or 64) is that plus the
// code. (In the dims' own order an operand takes half as many instructions
// again, and unpacking is what bounds single tokens over INT4 pages.)
__device__ __forceinline__ u32x4p_t codes_to_half(uint32_t w) {
  const half2_t lo = {(half_t)1032.0f, (half_t)1032.0f}, hi = {(half_t)72.0f, (half_t)72.0f};
  const uint32_t v = w >> 8;
  return u32x4p_t{as_u32(as_half2(bfi(0x000F000Fu, w, 0x64006400u)) - lo),
                  as_u32(as_half2(bfi(0x00F000F0u, w, 0x54005400u)) - hi),
                  as_u32(as_half2(bfi(0x000F000Fu, v, 0x64006400u)) - lo),
                  as_u32(as_half2(bfi(0x00F000F0u, v, 0x54005400u)) - hi)};
}
// Eight elements of a query row in that order.
__device__ __forceinline__ u32x4p_t in_code_order(u32x4p_t q) {
  return u32x4p_t{__builtin_amdgcn_perm(q[2], q[0], 0x05040100u), __builtin_amdgcn_perm(q[2], q[0], 0x07060302u),
                  __builtin_amdgcn_perm(q[3], q[1], 0x05040100u), __builtin_amdgcn_perm(q[3], q[1], 0x07060302u)};
}

// 64 keys of one head as operands of v_mfma_f32_16x16x32: page g's keys are
// the rows of four (two) operands; lane l holds key l % 16 and of every 64
// dims the 16 from 16 (l / 16) on, in two operands. Products come out with the
// query row in the lane's column l % 16 and keys 4 (l / 16) + r in register r.
template <int FMT, int D>
struct Keys {
  static constexpr int NCH = D / 32, NG = D / 64;
  static constexpr bool CODES = FMT == MEMOPT_KV_INT4;
  uint32_t linked;  // bit g: page g is there
  uint32_t w[CODES ? 4 : 1][NCH];
  uint4 sc[CODES ? 4 : 1][NG];
  u32x4p_t rows[CODES ? 1 : 4][NCH];

  // Block-table entries of the pages of 64 keys, -1 past the end.
  static __device__ __forceinline__ int4 entries(const ScoresParams &p, int32_t b, int32_t key0, int32_t len) {
    int32_t e[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int32_t key = key0 + 16 * g, c = key >> 4;
      e[g] = key < len ? uniform_entry(p.bt + (int64_t)b * p.M + (CODES ? c : p.by_chunks(c))) : -1;
    }
    return int4{e[0], e[1], e[2], e[3]};
  }
  __device__ __forceinline__ void load(const ScoresParams &p, const int4 &pages, int32_t h, int32_t key0) {
    const int lane = threadIdx.x & 63, t = lane & 15, kq = lane >> 4;
    constexpr int BPL = D / 8;
    linked = 0;
    const uint8_t *at[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int32_t c = (key0 >> 4) + g, first = CODES ? 0 : 16 * (c - p.by_chunks(c) * (int32_t)p.by_chunks.d);
      const int32_t page = g == 0 ? pages.x : g == 1 ? pages.y : g == 2 ? pages.z : pages.w;
      const bool ok = page >= 0 && page < p.nb;
      linked |= (ok ? 1u : 0u) << g;
      at[g] = ok ? p.k + (int64_t)page * p.k_ps + h * p.k_hs + first * p.k_ts : nullptr;
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (!((linked >> g) & 1)) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          if constexpr (CODES) w[g][c] = 0x88888888u;
          else rows[g][c] = (u32x4p_t){};
        }
        if constexpr (CODES)
#pragma unroll
          for (int i = 0; i < NG; ++i) sc[g][i] = uint4{0, 0, 0, 0};
      } else if constexpr (CODES) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          if constexpr (D == 128) {
            const uint2 x = *reinterpret_cast<const uint2 *>(at[g] + (8 * (t & 7) + 4 * i + kq) * BPL + (t >> 3) * 8);
            w[g][2 * i] = x.x;
            w[g][2 * i + 1] = x.y;
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              w[g][j] = *reinterpret_cast<const uint32_t *>(at[g] + (8 * (t & 7) + 2 * kq + j) * BPL + (t >> 3) * 4);
          }
          sc[g][i] = *reinterpret_cast<const uint4 *>(at[g] + 16 * D + 32 * i + 16 * (kq & 1));
        }
      } else {
#pragma unroll
        for (int c = 0; c < NCH; ++c)
          rows[g][c] = *reinterpret_cast<const u32x4p_t *>(at[g] + t * p.k_ts + 2 * (64 * (c >> 1) + 16 * kq + 8 * (c & 1)));
      }
    }
  }
  // The same for codes by way of LDS, a tile ahead: fetch() starts copies of the four pages' codes into the wave's 4 KiB
  // at `to` and a read of their scales, take() waits for them, page() brings page g's. A copy's lanes lie side by side;
  // lanes that read the operand layout from memory, 128 bytes apart, take 64 accesses of the cache where a copy
  // takes 16, which bounded the kernel (32 sequences of up to 8192 tokens: 17.3 M accesses and 42 us, now 4.4 M and
  // 33). (16-byte pieces are swizzled by the token.)
  uint32_t scales;  // lane 16 g + i: word i of page g's
  __device__ __forceinline__ void fetch(const ScoresParams &p, const int4 &pages, int32_t h, const uint8_t *to) {
    const int lane = threadIdx.x & 63;
    constexpr int PPT = D / 16;  // pieces of a token pair
    const int row = lane / PPT;
    const uint32_t off[1] = {(uint32_t)(16 * (PPT * row + ((lane % PPT) ^ (row % PPT))))};
    linked = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int32_t page = g == 0 ? pages.x : g == 1 ? pages.y : g == 2 ? pages.z : pages.w;
      const bool ok = page >= 0 && page < p.nb;
      linked |= (ok ? 1u : 0u) << g;
      lds_dma<0, 1>(uniform_rsrc(p.k + (int64_t)(ok ? page : 0) * p.k_ps + h * p.k_hs, ok ? 8 * D : 0),
                    lds_u32(to) + 1024 * g, off, 0);
    }
    const int32_t mine = lane < 32 ? (lane < 16 ? pages.x : pages.y) : (lane < 48 ? pages.z : pages.w);
    scales = *reinterpret_cast<const uint32_t *>(p.k + (int64_t)(mine >= 0 && mine < p.nb ? mine : 0) * p.k_ps + h * p.k_hs +
                                                 16 * D + 4 * (lane % (8 * NG)));
  }
  __device__ __forceinline__ void take(uint32_t *s_scales) {
    asm volatile("s_waitcnt vmcnt(0)" : "+v"(scales) : : "memory");
    s_scales[threadIdx.x & 63] = scales;
  }
  __device__ __forceinline__ void page(int g, const uint8_t *from, const uint32_t *s_scales) {
    const int lane = threadIdx.x & 63, t = lane & 15, kq = lane >> 4;
    const uint8_t *at = from + 1024 * g + (D == 128 ? 8 : 4) * (t >> 3);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      if constexpr (D == 128) {
        const uint2 x = *reinterpret_cast<const uint2 *>(at + 16 * (8 * (t & 7) + ((4 * i + kq) ^ (t & 7))));
        w[g][2 * i] = x.x;
        w[g][2 * i + 1] = x.y;
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          w[g][j] = *reinterpret_cast<const uint32_t *>(at + 16 * (4 * (t & 7) + (kq ^ (t & 3))) + 8 * j);
      }
      sc[g][i] = *reinterpret_cast<const uint4 *>(s_scales + 16 * g + 8 * i + 4 * (kq & 1));
    }
  }
  // Page g's operands, and the factors of the register's keys.
  __device__ __forceinline__ void operands(int g, u32x4p_t (&a)[NCH], f32x4p_t (&f)[NG]) const {
    const int kq = (threadIdx.x & 63) >> 4, sh = 16 * (kq >> 1);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if constexpr (CODES) a[c] = codes_to_half(w[g][c]);
      else a[c] = rows[g][c];
    }
    if constexpr (CODES) {
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const uint32_t s[4] = {sc[g][i].x, sc[g][i].y, sc[g][i].z, sc[g][i].w};
#pragma unroll
        for (int r = 0; r < 4; ++r) f[i][r] = (float)__builtin_bit_cast(half_t, (uint16_t)(s[r] >> sh));
      }
    }
  }
  // q . k of a page's keys against 16 query rows (INT4: q in_code_order).
  static __device__ __forceinline__ f32x4p_t scores(const u32x4p_t (&a)[NCH], const f32x4p_t (&f)[NG], const u32x4p_t (&q)[NCH]) {
    f32x4p_t c[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      if (CODES || i == 0) c[i] = (f32x4p_t){};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f32x4p_t &acc = c[CODES ? i : 0];
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8s_t, a[2 * i + j]),
                                                     __builtin_bit_cast(f16x8s_t, q[2 * i + j]), acc, 0, 0, 0);
      }
    }
    if constexpr (!CODES) return c[0];
    f32x4p_t x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = NG == 1 ? c[0][r] * f[0][r] : fmaf(c[NG - 1][r], f[NG - 1][r], c[0][r] * f[0][r]);
    return x;
  }
};

// Hides what a row at position `pos` does not see of page g's keys (key: the
// lane's first); ok: the row exists.
__device__ __forceinline__ f32x4p_t hide(const ScoresParams &p, f32x4p_t x, int32_t key, int32_t pos, int32_t len, bool ok) {
  const int32_t last = ok ? min(pos, len - 1) : -1;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int32_t j = key + r;
    x[r] = (j <= last) & ((j > pos - p.W) | (j < p.sinks)) ? x[r] : -INFINITY;
  }
  return x;
}

// ---------------------------------------------------------------------------
// Few rows (decode): up to kFewRows rows per sequence and key head
// ---------------------------------------------------------------------------
// The weights relative to a wave's maximum are kept (8 bytes written and read
// per row and key) instead of meeting the keys again in the form for chunks,
// whose tiles have 32 rows. In us, here / there, 32 sequences of up to 8192
// tokens, 8 key heads of 128: INT4 1 row 46 / 207, 4: 49 / 208, 8: 55 / 208,
// 16: 72 / 203; fp16 101 / 203, 110 / 205, 117 / 205, 137 / 204; 2 key heads of
// 64, 16 rows: 25 / 43 and 28 / 44. One sequence of 1024: 16 / 19. The form is the
// call's, by its longest query: the lengths are on the device.
// Bound by vector instructions (unpacking, scales and weights: 0.62 of the
// units' time) and by the chain table, keys, weights of each tile: 32
// sequences of up to 8192 tokens, 8 key heads of 4 rows, 128: 33 us of which
// the bytes take 16, and 13 for the second launch.

template <int FMT, int D>
__global__ __launch_bounds__(256, 4) void few_rows_kernel(const ScoresParams p, const int32_t tiles_each) {
  using K = Keys<FMT, D>;
  const int32_t h = (int32_t)(blockIdx.x % p.Hk), b = blockIdx.y;
  const int lane = threadIdx.x & 63, n = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ScoredSeq s = scored_seq(p, b);
  const int32_t kt0 = (int32_t)(blockIdx.x / p.Hk) * tiles_each;
  const int32_t kt1 = min(min(kt0 + tiles_each, p.kts), (s.len + kTileKeys - 1) / kTileKeys);
  if (s.rows == 0 || kt0 >= kt1) return;
  const bool ok = n < s.rows;
  const int32_t tok = p.by_g(min(n, s.rows - 1)), pos = s.pos0 + tok, last = s.pos0 + s.rows / p.G - 1;
  u32x4p_t q[K::NCH];
  const uint16_t *src = p.q + (int64_t)(s.start + tok) * p.q_ts + ((int64_t)h * p.G + min(n, s.rows - 1) - tok * p.G) * p.q_hs;
#pragma unroll
  for (int c = 0; c < K::NCH; ++c) {
    q[c] = *reinterpret_cast<const u32x4p_t *>(src + 64 * (c >> 1) + 16 * kq + 8 * (c & 1));
    if constexpr (K::CODES) q[c] = in_code_order(q[c]);
  }
  const int64_t unit = (int64_t)b * p.Hk + h;
  auto met = [&](int32_t kt) {
    int32_t lo, hi;
    queries_of(p, s, s.rows / p.G, kt * kTileKeys, (kt + 1) * kTileKeys, lo, hi);
    return kt < kt1 && hi > lo;
  };
  auto entries_at = [&](int32_t kt) { return K::entries(p, b, kt * kTileKeys + 64 * wave, met(kt) ? s.len : 0); };
  __shared__ __attribute__((aligned(16))) uint8_t s_codes[K::CODES ? 4 : 1][2][K::CODES ? 4096 : 1];
  __shared__ __attribute__((aligned(16))) uint32_t s_scales[4][64];
  K keys;
  int4 pages = entries_at(kt0);
  if constexpr (K::CODES) {
    keys.fetch(p, pages, h, s_codes[wave][0]);
    pages = entries_at(kt0 + 1);
  }
  for (int32_t kt = kt0; kt < kt1; ++kt) {
    const int32_t key0 = kt * kTileKeys + 64 * wave, buf = (kt - kt0) & 1;
    uint32_t linked;
    if constexpr (K::CODES) {
      keys.take(s_scales[wave]);
      linked = keys.linked;
      if (kt + 1 < kt1) keys.fetch(p, pages, h, s_codes[wave][buf ^ 1]);
      pages = entries_at(kt + 2);
      if (!met(kt)) continue;
    } else {
      const int4 here = pages;
      pages = entries_at(kt + 1);
      if (!met(kt)) continue;
      keys.load(p, here, h, key0);
      linked = keys.linked;
    }
    // (rows past the last are not stored: what their lanes hold does not matter)
    const bool full = key0 + 63 <= s.pos0 && key0 + 64 <= s.len && linked == 15u &&
                      (key0 > last - p.W || key0 + 64 <= p.sinks);
    f32x4p_t x[4];
    float m = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u32x4p_t a[K::NCH];
      f32x4p_t f[K::NG];
      if constexpr (K::CODES) keys.page(g, s_codes[wave][buf], s_scales[wave]);
      keys.operands(g, a, f);
      x[g] = K::scores(a, f, q);
      if (!full) x[g] = hide(p, x[g], key0 + 16 * g + 4 * kq, pos, s.len, (linked >> g) & 1);
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, x[g][r]);
    }
    // Weights are relative to the maximum of the wave's 64 keys: no wave waits for another.
    m = max_over_quarters(m) * p.qk_scale_log2;
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    float *dst = p.probs + (unit * p.max_rows + n) * ((int64_t)p.kts * kTileKeys) + key0 + 4 * kq;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[g][r] = fast_exp2(fmaf(x[g][r], p.qk_scale_log2, -ref));
        l += x[g][r];
      }
      if (ok) *reinterpret_cast<f32x4p_t *>(dst + 16 * g) = x[g];
    }
    l = sum_over_quarters(l);
    // (keys without a maximum add nothing, unless all that the row sees of them is NaN)
    if (ok && kq == 0) p.ml[((unit * p.kts + kt) * 4 + wave) * p.max_rows + n] = float2{l == 0.0f ? m : fmaxf(m, -3e38f), l};
  }
}

// out = scores + the rows' weights: four keys a thread. Also the whole of a
// call without rows.
static constexpr int kFinishTiles = 4;
__global__ __launch_bounds__(256) void finish_kernel(const ScoresParams p) {
  __shared__ float s_f[kFewRows][4 * kFinishTiles];  // [row][64 keys]
  const int32_t h = (int32_t)(blockIdx.x % p.Hk), kt0 = (int32_t)(blockIdx.x / p.Hk) * kFinishTiles, b = blockIdx.y;
  const ScoredSeq s = scored_seq(p, b);
  const int64_t unit = (int64_t)b * p.Hk + h;
  const int32_t key0 = kt0 * kTileKeys;
  float before[kFinishTiles], w[kFinishTiles];
#pragma unroll
  for (int k = 0; k < kFinishTiles; ++k) {
    const int32_t j = key0 + kTileKeys * k + (int32_t)threadIdx.x;
    before[k] = p.scores && j < p.L ? p.scores[unit * p.L + j] : 0.0f;
    w[k] = 0.0f;
  }
  if (s.rows > 0 && key0 < s.len) {
    const int32_t tiles = (s.len + kTileKeys - 1) / kTileKeys;
    auto met = [&](int32_t t) {
      int32_t lo, hi;
      queries_of(p, s, s.rows / p.G, t * kTileKeys, (t + 1) * kTileKeys, lo, hi);
      return hi > lo;
    };
    // Weights of four rows at a time, all reads under way together, the first four while the sums are put together
    // (tiles that no row met hold anything: their values are not used).
    const float *src = p.probs + unit * p.max_rows * ((int64_t)p.kts * kTileKeys) + threadIdx.x;
    float x[kFinishTiles][4];
    auto read = [&](int32_t r0) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < kFinishTiles; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          x[k][r] = src[(int64_t)min(r0 + r, s.rows - 1) * p.kts * kTileKeys + kTileKeys * min(kt0 + k, tiles - 1)];
    };
    read(0);
    // Row threadIdx / 16's maximum and sum, by 16 lanes over the 64-key parts.
    const int32_t row = threadIdx.x >> 4, lane16 = threadIdx.x & 15;
    const float2 *ml = p.ml + unit * p.kts * 4 * p.max_rows + row;
    float m = -INFINITY, l = 0.0f;
    if (row < s.rows)
      for (int32_t t0 = lane16; t0 < 4 * tiles; t0 += 16 * 8) {
        float2 x[8];  // (eight reads in flight)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ml[(int64_t)min(t0 + 16 * i, 4 * tiles - 1) * p.max_rows];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int32_t t = t0 + 16 * i;
          const float top = fmaxf(m, x[i].x);
          if (t >= 4 * tiles || !met(t >> 2) || top == -INFINITY) continue;
          l = l * fast_exp2(m - top) + x[i].y * fast_exp2(x[i].x - top);
          m = top;
        }
      }
    float top = fmaxf(m, xor1(m));
    top = fmaxf(top, xor2(top));
    top = fmaxf(top, half_mirror(top));
    top = fmaxf(top, dpp_f32<0x140>(top));
    l = m == -INFINITY ? 0.0f : l * fast_exp2(m - top);
    l += xor1(l);
    l += xor2(l);
    l += half_mirror(l);
    l += dpp_f32<0x140>(l);
    if (row < s.rows) {
      const int32_t t = 4 * kt0 + lane16;
      const float here = t < 4 * tiles && met(t >> 2) ? ml[(int64_t)t * p.max_rows].x : -INFINITY;
      // (keys without a visible one of this row have the reference 0 and zeros)
      s_f[row][lane16] = l == 0.0f || here == -INFINITY ? 0.0f : fast_exp2(here - top) / l;
    }
    __syncthreads();
    bool in[kFinishTiles];
#pragma unroll
    for (int k = 0; k < kFinishTiles; ++k)
      in[k] = kt0 + k < tiles && met(kt0 + k) && key0 + kTileKeys * k + (int32_t)threadIdx.x < s.len;
    for (int32_t r0 = 0;;) {
#pragma unroll
      for (int k = 0; k < kFinishTiles; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool use = in[k] && r0 + r < s.rows && x[k][r] != 0.0f;  // (a hidden key takes no part in a row of NaN)
          w[k] = use ? fmaf(x[k][r], s_f[min(r0 + r, kFewRows - 1)][4 * k + (threadIdx.x >> 6)], w[k]) : w[k];
        }
      r0 += 4;
      if (r0 >= s.rows) break;
      read(r0);
    }
  }
#pragma unroll
  for (int k = 0; k < kFinishTiles; ++k) {
    const int32_t j = key0 + kTileKeys * k + (int32_t)threadIdx.x;
    if (j < p.L) p.out[unit * p.L + j] = before[k] + w[k];
  }
}

// ---------------------------------------------------------------------------
// Chunks: rows stream past the keys twice
// ---------------------------------------------------------------------------
// Bound by vector instructions: the softmax's exponentials and sums, 0.75 of
// the units' time in the first pass and 0.60 in the second, the matrix units
// 0.31. The last 512 tokens of four prompts of up to 6000 tokens, 32 heads
// over 8, 128, fp16: 120 + 6 + 123 + 5 us (passes, rows' sums, parts).

// SUM = false: every row's maximum and sum over the tile's keys; true: every
// key's weights, with the rows' lse known, and the result.
template <int FMT, int D, bool SUM>
__global__ __launch_bounds__(256, 2) void chunk_rows_kernel(const ScoresParams p) {
  using K = Keys<FMT, D>;
  constexpr int NCH = K::NCH, TR = 32, RB = 2 * D, CPR = RB / 16, RPC = 1024 / RB, NC = TR / RPC / 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds_q[2][TR * RB];
  __shared__ float2 s_ml[2][4][TR];
  const int32_t h = (int32_t)(blockIdx.x % p.Hk), tp = (int32_t)(blockIdx.x / p.Hk), kt = tp / p.parts, part = tp % p.parts;
  const int32_t b = blockIdx.y;
  const int lane = threadIdx.x & 63, n = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ScoredSeq s = scored_seq(p, b);
  const int32_t key0 = kt * kTileKeys + 64 * wave;
  int32_t lo, hi;
  queries_of(p, s, s.rows / p.G, kt * kTileKeys, (kt + 1) * kTileKeys, lo, hi);
  f32x4p_t w[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) w[g] = (f32x4p_t){};
  // This workgroup's part of the tiles of TR rows from the first that sees a key to the last.
  const int32_t ta = lo * p.G / TR, tn = (hi * p.G + TR - 1) / TR - ta;
  const int32_t t0 = ta + (int32_t)((int64_t)tn * part / p.parts), t1 = ta + (int32_t)((int64_t)tn * (part + 1) / p.parts);
  if (hi > lo && t1 > t0) {
    K keys;
    keys.load(p, K::entries(p, b, key0, s.len), h, key0);
    const uint32_t linked = keys.linked;
    u32x4p_t a[4][NCH];
    f32x4p_t f[4][K::NG];
#pragma unroll
    for (int g = 0; g < 4; ++g) keys.operands(g, a[g], f[g]);
    const int64_t row_base = (int64_t)s.start * p.G;
    auto q_swz = [](int row) { return CPR == 16 ? row & 15 : (row >> 1) & 7; };
    // Rows past the last are copies of it: their weights are zeros.
    auto load_q = [&](int32_t t, int buf) __attribute__((always_inline)) {
      const int32_t tok0 = p.by_g(t * TR);
      const uint8_t *base = reinterpret_cast<const uint8_t *>(p.q + (int64_t)(s.start + tok0) * p.q_ts + (int64_t)h * p.G * p.q_hs);
      const auto rsrc = uniform_rsrc(base, 0x7FFFFFFF);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int lrow = (wave * NC + c) * RPC + lane / CPR;
        const int32_t row = min(t * TR + lrow, s.rows - 1), tok = p.by_g(row);
        const uint32_t off[1] = {(uint32_t)(2 * ((tok - tok0) * (int32_t)p.q_ts + (row - tok * p.G) * (int32_t)p.q_hs) +
                                            16 * ((lane % CPR) ^ q_swz(lrow)))};
        lds_dma<0, 1>(rsrc, lds_u32(lds_q[buf]) + (uint32_t)(wave * NC + c) * 1024, off, 0);
      }
    };
    auto load_lse = [&](int32_t t, float (&v)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int32_t row = t * TR + 16 * i + n;
        v[i] = SUM && row < s.rows ? p.lse[(int64_t)h * p.T * p.G + row_base + row] : INFINITY;
      }
    };
    auto publish = [&]() __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __syncthreads();
    };
    float lse[2], lse_next[2];
    load_q(t0, 0);
    load_lse(t0, lse_next);
    publish();
    for (int32_t t = t0; t < t1; ++t) {
      const int buf = (t - t0) & 1;
#pragma unroll
      for (int i = 0; i < 2; ++i) lse[i] = lse_next[i];
      if (t + 1 < t1) {
        load_lse(t + 1, lse_next);
        load_q(t + 1, buf ^ 1);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int32_t r0 = t * TR + 16 * i, row = r0 + n;
        const int32_t pos = s.pos0 + p.by_g(min(row, s.rows - 1));
        const int32_t first = s.pos0 + p.by_g(min(r0, s.rows - 1)), last = s.pos0 + p.by_g(min(r0 + 15, s.rows - 1));
        const bool full = r0 + 15 < s.rows && key0 + 63 <= first && key0 + 64 <= s.len && linked == 15u &&
                          (key0 > last - p.W || key0 + 64 <= p.sinks);
        u32x4p_t q[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c)
          q[c] = *reinterpret_cast<const u32x4p_t *>(lds_q[buf] + (16 * i + n) * RB +
                                                     16 * ((8 * (c >> 1) + 2 * kq + (c & 1)) ^ q_swz(16 * i + n)));
        if constexpr (K::CODES)
#pragma unroll
          for (int c = 0; c < NCH; ++c) q[c] = in_code_order(q[c]);
        if constexpr (SUM) {
          if (full) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const f32x4p_t x = K::scores(a[g], f[g], q);
#pragma unroll
              for (int r = 0; r < 4; ++r) w[g][r] += fast_exp2(fmaf(x[r], p.qk_scale_log2, -lse[i]));
            }
          } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const f32x4p_t x = hide(p, K::scores(a[g], f[g], q), key0 + 16 * g + 4 * kq, pos, s.len,
                                      row < s.rows && ((linked >> g) & 1));
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float y = fast_exp2(fmaf(x[r], p.qk_scale_log2, -lse[i]));
                w[g][r] += x[r] == -INFINITY ? 0.0f : y;  // (a hidden key takes no part in a row of NaN)
              }
            }
          }
        } else {
          f32x4p_t x[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            x[g] = K::scores(a[g], f[g], q);
            if (!full) x[g] = hide(p, x[g], key0 + 16 * g + 4 * kq, pos, s.len, row < s.rows && ((linked >> g) & 1));
          }
          float m = x[0][0], l = 0.0f;
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) m = fmaxf(m, x[g][r]);
          m = max_over_quarters(m) * p.qk_scale_log2;
          const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) l += fast_exp2(fmaf(x[g][r], p.qk_scale_log2, -ref));
          l = sum_over_quarters(l);
          // (keys without a maximum add nothing, unless all that the row sees of them is NaN)
          if (kq == 0) s_ml[buf][wave][16 * i + n] = float2{l == 0.0f ? m : fmaxf(m, -3e38f), l};
        }
      }
      publish();
      if (!SUM && threadIdx.x < TR && t * TR + (int32_t)threadIdx.x < s.rows) {
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, s_ml[buf][i][threadIdx.x].x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = s_ml[buf][i][threadIdx.x];
          if (v.x != -INFINITY) l += v.y * fast_exp2(v.x - m);
        }
        p.ml[((int64_t)h * p.kts + kt) * p.T * p.G + row_base + t * TR + threadIdx.x] = float2{m, l};
      }
    }
  }
  if constexpr (SUM) {
    const int64_t unit = (int64_t)b * p.Hk + h;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = w[g][r];
        v += xor1(v);
        v += xor2(v);
        v += half_mirror(v);
        v += dpp_f32<0x140>(v);
        const int32_t j = key0 + 16 * g + 4 * kq + r;
        if (n == 0 && p.parts > 1) p.sums[((int64_t)part * p.B * p.Hk + unit) * ((int64_t)p.kts * kTileKeys) + j] = v;
        else if (n == 0 && j < p.L) p.out[unit * p.L + j] = (p.scores ? p.scores[unit * p.L + j] : 0.0f) + v;
      }
  }
}

// lse of every row: a thread per row and key head.
__global__ __launch_bounds__(256) void lse_kernel(const ScoresParams p) {
  const int32_t h = (int32_t)(blockIdx.x % p.Hk), row = (int32_t)(blockIdx.x / p.Hk) * 256 + (int32_t)threadIdx.x;
  const ScoredSeq s = scored_seq(p, blockIdx.y);
  if (row >= s.rows) return;
  const int32_t pos = s.pos0 + p.by_g(row), tiles = (min(s.len, pos + 1) + kTileKeys - 1) / kTileKeys;
  const float2 *src = p.ml + (int64_t)h * p.kts * p.T * p.G + (int64_t)s.start * p.G + row;
  float m = -INFINITY, l = 0.0f;
  for (int32_t t0 = 0; t0 < tiles; t0 += 8) {
    float2 x[8];  // (eight reads in flight)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = src[(int64_t)min(t0 + i, tiles - 1) * p.T * p.G];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int32_t t = t0 + i;
      const float top = fmaxf(m, x[i].x);
      if (t >= tiles || !meets(p, pos, t * kTileKeys, (t + 1) * kTileKeys) || top == -INFINITY) continue;
      l = l * fast_exp2(m - top) + x[i].y * fast_exp2(x[i].x - top);
      m = top;
    }
  }
  p.lse[(int64_t)h * p.T * p.G + (int64_t)s.start * p.G + row] = l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// out = scores + the parts' sums, in their order.
__global__ __launch_bounds__(256) void add_parts_kernel(const ScoresParams p) {
  const int32_t h = (int32_t)(blockIdx.x % p.Hk), j = (int32_t)(blockIdx.x / p.Hk) * kTileKeys + (int32_t)threadIdx.x;
  if (j >= p.L) return;
  const int64_t unit = (int64_t)blockIdx.y * p.Hk + h, row = (int64_t)p.kts * kTileKeys;
  const float *src = p.sums + unit * row + j;
  float v = p.scores ? p.scores[unit * p.L + j] : 0.0f;
  float w = 0.0f;
  if (j < row)
    for (int i = 0; i < p.parts; ++i) w += src[(int64_t)i * p.B * p.Hk * row];
  p.out[unit * p.L + j] = v + w;
}

struct ScoresPlan {
  bool few;
  int32_t max_rows, kts, parts;
  int32_t group;  // few rows: sequences whose weights the workspace holds at once
  int64_t second, third, total;  // offsets of probs or lse behind ml, and of the parts' sums
};
static constexpr int kMaxParts = 8;
// Weights of few rows are kept for as many sequences at a time as this holds, one at least: all of a batch would be
// requests x rows x the longest context allowed, whatever the contexts are. (64 requests of 65536 tokens and 8 x 16
// rows, 2.1 GB: all at once 1406 us, by 1 GiB 1423, 512 MiB 1470, 256 MiB 1495; the same with 20 live at 3000
// tokens, where each group of sequences costs its launches: 100, 107, 147, 158.)
static constexpr int64_t kMaxProbs = 1LL << 30;
static int64_t scored_keys(const memopt_scores_desc &d) {
  return std::min<int64_t>((int64_t)d.max_blocks_per_seq * d.block_size, std::max(0, d.max_seq_len));
}
static ScoresPlan scores_plan(const memopt_scores_desc &d) {
  const int64_t G = d.num_heads / d.num_kv_heads, rows = (int64_t)std::min(d.max_query_len, d.tokens) * G;
  ScoresPlan pl = {};
  pl.few = rows <= kFewRows;
  pl.max_rows = (int32_t)rows;
  pl.kts = (int32_t)((scored_keys(d) + kTileKeys - 1) / kTileKeys);
  const int64_t probs = 4LL * d.num_kv_heads * rows * pl.kts * kTileKeys;  // of one sequence
  pl.group = (int32_t)std::min<int64_t>(d.batch, std::max<int64_t>(1, kMaxProbs / std::max<int64_t>(1, probs)));
  const int64_t ml = 8LL * pl.kts * d.num_kv_heads * (pl.few ? 4LL * pl.group * rows : d.tokens * G);
  pl.second = (ml + 255) / 256 * 256;
  const int64_t units = (int64_t)d.batch * d.num_kv_heads;
  pl.third = pl.second + (pl.few ? pl.group * probs : (4LL * d.num_kv_heads * d.tokens * G + 255) / 256 * 256);
  // Workgroups that share a key tile's rows: as many as make sixteen for each compute unit, with 256 rows or more each
  // (four prompts' last 512 tokens, 2.25 key tiles with keys for each unit: whole 306 us, four workgroups for each unit
  // 267, eight 244, sixteen 243, 32 247).
  pl.parts = (int32_t)std::min<int64_t>({kMaxParts, std::max<int64_t>(1, rows / 256),
                                         16 * compute_units() / std::max<int64_t>(1, pl.kts * units) + 1});
  pl.total = pl.third + (pl.few || pl.parts == 1 ? 0 : 4LL * pl.parts * units * pl.kts * kTileKeys);
  if (rows == 0 || pl.kts == 0) pl.total = 0;
  return pl;
}

static int validate_scores(const memopt_scores_desc &d) {
  MEMOPT_REQUIRE(d.tokens >= 0 && d.batch >= 0 && d.max_query_len >= 0 && d.scores_len >= 0, MEMOPT_ERR_INVALID,
                 "attention_scores: negative size");
  MEMOPT_REQUIRE(d.num_heads > 0 && d.num_kv_heads > 0 && d.num_heads % d.num_kv_heads == 0, MEMOPT_ERR_INVALID,
                 "attention_scores: num_heads must be a positive multiple of num_kv_heads");
  MEMOPT_REQUIRE(d.kv_format == MEMOPT_KV_FP16 || d.kv_format == MEMOPT_KV_INT4, MEMOPT_ERR_UNSUPPORTED,
                 "attention_scores: the cache must be an fp16 pool or INT4 pages");
  MEMOPT_REQUIRE(d.head_dim == 64 || d.head_dim == 128, MEMOPT_ERR_UNSUPPORTED,
                 "attention_scores: head_dim must be 64 or 128");
  MEMOPT_REQUIRE(d.num_kv_blocks > 0 && d.max_blocks_per_seq > 0 && d.block_size > 0, MEMOPT_ERR_INVALID,
                 "attention_scores: empty cache or block table");
  MEMOPT_REQUIRE(d.kv_format == MEMOPT_KV_FP16 ? d.block_size % 16 == 0 : d.block_size == 16, MEMOPT_ERR_UNSUPPORTED,
                 "attention_scores: pages must hold 16 tokens (fp16 pools: a multiple of 16)");
  MEMOPT_REQUIRE((int64_t)d.max_blocks_per_seq * d.block_size <= 1 << 30 && d.scores_len <= 1 << 30,
                 MEMOPT_ERR_UNSUPPORTED, "attention_scores: block tables and scores of up to 2^30 tokens");
  const int64_t G = d.num_heads / d.num_kv_heads;
  const int64_t tiles = (std::max<int64_t>(scored_keys(d), d.scores_len) + kTileKeys - 1) / kTileKeys;
  MEMOPT_REQUIRE((int64_t)d.tokens * d.num_heads <= INT32_MAX - 255 && d.batch <= 65535 &&
                     tiles * d.num_kv_heads * std::max(1, d.batch) < (1LL << 24) &&
                     ((int64_t)d.tokens * G + 255) / 256 * d.num_kv_heads * std::max(1, d.batch) < (1LL << 24),
                 MEMOPT_ERR_UNSUPPORTED, "attention_scores: too many (row, token) tiles for one call");
  MEMOPT_REQUIRE(d.q_token_stride >= 0 && d.q_head_stride >= 0 &&
                     d.q_token_stride < (1LL << 30) && d.q_head_stride < (1LL << 30) &&
                     31 * d.q_token_stride + (G - 1) * d.q_head_stride < (1LL << 29),
                 MEMOPT_ERR_UNSUPPORTED, "attention_scores: query rows lie too far apart");
  MEMOPT_REQUIRE(((uintptr_t)d.query & 15) == 0 && d.q_token_stride % 8 == 0 && d.q_head_stride % 8 == 0 &&
                     ((uintptr_t)d.key_cache & 15) == 0 && ((uintptr_t)d.workspace & 15) == 0,
                 MEMOPT_ERR_INVALID, "attention_scores: rows, cache and workspace must be 16-byte aligned");
  return MEMOPT_OK;
}

template <int FMT, int D>
static int launch_scores(const ScoresParams &p, const ScoresPlan &pl, hipStream_t s) {
  const unsigned tiles = (unsigned)((std::max<int64_t>(p.max_keys, p.L) + kTileKeys - 1) / kTileKeys);
  const dim3 over_keys((unsigned)pl.kts * pl.parts * p.Hk, p.B), over_scores(tiles * p.Hk, p.B);
  const dim3 finish((tiles + kFinishTiles - 1) / kFinishTiles * p.Hk, p.B);
  int rc;
  if (pl.total == 0) {
    hipLaunchKernelGGL(finish_kernel, finish, dim3(256), 0, s, p);
    return check_launch("attention_scores");
  }
  if (pl.few) {
    // Tiles of a workgroup: as many as leave each compute unit sixteen workgroups (four are resident), at most
    // eight (32 sequences of up to 8192 tokens: four per unit 37.6 us, eight 35.1, sixteen 33.5, 32 36.9).
    const int64_t each = std::min<int64_t>(8, std::max<int64_t>(1, (int64_t)pl.kts * p.Hk * pl.group / (16 * compute_units())));
    ScoresParams g = p;
    for (int32_t b = 0; b < p.B; b += pl.group) {
      const unsigned n = (unsigned)std::min(pl.group, p.B - b);
      g.bt = p.bt + (int64_t)b * p.M;
      g.ctx = p.ctx + b;
      g.starts = p.starts + b;
      g.scores = p.scores ? p.scores + (int64_t)b * p.Hk * p.L : nullptr;
      g.out = p.out + (int64_t)b * p.Hk * p.L;
      const dim3 grid((unsigned)((pl.kts + each - 1) / each * p.Hk), n);
      hipLaunchKernelGGL((few_rows_kernel<FMT, D>), grid, dim3(256), 0, s, g, (int32_t)each);
      if ((rc = check_launch("attention_scores(rows)")) != MEMOPT_OK) return rc;
      hipLaunchKernelGGL(finish_kernel, dim3(finish.x, n), dim3(256), 0, s, g);
      if ((rc = check_launch("attention_scores(finish)")) != MEMOPT_OK) return rc;
    }
    return MEMOPT_OK;
  }
  hipLaunchKernelGGL((chunk_rows_kernel<FMT, D, false>), over_keys, dim3(256), 0, s, p);
  if ((rc = check_launch("attention_scores(maxima)")) != MEMOPT_OK) return rc;
  hipLaunchKernelGGL(lse_kernel, dim3((unsigned)((p.max_rows + 255) / 256 * p.Hk), p.B), dim3(256), 0, s, p);
  if ((rc = check_launch("attention_scores(lse)")) != MEMOPT_OK) return rc;
  hipLaunchKernelGGL((chunk_rows_kernel<FMT, D, true>), pl.parts > 1 ? over_keys : over_scores, dim3(256), 0, s, p);
  if ((rc = check_launch("attention_scores(sums)")) != MEMOPT_OK || pl.parts == 1) return rc;
  hipLaunchKernelGGL(add_parts_kernel, over_scores, dim3(256), 0, s, p);
  return check_launch("attention_scores(parts)");
}

}  // namespace memopt

using namespace memopt;

extern "C" int memopt_scores_workspace_size(const memopt_scores_desc *desc, int64_t *bytes) {
  MEMOPT_REQUIRE(desc && bytes, MEMOPT_ERR_INVALID, "scores_workspace_size: null pointer");
  *bytes = 0;
  int rc = validate_scores(*desc);
  if (rc != MEMOPT_OK || desc->batch == 0 || desc->scores_len == 0) return rc;
  *bytes = scores_plan(*desc).total;
  return MEMOPT_OK;
}

extern "C" int memopt_attention_scores(const memopt_scores_desc *desc, void *stream) {
  MEMOPT_REQUIRE(desc, MEMOPT_ERR_INVALID, "attention_scores: null descriptor");
  const memopt_scores_desc &d = *desc;
  int rc = validate_scores(d);
  if (rc != MEMOPT_OK || d.batch == 0 || d.scores_len == 0) return rc;
  const ScoresPlan pl = scores_plan(d);
  MEMOPT_REQUIRE(d.out && d.context_lens && d.query_starts && (pl.total == 0 || (d.query && d.key_cache && d.block_tables)),
                 MEMOPT_ERR_INVALID, "attention_scores: null pointer");
  MEMOPT_REQUIRE(pl.total == 0 || (d.workspace && d.workspace_bytes >= pl.total), MEMOPT_ERR_INVALID,
                 "attention_scores: workspace needs " + std::to_string(pl.total) + " bytes");
  const int64_t sums = 4LL * d.batch * d.num_kv_heads * d.scores_len;
  MEMOPT_REQUIRE(d.out == d.scores || !overlap({d.out, sums}, {d.scores, d.scores ? sums : 0}), MEMOPT_ERR_INVALID,
                 "attention_scores: out must be scores, or not overlap it");
  ScoresParams p = {};
  p.q = (const uint16_t *)d.query;
  p.q_ts = d.q_token_stride;
  p.q_hs = d.q_head_stride;
  p.k = (const uint8_t *)d.key_cache;
  p.T = pl.total == 0 ? 0 : d.tokens;
  p.B = d.batch;
  p.Hk = d.num_kv_heads;
  p.G = d.num_heads / d.num_kv_heads;
  p.by_g = Divisor::of((uint32_t)p.G);
  p.by_chunks = Divisor::of((uint32_t)d.block_size / 16);
  if (d.kv_format == MEMOPT_KV_INT4) {
    p.k_hs = Int4Page(d.head_dim).block;
    p.k_ps = p.Hk * p.k_hs;
  } else {
    p.k_hs = 2 * d.head_dim;
    p.k_ts = p.Hk * p.k_hs;
    p.k_ps = d.block_size * p.k_ts;
  }
  p.bt = d.block_tables;
  p.ctx = d.context_lens;
  p.starts = d.query_starts;
  p.nb = d.num_kv_blocks;
  p.scores = d.scores;
  p.out = d.out;
  p.M = d.max_blocks_per_seq;
  p.bs = d.block_size;
  p.W = std::min(effective_window(d.window_size, d.max_seq_len), 1 << 30);  // (position - W stays in 32 bits)
  p.sinks = std::max(0, d.num_sink_tokens);
  p.L = d.scores_len;
  p.max_keys = (int32_t)scored_keys(d);
  p.max_rows = pl.max_rows;
  p.kts = pl.kts;
  p.qk_scale_log2 = 1.4426950408889634f / sqrtf((float)d.head_dim);
  p.ml = (float2 *)d.workspace;
  (pl.few ? p.probs : p.lse) = (float *)((uint8_t *)d.workspace + pl.second);
  p.parts = pl.few ? 1 : pl.parts;
  p.sums = (float *)((uint8_t *)d.workspace + pl.third);
  hipStream_t s = (hipStream_t)stream;
  if (d.kv_format == MEMOPT_KV_INT4)
    return d.head_dim == 128 ? launch_scores<MEMOPT_KV_INT4, 128>(p, pl, s) : launch_scores<MEMOPT_KV_INT4, 64>(p, pl, s);
  return d.head_dim == 128 ? launch_scores<MEMOPT_KV_FP16, 128>(p, pl, s) : launch_scores<MEMOPT_KV_FP16, 64>(p, pl, s);
}
