// latent_prompt.hip — causal attention over whole packed prompts with keys of
// two parts: one per head, and a rotary one that all heads share (gfx950
// matrix cores). The expanded form of latent attention: keys and values as
// the up-projection of the latents leaves them.
//
// For query row i of a sequence and head h:
//   s_ij = (q_ih[0 .. D) . k_jh + q_ih[D .. D + P) . r_j) scale,
//   o_i = sum_j softmax_j(s_ij) v_jh,   j <= i and (j < sinks or j > i - W)
// One pass over the keys with a running maximum and sum, as in prompt.hip: a
// workgroup takes 128 rows of a head (32 per wave, the columns of both
// products) against tiles of 64 keys in LDS. The shared part is copied into
// every head's tile, so that no head's keys are ever joined in memory.
//
// Measured (128 + 64; medians): three prompts of up to 9000 tokens, 32 heads,
// fp16: 0.89-0.96 ms, 0.91-0.97 PFLOP/s, 0.74-0.79 of the library's rate on a large product: a
// wave's softmax stands between its two products, and the other workgroup on
// the compute unit fills in (of 256 registers 234 are taken: neither a second
// set of scores nor copies dealt over the products fit without spills). 24 prompts of 20 to 2500 tokens, 16 heads, bf16:
// 138-148 us, 0.65 PFLOP/s of what the mask leaves: masked tiles are whole
// products, and 2016 workgroups are four rounds of the GPU.
#include <algorithm>
#include <cmath>

#include "attention.hpp"
#include "lds_dma.hpp"
#include "tiles.hpp"

namespace memopt {

struct ExpandedParams {
  const uint16_t *q, *k, *r, *v;
  uint16_t *out;
  int64_t q_ts, q_hs, k_ts, k_hs, r_ts, v_ts, v_hs, o_ts, o_hs;
  const int32_t *starts;
  int32_t T, B, H, G, W, sinks;  // G = 1: every head has keys of its own
  float scale_log2;
};

// A tile of 64 rows of N elements in LDS: 16-byte pieces, swizzled so that the
// reads of one piece of eight rows (and for values, of 32 bytes of four rows)
// meet no bank twice.
template <int N>
struct TileRows {
  static constexpr int RB = 2 * N, CPR = RB / 16, RPC = 1024 / RB, NC = 64 / RPC / 4;  // NC copies per wave
  static __device__ __forceinline__ int key_swz(int row) {
    return CPR == 16 ? row & 15 : CPR == 8 ? (row >> 1) & 7 : (row >> 2) & 3;
  }
  static __device__ __forceinline__ int value_swz(int row) { return CPR == 16 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }
};

template <class E, int D, int P>
__global__ __launch_bounds__(256, 2) void latent_prompt_kernel(const ExpandedParams p) {
  using K = TileRows<D>;
  using RP = TileRows<P>;
  constexpr int TK = 64, R = 128, NCK = D / 16, NCH = (D + P) / 16, NDB = D / 32;
  __shared__ __attribute__((aligned(16))) uint8_t lds_k[2][TK * K::RB], lds_r[2][TK * RP::RB], lds_v[2][TK * K::RB];
  const int lane = threadIdx.x & 63, n = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroup i runs on XCD i % 8: a head's workgroups share an XCD and its L2 where the heads deal out evenly.
  const int32_t h = (int32_t)(blockIdx.x % p.H);
  Tile tile;
  if (!find_tile<R, false>(p, (int32_t)(blockIdx.x / p.H), tile)) return;
  const Rows seq = rows_of(p.starts, p.T, __builtin_amdgcn_readfirstlane(tile.b));
  const int32_t len = __builtin_amdgcn_readfirstlane(seq.n), start = __builtin_amdgcn_readfirstlane(seq.start);
  const int32_t q0 = R * __builtin_amdgcn_readfirstlane(tile.t), qw0 = q0 + 32 * wave, row = qw0 + n;

  u32x4p_t qf[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) qf[c] = (u32x4p_t){};
  if (row < len) {
    const uint16_t *src = p.q + (int64_t)(start + row) * p.q_ts + h * p.q_hs + 8 * hl;
#pragma unroll
    for (int c = 0; c < NCH; ++c) qf[c] = *reinterpret_cast<const u32x4p_t *>(src + 16 * c);
  }

  // Tiles of the workgroup: sinks, then the window of its rows.
  const int32_t hi = min(len, q0 + R), sink_tiles = (min(p.sinks, hi) + TK - 1) / TK;
  const int32_t t_first = max(max(0, q0 - p.W + 1) / TK, sink_tiles);
  const int32_t n_tiles = sink_tiles + max(0, (hi + TK - 1) / TK - t_first);
  auto tile_base = [&](int32_t it) { return (it < sink_tiles ? it : t_first + (it - sink_tiles)) * TK; };

  const uint32_t k_rb = 2 * (uint32_t)p.k_ts, r_rb = 2 * (uint32_t)p.r_ts, v_rb = 2 * (uint32_t)p.v_ts;
  uint32_t k_off[K::NC], v_off[K::NC], r_off[RP::NC];
#pragma unroll
  for (int c = 0; c < K::NC; ++c) {
    const int lr = (wave * K::NC + c) * K::RPC + lane / K::CPR, j = lane % K::CPR;
    k_off[c] = lr * k_rb + 16 * (j ^ K::key_swz(lr)) - c * 1024;
    v_off[c] = lr * v_rb + 16 * (j ^ K::value_swz(lr)) - c * 1024;
  }
#pragma unroll
  for (int c = 0; c < RP::NC; ++c) {
    const int lr = (wave * RP::NC + c) * RP::RPC + lane / RP::CPR, j = lane % RP::CPR;
    r_off[c] = lr * r_rb + 16 * (j ^ RP::key_swz(lr)) - c * 1024;
  }
  const uint8_t *k_base = reinterpret_cast<const uint8_t *>(p.k + start * p.k_ts + h * p.k_hs);
  const uint8_t *r_base = reinterpret_cast<const uint8_t *>(p.r + start * p.r_ts);
  const uint8_t *v_base = reinterpret_cast<const uint8_t *>(p.v + start * p.v_ts + h * p.v_hs);
  // Rows past the sequence lie outside a tile's range and read as zeros.
  auto rows_at = [&](const uint8_t *base, uint32_t rb, int32_t key0, int width) __attribute__((always_inline)) {
    return uniform_rsrc(base + (int64_t)key0 * rb, (int)((min(TK, len - key0) - 1) * rb + width));
  };
  auto load = [&](int32_t it, int buf) __attribute__((always_inline)) {
    const int32_t tb = tile_base(it);
    lds_dma_range<0, K::NC>(rows_at(k_base, k_rb, tb, K::RB), lds_u32(lds_k[buf]) + wave * K::NC * 1024, k_off, 0);
    lds_dma_range<0, RP::NC>(rows_at(r_base, r_rb, tb, RP::RB), lds_u32(lds_r[buf]) + wave * RP::NC * 1024, r_off, 0);
    lds_dma_range<0, K::NC>(rows_at(v_base, v_rb, tb, K::RB), lds_u32(lds_v[buf]) + wave * K::NC * 1024, v_off, 0);
  };

  uint32_t ka[NCH], va[NDB];
#pragma unroll
  for (int c = 0; c < NCH; ++c)
    ka[c] = c < NCK ? n * K::RB + 16 * ((2 * c + hl) ^ K::key_swz(n))
                    : n * RP::RB + 16 * ((2 * (c - NCK) + hl) ^ RP::key_swz(n));
  const int i16 = lane & 15, vrow = 4 * hl + (i16 >> 2);
#pragma unroll
  for (int db = 0; db < NDB; ++db)
    va[db] = vrow * K::RB + 16 * ((4 * db + 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ K::value_swz(vrow)) + 8 * (i16 & 1);

  f32x16_t o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = (f32x16_t){};
  // x = scale_log2 s + ncm is the exp2 argument; a new maximum lands at kTop and
  // the next rescale comes past kTop + 8 (prompt.hip).
  constexpr float kTop = E::kTop;
  float ncm = 0.0f, thr = -INFINITY, lsum = 0.0f;
  uint32_t odd = 0;  // nonzero where a masked tile's V held inf or NaN
  const int32_t last_row = min(qw0 + 31, len - 1);
  auto sees = [&](int32_t tb) {
    return qw0 < len && tb <= last_row && (tb + TK > qw0 - p.W + 1 || tb < p.sinks);
  };
  auto whole = [&](int32_t tb) {
    return qw0 + 31 < len && tb + TK - 1 <= qw0 && (tb > last_row - p.W || tb + TK <= p.sinks);
  };

  if (n_tiles > 0) load(0, 0);
  for (int32_t it = 0; it < n_tiles; ++it) {
    const int buf = it & 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // this tile has arrived, and nobody reads the other buffer any more
    if (it + 1 < n_tiles) load(it + 1, buf ^ 1);
    const int32_t tb = tile_base(it);
    if (!sees(tb)) continue;
    const bool full = whole(tb);
    f32x16_t x[2];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      x[blk] = (f32x16_t){};
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const uint8_t *src = c < NCK ? lds_k[buf] + 32 * blk * K::RB : lds_r[buf] + 32 * blk * RP::RB;
        x[blk] = E::mfma(*reinterpret_cast<const u32x4p_t *>(src + ka[c]), qf[c], x[blk]);
      }
    }
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int r = 0; r < 16; ++r) x[blk][r] = fmaf(x[blk][r], p.scale_log2, ncm);
    if (!full) {
      // Register r of block blk holds key tb + 32 blk + 8 (r / 4) + 4 hl + r % 4.
      const int32_t key0 = tb + 4 * hl, last = row < len ? row - key0 : -1;
      const int32_t first = row - p.W + 1 - key0, sink = p.sinks - key0;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int32_t c = 32 * blk + 8 * (r >> 2) + (r & 3);
          x[blk][r] = (c <= last) & ((c >= first) | (c < sink)) ? x[blk][r] : -INFINITY;
        }
    }
    float t = x[0][0];
#pragma unroll
    for (int r = 1; r < 16; ++r) t = fmaxf(t, x[0][r]);
#pragma unroll
    for (int r = 0; r < 16; ++r) t = fmaxf(t, x[1][r]);
    t = both_halves_max(t);
    if (__any(t > thr)) {
      const bool first = thr == -INFINITY, found = t > -INFINITY;
      const float shift = first ? (found ? t - kTop : 0.0f) : fmaxf(t - kTop, 0.0f);
      const float alpha = first ? 1.0f : fast_exp2(-shift);  // (nothing summed before the first maximum)
      lsum *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[blk][r] -= shift;
      ncm -= shift;
      thr = first && !found ? thr : kTop + 8.0f;
    }
    // Weights enter the second product in 16 bits, and so the row's sum. (What the rounding leaves, as a second operand,
    // would bring the result's error from 1.96e-3 of its norm to its own rounding, 1.59e-3 (bf16), and the time of
    // short prompts from 144 to 174 us, of long ones from 923 to 1203.)
    u32x4p_t pb[4];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      pb[i >> 2][i & 3] = E::pack(fast_exp2(x[i >> 3][2 * (i & 7)]), fast_exp2(x[i >> 3][2 * (i & 7) + 1]));
#pragma unroll
    for (int i = 0; i < 16; ++i) lsum = E::dot2(pb[i >> 2][i & 3], E::kOnes, lsum);
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      u32x4p_t vf[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t *src = lds_v[buf] + 16 * i * K::RB;
        const u32x2p_t a = v_read(src, va[db]), b8 = v_read(src + 8 * K::RB, va[db]);
        vf[i] = u32x4p_t{a[0], a[1], b8[0], b8[1]};
      }
      if (!full) {
        // A weight of 0 must not meet an inf or NaN: a sum of zero times every element tells.
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) z = E::dot2(vf[i >> 2][i & 3], 0, z);
        if (__any(!(z == 0.0f))) {
#pragma unroll
          for (int i = 0; i < 16; ++i) vf[i >> 2][i & 3] = tame<E>(vf[i >> 2][i & 3], odd);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) o[db] = E::mfma(vf[i], pb[i], o[db]);
    }
  }

  if (__any(odd != 0)) {
    // inf and NaN in V entered the masked tiles as finite values. Rows that do
    // see one have inf or NaN in that column whatever its weight.
#pragma unroll 1
    for (int32_t it = 0; it < n_tiles; ++it) {
      const int32_t tb = tile_base(it);
      if (!sees(tb) || whole(tb)) continue;
#pragma unroll 1
      for (int32_t key = tb; key < min(tb + TK, len); ++key) {
        const uint16_t *src = reinterpret_cast<const uint16_t *>(v_base + (int64_t)key * v_rb) + 4 * hl;
        const bool see = row < len && key <= row && (key < p.sinks || key > row - p.W);
#pragma unroll
        for (int r = 0; r < 16 * NDB; ++r) {
          const uint16_t bits = src[8 * (r >> 2) + (r & 3)];
          if (see && (bits & E::kExponent) == E::kExponent) o[r >> 4][r & 15] += E::value(bits);
        }
      }
    }
  }

  const float l = xor32_sum(lsum), inv = l > 0.0f ? 1.0f / l : 0.0f;
  if (row >= len) return;
  uint16_t *dst = p.out + (int64_t)(start + row) * p.o_ts + h * p.o_hs + 4 * hl;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<u32x2p_t *>(dst + 32 * db + 8 * g) =
          u32x2p_t{E::pack(o[db][4 * g] * inv, o[db][4 * g + 1] * inv),
                   E::pack(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv)};
}

template <class E>
static void launch_expanded(const ExpandedParams &p, int32_t D, int32_t P, unsigned wgs, hipStream_t s) {
  if (D == 128 && P == 64) hipLaunchKernelGGL((latent_prompt_kernel<E, 128, 64>), dim3(wgs), dim3(256), 0, s, p);
  else if (D == 128) hipLaunchKernelGGL((latent_prompt_kernel<E, 128, 32>), dim3(wgs), dim3(256), 0, s, p);
  else if (P == 64) hipLaunchKernelGGL((latent_prompt_kernel<E, 64, 64>), dim3(wgs), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((latent_prompt_kernel<E, 64, 32>), dim3(wgs), dim3(256), 0, s, p);
}

}  // namespace memopt

using namespace memopt;

extern "C" int memopt_latent_prompt_attention(const memopt_latent_prompt_desc *desc, void *stream) {
  MEMOPT_REQUIRE(desc, MEMOPT_ERR_INVALID, "latent_prompt_attention: null descriptor");
  const memopt_latent_prompt_desc &d = *desc;
  MEMOPT_REQUIRE(d.dtype == MEMOPT_FP16 || d.dtype == MEMOPT_BF16, MEMOPT_ERR_INVALID,
                 "latent_prompt_attention: dtype must be fp16 or bf16");
  MEMOPT_REQUIRE(d.tokens >= 0 && d.batch >= 0 && d.num_heads > 0, MEMOPT_ERR_INVALID,
                 "latent_prompt_attention: negative size, or no heads");
  MEMOPT_REQUIRE((d.head_dim == 64 || d.head_dim == 128) && (d.rope_dim == 32 || d.rope_dim == 64), MEMOPT_ERR_UNSUPPORTED,
                 "latent_prompt_attention: head_dim must be 64 or 128, rope_dim 32 or 64");
  if (d.tokens == 0 || d.batch == 0) return MEMOPT_OK;
  MEMOPT_REQUIRE(d.query && d.key && d.rope_key && d.value && d.out && d.query_starts, MEMOPT_ERR_INVALID,
                 "latent_prompt_attention: null pointer");
  auto aligned = [](const void *x, int64_t ts, int64_t hs) {
    return ((uintptr_t)x & 15) == 0 && ts % 8 == 0 && hs % 8 == 0;
  };
  MEMOPT_REQUIRE(aligned(d.query, d.q_token_stride, d.q_head_stride) && aligned(d.key, d.k_token_stride, d.k_head_stride) &&
                     aligned(d.rope_key, d.r_token_stride, 0) && aligned(d.value, d.v_token_stride, d.v_head_stride) &&
                     aligned(d.out, d.o_token_stride, d.o_head_stride),
                 MEMOPT_ERR_INVALID, "latent_prompt_attention: rows must be 16-byte aligned");
  // (a tile of 64 rows lies in one 31-bit buffer range)
  auto in_range = [](int64_t ts, int64_t least) { return ts >= least && ts < (1LL << 23); };
  MEMOPT_REQUIRE(in_range(d.k_token_stride, d.head_dim) && in_range(d.v_token_stride, d.head_dim) &&
                     in_range(d.r_token_stride, d.rope_dim),
                 MEMOPT_ERR_UNSUPPORTED,
                 "latent_prompt_attention: key and value token strides must be a row to 2^23 - 1 elements");
  const int64_t tiles = ((int64_t)d.tokens + 127LL * std::min(d.batch, d.tokens)) / 128;
  MEMOPT_REQUIRE(d.tokens <= 1 << 30 && (int64_t)d.tokens * d.num_heads <= INT32_MAX - 255 &&
                     tiles * d.num_heads < (1LL << 24),
                 MEMOPT_ERR_UNSUPPORTED, "latent_prompt_attention: too many query rows");  // (a launch holds 2^32 - 1 threads)
  ExpandedParams p = {};
  p.q = (const uint16_t *)d.query;
  p.k = (const uint16_t *)d.key;
  p.r = (const uint16_t *)d.rope_key;
  p.v = (const uint16_t *)d.value;
  p.out = (uint16_t *)d.out;
  p.q_ts = d.q_token_stride;
  p.q_hs = d.q_head_stride;
  p.k_ts = d.k_token_stride;
  p.k_hs = d.k_head_stride;
  p.r_ts = d.r_token_stride;
  p.v_ts = d.v_token_stride;
  p.v_hs = d.v_head_stride;
  p.o_ts = d.o_token_stride;
  p.o_hs = d.o_head_stride;
  p.starts = d.query_starts;
  p.T = d.tokens;
  p.B = d.batch;
  p.H = d.num_heads;
  p.G = 1;
  p.W = d.window_size <= 0 ? 1 << 30 : std::min(d.window_size, 1 << 30);  // (position - W stays in 32 bits)
  p.sinks = std::max(0, d.num_sink_tokens);
  p.scale_log2 = 1.4426950408889634f * d.scale;
  const unsigned wgs = (unsigned)(tiles * d.num_heads);
  if (d.dtype == MEMOPT_FP16) launch_expanded<Fp16>(p, d.head_dim, d.rope_dim, wgs, (hipStream_t)stream);
  else launch_expanded<Bf16>(p, d.head_dim, d.rope_dim, wgs, (hipStream_t)stream);
  return check_launch("latent_prompt_attention");
}
