// packed.hip — attention of packed queries over a paged cache with grouped
// heads (gfx950 matrix cores): decode steps, a few tokens per sequence and
// chunks of prompts in one call, over INT4 pages and fp16 pools.
//
// For row i of sequence b (position pos_i = ctx - n + i) and query head h over
// key head h / G:
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(q . k_j / sqrt(D) - m),
//   j <= pos_i, j < ctx, and (j < sinks or j > pos_i - W), its page linked,
// the causal rule of attention.hpp key_range. INT4 elements are
// (code - 8) * scale.
//
// Why rows: the G query heads of a key head meet the same keys, so a key
// head's work on one sequence is n * G rows (row = token * G + head), and a
// block of 16 rows fills a matrix instruction that a lone query head would
// leave 15/16 empty. Every cached byte is read once per block of rows.
//
// Work: QN = 16 * QB rows of one (sequence, key head) are a block; a wave takes
// two 16-token chunks (32 tokens) of a block's visible ones per step. The steps
// of all blocks of a key head form one list, which is dealt to its workgroups
// of 4 waves in equal runs, whatever the sequences' lengths (by sequence and
// split, a batch of 2700 to 8192 tokens ran as long as its longest part). A
// block whose steps fall to one workgroup is finished there; else each
// leaves partial sums, and the last to arrive adds them up. Layout, as in direct.hip:
//  * S^T = K Q^T on v_mfma_f32_16x16x32_f16, one product per token half t: row
//    r of the A operand is token r % 8 + 8 t of chunk r / 8, which is how a
//    page interleaves its tokens. Over pages each product covers dims of one
//    scale group, so K enters as exact codes and the two groups' sums are
//    scaled in 32 bits: no rounding of K, and no multiply per element.
//  * lane (n, g) = (lane % 16, lane / 16) holds for row n the scores of tokens
//    p and p + 8, p = 4 (g % 2) .. + 3, of chunk g / 2; the same lane is column
//    n, k-group g of the B operand of O^T += V^T P^T, so probabilities stay in
//    their lane, and a page's V word unpacks into one register of four
//    operands.
// Output row rr of V^T product i is dim (D / 16) rr + i.
#include <algorithm>
#include <cmath>

#include "attention.hpp"
#include "page_format.hpp"

namespace memopt {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

struct PackedParams {
  const half_t *q;
  half_t *out;
  int64_t q_ts, q_hs, o_ts, o_hs;  // elements
  const int32_t *cu, *ctx, *bt;
  int32_t T, B, Hq, Hk, G, M, bs;
  int64_t nb;
  const uint8_t *k, *v;          // INT4 pages: k = the page buffer
  int64_t kv_ps, kv_hs, kv_ts;   // bytes
  int32_t W, sinks;
  float qk_scale_log2;
  int32_t wgs, blocks;           // workgroups per key head; blocks that ws_cnt has counters for
  uint32_t *ws_cnt;              // [blocks * Hk] arrivals; zero between calls
  float *ws_o, *ws_ml;           // [2 * wgs * Hk][QN][D], [2 * wgs * Hk][QN][2]: see partial_slot
};

// Workgroups per key head, so partial sums of a block, at most: their weights
// take the place of the waves' sums in LDS.
static constexpr int max_workgroups(int D) { return 4 * D; }

// Inclusive prefix sum over the wave (DPP row shifts, then row broadcasts),
// saturating: query starts that do not ascend can count rows more than once.
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

// What rows at positions pos_lo .. pos_hi of a context see, in 16-token
// chunks: the sinks [0, sc), then the window [wc0, wc0 + n - sc).
struct Visible {
  int32_t sc, wc0, n;
};
__device__ __forceinline__ Visible visible_chunks(const PackedParams &p, int32_t kv_lim, int32_t pos_lo,
                                                  int32_t pos_hi) {
  const int32_t hi = max(0, min(kv_lim, pos_hi + 1));
  Visible v;
  v.sc = (min(p.sinks, hi) + 15) >> 4;
  v.wc0 = max(max(0, pos_lo - p.W + 1) >> 4, v.sc);
  v.n = v.sc + max(0, ((hi + 15) >> 4) - v.wc0);
  return v;
}

// A sequence's rows and, in the list of steps, its blocks: each takes `steps`
// places, as many as its widest block can need (at least one, so that rows
// which see nothing are written, too).
struct Seq {
  int32_t start, n, ctx, kv_lim, blocks, steps;
};
template <int QN>
__device__ __forceinline__ Seq sequence(const PackedParams &p, int32_t b) {
  Seq q;
  q.start = min(max(p.cu[b], 0), p.T);
  q.n = min(max(p.cu[b + 1], q.start), p.T) - q.start;
  q.ctx = p.ctx[b];
  q.kv_lim = (int32_t)min((int64_t)q.ctx, (int64_t)p.M * p.bs);
  q.blocks = (q.n * p.G + QN - 1) / QN;
  const int32_t pos0 = q.ctx - q.n;
  int32_t n = visible_chunks(p, q.kv_lim, pos0, q.ctx - 1).n;
  if (q.blocks > 1) n = min(n, ((min(p.sinks, max(q.kv_lim, 0)) + 15) >> 4) + ((p.W + QN / p.G + 1) >> 4) + 2);
  q.steps = max(1, (n + 1) >> 1);
  return q;
}

// Raw registers of one step, by cache format.
template <int D, int FMT>
struct PackedK;
template <int D>
struct PackedK<D, MEMOPT_KV_INT4> {
  uint32_t w[D / 16];      // word of product kk, half t: see k_operand
  u32x4_t sc[D / 64];      // this lane's score rows: pair (p_i, p_i + 8) of group j in sc[j][i]
};
template <int D>
struct PackedK<D, MEMOPT_KV_FP16> {
  u32x4_t w[2][D / 32];
};
template <int D, int FMT>
struct PackedV;
template <int D>
struct PackedV<D, MEMOPT_KV_INT4> {
  uint32_t w[4][D / 64];  // [p_i][unit]
  u32x4_t sc;             // pair (p_i, p_i + 8) in word i
};
template <int D>
struct PackedV<D, MEMOPT_KV_FP16> {
  uint32_t w[8][D / 32];  // token e: D / 16 halves
};

template <int D, int FMT, int QB>
__global__ __launch_bounds__(256, QB == 1 ? (FMT == MEMOPT_KV_INT4 || D == 64 ? 4 : 2) : 2) void packed_kernel(
    const PackedParams p) {
  constexpr int NW = 4, NT = 64 * NW, KK = D / 32, ND = D / 16, QN = 16 * QB;
  constexpr bool PAGES = FMT == MEMOPT_KV_INT4;
  constexpr int NG = PAGES ? D / 64 : 1;  // score sums per (row, token)
  constexpr int OS = D + 4;               // row stride of s_o: 16 rows of D floats would share a bank
  __shared__ __attribute__((aligned(16))) float s_o[NW][QN][OS];
  __shared__ float s_ml[NW][QN][2];
  __shared__ int s_last;
  static_assert(NW * OS >= max_workgroups(D), "the weights of a merge fit s_o");

  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t kvh = blockIdx.x % p.Hk, wg = blockIdx.x / p.Hk;

  // The list's length; then the sequence that holds this workgroup's first place.
  uint32_t sum = 0;
  for (int32_t b0 = 0; b0 < p.B; b0 += 64) {
    uint32_t c = 0;
    if (b0 + lane < p.B) {
      const Seq q = sequence<QN>(p, b0 + lane);
      c = (uint32_t)q.blocks * (uint32_t)q.steps;
    }
    sum = __builtin_elementwise_add_sat(sum, (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(c), 63));
  }
  // (past 2^31 only where sequences overlap: nothing is computed then)
  const int32_t total = (int32_t)sum;
  // Runs of one step per wave at least: shorter ones cost more to merge than they save.
  const int32_t wgs = min(p.wgs, max(1, total / NW));
  if (total <= 0 || wg >= wgs) return;
  const int32_t run = total / wgs, longer = total - run * wgs;  // the first `longer` runs have one place more
  int32_t at = wg * run + min(wg, longer);
  const int32_t stop = at + run + (wg < longer ? 1 : 0);
  auto wg_of = [&](int32_t x) {
    const int32_t edge = longer * (run + 1);
    return x < edge ? x / (run + 1) : longer + (x - edge) / run;
  };
  int32_t seq_at = 0, seq_blocks = 0, b = 0;  // places and blocks before sequence b
  for (int32_t b0 = 0; b0 < p.B; b0 += 64) {
    uint32_t c = 0, nb = 0;
    if (b0 + lane < p.B) {
      const Seq q = sequence<QN>(p, b0 + lane);
      nb = q.blocks;
      c = nb * (uint32_t)q.steps;
    }
    const int32_t incl = (int32_t)wave_scan(c), blocks = (int32_t)wave_scan(nb);
    const int32_t sum64 = __builtin_amdgcn_readlane(incl, 63);
    if (at < seq_at + sum64) {
      const int src = __builtin_ctzll(__ballot(at < seq_at + incl));
      b = b0 + src;
      seq_at += __builtin_amdgcn_readlane(incl, src) - __builtin_amdgcn_readlane((int)c, src);
      seq_blocks += __builtin_amdgcn_readlane(blocks, src) - __builtin_amdgcn_readlane((int)nb, src);
      break;
    }
    seq_at += sum64;
    seq_blocks += __builtin_amdgcn_readlane(blocks, 63);
  }

  // Block by block of this workgroup's run.
  Seq seq = sequence<QN>(p, b);
  while (at < stop) {
  while (at >= seq_at + seq.blocks * seq.steps) {  // (sequences without rows take no place)
    seq_at += seq.blocks * seq.steps;
    seq_blocks += seq.blocks;
    seq = sequence<QN>(p, ++b);
  }
  const int32_t block = (at - seq_at) / seq.steps;
  if (seq_blocks + block >= p.blocks) return;  // sequences overlap: past the counters
  const int32_t block_at = seq_at + block * seq.steps;
  const int32_t row0 = block * QN, rows = seq.n * p.G, ctx = seq.ctx, kv_lim = seq.kv_lim;
  const int32_t pos0 = ctx - seq.n;  // position of the sequence's first query
  const int32_t pos_lo = pos0 + row0 / p.G, pos_hi = pos0 + (min(row0 + QN, rows) - 1) / p.G;
  const Visible vis = visible_chunks(p, kv_lim, pos_lo, pos_hi);
  const int32_t sc = vis.sc, wc0 = vis.wc0, n_vis = vis.n;
  const int32_t begin = at - block_at, end = min(min(stop - block_at, seq.steps), (n_vis + 1) >> 1);
  at = min(stop, block_at + seq.steps);

  // Q as the B operand: column r = row, k-group g; dims of product kk as the K
  // operand holds them (pages: 16 g + 8 (kk % 2) of scale group kk / 2, in
  // nibble-unpack order; fp16: 32 kk + 8 g).
  h8_t qf[QB][KK];
  int32_t row_pos[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int32_t row = row0 + 16 * qb + r, tok = row / p.G;
    row_pos[qb] = pos0 + tok;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      h8_t x = {};
      if (row < rows) {
        const int d0 = PAGES ? 64 * (kk >> 1) + 16 * g + 8 * (kk & 1) : 32 * kk + 8 * g;
        const h8_t y = __builtin_bit_cast(
            h8_t, *reinterpret_cast<const u32x4_t *>(p.q + (int64_t)(seq.start + tok) * p.q_ts +
                                                     (int64_t)(kvh * p.G + row - tok * p.G) * p.q_hs + d0));
        if (PAGES) {
          x[0] = y[0]; x[1] = y[4]; x[2] = y[1]; x[3] = y[5];
          x[4] = y[2]; x[5] = y[6]; x[6] = y[3]; x[7] = y[7];
        } else {
          x = y;
        }
      }
      qf[qb][kk] = x;
    }
  }

  f32x4_t o[QB][ND];
  float ncm[QB], thr[QB], lsum[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
    for (int i = 0; i < ND; ++i) o[qb][i] = (f32x4_t){};
    ncm[qb] = 0.0f;
    thr[qb] = -INFINITY;
    lsum[qb] = 0.0f;
  }

  // Chunk i of the visible list: logical chunk, and its byte offset in the
  // cache (chunk 0 of page 0, always mapped, if there is none).
  struct Chunk {
    int32_t lc;
    bool ok;
    int64_t kv;
  };
  const int32_t *btrow = p.bt + (int64_t)b * p.M;
  const int32_t cpp = PAGES ? 1 : p.bs >> 4;
  const int32_t nb32 = (int32_t)min(p.nb, (int64_t)INT32_MAX);
  struct Entry {  // a chunk's block-table entry, not yet waited for
    int32_t lc, page, phys;
    bool in;
  };
  auto fetch = [&](int32_t i) __attribute__((always_inline)) {
    Entry e;
    e.lc = i < sc ? i : wc0 + (i - sc);
    e.in = i < n_vis;
    e.page = cpp == 1 ? e.lc : e.lc / cpp;
    e.phys = btrow[e.in ? e.page : 0];  // n_vis > 0 here, so the row has an entry 0
    return e;
  };
  auto resolve = [&](const Entry &e) __attribute__((always_inline)) {
    Chunk c;
    c.lc = e.lc;
    c.ok = e.in && e.phys >= 0 && e.phys < nb32;
    c.kv = (int64_t)(c.ok ? e.phys : 0) * p.kv_ps + (int64_t)kvh * p.kv_hs +
           (int64_t)(c.ok ? 16 * (e.lc - e.page * cpp) : 0) * p.kv_ts;
    return c;
  };

  const Int4Page f(D);
  PackedK<D, FMT> kr;
  PackedV<D, FMT> vr;
  // K of two chunks: lane row r is tokens r % 8 and r % 8 + 8 of chunk r / 8.
  auto load_k = [&](const Chunk &ca, const Chunk &cb) __attribute__((always_inline)) {
    const int pr = r & 7;
    const uint8_t *base = p.k + (r < 8 ? ca.kv : cb.kv);
    if constexpr (PAGES) {
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        // D = 128: lane group 4 j + g of the page (16 dims of scale group j); D = 64: groups 2 g and 2 g + 1
        const int c = D == 128 ? 4 * j + g : 2 * g;
        const u32x4_t x = *reinterpret_cast<const u32x4_t *>(base + f.kcodes + (8 * pr + c) * f.BPL);
#pragma unroll
        for (int w = 0; w < 4; ++w) kr.w[4 * j + w] = x[w];
        kr.sc[j] = *reinterpret_cast<const u32x4_t *>(p.k + (g < 2 ? ca.kv : cb.kv) + f.kscales +
                                                      2 * (16 * j + 8 * (g & 1)));
      }
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          kr.w[t][kk] = *reinterpret_cast<const u32x4_t *>(base + (int64_t)(pr + 8 * t) * p.kv_ts +
                                                           2 * (32 * kk + 8 * g));
    }
  };
  // V of two chunks: lane (r, g) holds dims [D/16 r, D/16 (r + 1)) of tokens
  // p_i, p_i + 8, p_i = 4 (g % 2) + i, of chunk g / 2 (element 2 i + t).
  auto load_v = [&](const Chunk &ca, const Chunk &cb) __attribute__((always_inline)) {
    const int p0 = 4 * (g & 1);
    const int64_t cbase = g < 2 ? ca.kv : cb.kv;
    if constexpr (PAGES) {
      const uint8_t *base = p.k + cbase;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t *src = base + f.vcodes + 8 * (p0 + i) * f.BPL + (D / 16) * r;
        if constexpr (D == 128) {
          const u32x2_t x = *reinterpret_cast<const u32x2_t *>(src);
          vr.w[i][0] = x[0];
          vr.w[i][1] = x[1];
        } else {
          vr.w[i][0] = *reinterpret_cast<const uint32_t *>(src);
        }
      }
      vr.sc = *reinterpret_cast<const u32x4_t *>(base + f.vscales + 2 * ((r * (D / 16) / 64) * 16 + 2 * p0));
    } else {
      const uint8_t *base = p.v + cbase;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint8_t *src = base + (int64_t)(p0 + (e >> 1) + 8 * (e & 1)) * p.kv_ts + (D / 8) * r;
        if constexpr (D == 128) {
          const u32x4_t x = *reinterpret_cast<const u32x4_t *>(src);
#pragma unroll
          for (int j = 0; j < 4; ++j) vr.w[e][j] = x[j];
        } else {
          const u32x2_t x = *reinterpret_cast<const u32x2_t *>(src);
          vr.w[e][0] = x[0];
          vr.w[e][1] = x[1];
        }
      }
    }
  };

  const half2_t b1032 = {(half_t)1032.0f, (half_t)1032.0f}, b72 = {(half_t)72.0f, (half_t)72.0f};
  // The eight codes of a word, less 8, in nibble-unpack order (exact).
  auto codes = [&](uint32_t w) __attribute__((always_inline)) {
    const uint32_t w8 = w >> 8;
    return u32x4_t{as_u32(as_half2(bfi(0x000F000Fu, w, 0x64006400u)) - b1032),
                   as_u32(as_half2(bfi(0x00F000F0u, w, 0x54005400u)) - b72),
                   as_u32(as_half2(bfi(0x000F000Fu, w8, 0x64006400u)) - b1032),
                   as_u32(as_half2(bfi(0x00F000F0u, w8, 0x54005400u)) - b72)};
  };
  auto k_operand = [&](int t, int kk) __attribute__((always_inline)) {
    if constexpr (PAGES) {
      return __builtin_bit_cast(h8_t, codes(D == 128 ? kr.w[4 * (kk >> 1) + 2 * t + (kk & 1)] : kr.w[2 * kk + t]));
    } else {
      return __builtin_bit_cast(h8_t, kr.w[t][kk]);
    }
  };

  const half2_t ones = {(half_t)1.0f, (half_t)1.0f};
  // exp2 argument of a new maximum: probabilities lie in (0, 2^15], so fp16
  // holds those down to 2^-21 of the largest as normal numbers.
  constexpr float kTop = 7.0f;
  auto step = [&](const Chunk &ca, const Chunk &cb, const Chunk &na, const Chunk &nb_, bool more)
                  __attribute__((always_inline)) {
    f32x4_t s[QB][NG][2];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      constexpr int PG = KK / NG;  // products per sum
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const h8_t a = k_operand(t, kk);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
          s[qb][kk / PG][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              a, qf[qb][kk], kk % PG == 0 ? (f32x4_t){} : s[qb][kk / PG][t], 0, 0, 0);
      }
    }
    // exp2 arguments; element 2 i + t: token key0 + i + 8 t
    float x[QB][8];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float y = s[qb][0][e & 1][e >> 1];
        if constexpr (PAGES) {
          y *= (float)as_half2(kr.sc[0][e >> 1])[e & 1];
          if constexpr (NG == 2) y = fmaf(s[qb][1][e & 1][e >> 1], (float)as_half2(kr.sc[1][e >> 1])[e & 1], y);
        }
        x[qb][e] = fmaf(y, p.qk_scale_log2, ncm[qb]);
      }
    if (more) load_k(na, nb_);

    // Every (token, row) of the step visible: no mask (wave-uniform).
    const int32_t ta = ca.lc * 16, tb = cb.lc * 16;
    auto chunk_full = [&](const Chunk &c, int32_t t0) {
      return c.ok && t0 + 16 <= kv_lim && t0 + 15 <= pos_lo && (t0 >= pos_hi - p.W + 1 || t0 + 16 <= p.sinks);
    };
    const bool full = chunk_full(ca, ta) && chunk_full(cb, tb);
    const int32_t key0 = (g < 2 ? ta : tb) + 4 * (g & 1);
    const bool c_ok = g < 2 ? ca.ok : cb.ok;
    h8_t pf[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (!full) {
        const int32_t last = c_ok ? min(row_pos[qb], kv_lim - 1) - key0 : -1;
        const int32_t first_w = row_pos[qb] - p.W + 1 - key0, end_s = p.sinks - key0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int32_t c = (e >> 1) + 8 * (e & 1);
          x[qb][e] = (c <= last) & ((c >= first_w) | (c < end_s)) ? x[qb][e] : -INFINITY;
        }
      }
      float t = x[qb][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) t = fmaxf(t, x[qb][e]);
      if (__any(t > thr[qb])) {  // wave-uniform, rare after the first steps
        // the row's four lanes agree on the new maximum
        auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(t), __float_as_uint(t), false, false);
        t = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t), false, false);
        t = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        const bool first = thr[qb] == -INFINITY, found = t > -INFINITY;
        const float shift = first ? (found ? t - kTop : 0.0f) : fmaxf(t - kTop, 0.0f);
        const float alpha = first ? (found ? 0.0f : 1.0f) : (shift > 0.0f ? fast_exp2(-shift) : 1.0f);
        lsum[qb] *= alpha;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[qb][i] *= alpha;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[qb][e] -= shift;
        ncm[qb] -= shift;
        thr[qb] = (first && !found) ? thr[qb] : kTop + 8.0f;
      }
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[qb][e] = fast_exp2(x[qb][e]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = as_u32(half2_t{(half_t)x[qb][2 * i], (half_t)x[qb][2 * i + 1]});
        lsum[qb] = __builtin_amdgcn_fdot2(as_half2(w[i]), ones, lsum[qb], false);
      }
      pf[qb] = __builtin_bit_cast(h8_t, u32x4_t{w[0], w[1], w[2], w[3]});
    }

    // A weight of 0 must not meet an inf or NaN of V. Tokens that no row of the
    // block sees (behind the context, unlinked, outside the window) become
    // zeros; among those that only some rows see, odd values are left out
    // and added below to the rows that see them.
    bool odd = false;
    uint32_t odd_e = 0;
    if (!full) {
      const int32_t last = c_ok ? min(pos_hi, kv_lim - 1) - key0 : -1;
      const int32_t first_w = pos_lo - p.W + 1 - key0, end_s = p.sinks - key0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int32_t c = (e >> 1) + 8 * (e & 1);
        bool live = (c <= last) & ((c >= first_w) | (c < end_s));
        bool bad = false;
        if constexpr (PAGES) {  // 8 * scale past the fp16 range
          bad = ((vr.sc[e >> 1] >> (16 * (e & 1))) & 0x7FFFu) >= 0x7000u;
        } else {
          uint32_t any = 0;
#pragma unroll
          for (int j = 0; j < D / 32; ++j) any |= (vr.w[e][j] & 0x7C007C00u) + 0x04000400u;
          bad = (any & 0x80008000u) != 0;
        }
        bad = bad && live && pos_lo != pos_hi;
        odd |= bad;
        odd_e |= bad ? 1u << e : 0u;
        live = live && !bad;
        if constexpr (PAGES) {
          vr.sc[e >> 1] &= live ? ~0u : (e & 1) ? 0x0000FFFFu : 0xFFFF0000u;
        } else {
#pragma unroll
          for (int j = 0; j < D / 32; ++j) vr.w[e][j] = live ? vr.w[e][j] : 0u;
        }
      }
      odd = __any(odd);
    }
    auto pv = [&](int i, u32x4_t a) __attribute__((always_inline)) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
        o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), pf[qb], o[qb][i], 0, 0, 0);
    };
    if constexpr (PAGES) {
#pragma unroll
      for (int u = 0; u < D / 64; ++u) {
        u32x4_t y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = codes(vr.w[i][u]);
#pragma unroll
          for (int j = 0; j < 4; ++j) y[i][j] = as_u32(as_half2(y[i][j]) * as_half2(vr.sc[i]));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) pv(4 * u + j, u32x4_t{y[0][j], y[1][j], y[2][j], y[3][j]});
      }
    } else {
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        u32x4_t a;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          a[j] = __builtin_amdgcn_perm(vr.w[2 * j + 1][i >> 1], vr.w[2 * j][i >> 1], (i & 1) ? 0x07060302u : 0x05040100u);
        pv(i, a);
      }
    }
    if (odd) {
      // Token by token; a lane adds its quarter of the dims.
#pragma unroll 1
      for (int tk = 0; tk < 32; ++tk) {
        const int t = tk & 15, pp = t & 7, half = t >> 3;
        const int owner = 2 * (tk >> 4) + (pp >> 2), elem = 2 * (pp & 3) + half;  // lane group, element
        // (over pages the two scale groups of a token are odd apart from each other, so any lane of the group counts)
        if ((__ballot((odd_e >> elem) & 1) & (0xFFFFull << (16 * owner))) == 0) continue;
        const Chunk &c = tk < 16 ? ca : cb;
        const int32_t key = c.lc * 16 + t;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          float pe = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) pe = e == elem ? x[qb][e] : pe;
          pe = __shfl(pe, r + 16 * owner, 64);
          const bool see = key <= min(row_pos[qb], kv_lim - 1) &&
                           (key < p.sinks || key >= row_pos[qb] - p.W + 1);
#pragma unroll
          for (int d = 0; d < D / 4; ++d) {
            const int dim = (D / 4) * g + d;
            float y;
            bool bad;
            if constexpr (PAGES) {
              const uint8_t *blk = p.k + c.kv;
              const half_t sv = reinterpret_cast<const half_t *>(blk + f.vscales)[f.scale_idx(t, dim / 64)];
              bad = (__builtin_bit_cast(uint16_t, sv) & 0x7FFFu) >= 0x7000u;
              y = (float)(int)((blk[f.vcodes + f.v_byte(t, dim)] >> (4 * (dim & 1))) & 15) - 8.0f;
              y *= (float)sv;
            } else {
              // the whole token's row was left out on the lanes that found something odd in it
              const half_t *rowp = reinterpret_cast<const half_t *>(p.v + c.kv + (int64_t)t * p.kv_ts);
              bad = false;
#pragma unroll
              for (int z = 0; z < ND; ++z)
                bad |= (__builtin_bit_cast(uint16_t, rowp[dim / ND * ND + z]) & 0x7C00u) == 0x7C00u;
              y = (float)rowp[dim];
            }
            if (see && bad) o[qb][d % ND][d / ND] = fmaf(pe, y, o[qb][d % ND][d / ND]);
          }
        }
      }
    }
    if (more) load_v(na, nb_);
  };

  int32_t st = begin + wave;
  if (st < end) {
    Entry ea = fetch(2 * (st + NW)), eb = fetch(2 * (st + NW) + 1);
    Chunk ca = resolve(fetch(2 * st)), cb = resolve(fetch(2 * st + 1));
    load_k(ca, cb);
    load_v(ca, cb);
    for (; st < end; st += NW) {
      const Chunk na = resolve(ea), nb_ = resolve(eb);
      ea = fetch(2 * (st + 2 * NW));
      eb = fetch(2 * (st + 2 * NW) + 1);
      step(ca, cb, na, nb_, st + NW < end);
      ca = na;
      cb = nb_;
    }
  }

  // Merge of the waves. Lane (n, g) holds dims [D/4 g, D/4 (g + 1)) of row n:
  // row 4 g + reg of V^T product i is dim D/16 (4 g + reg) + i.
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float l = xor32_sum(xor16_sum(lsum[qb]));
    const int row = 16 * qb + r;
#pragma unroll
    for (int reg = 0; reg < 4; ++reg)
#pragma unroll
      for (int i = 0; i < ND; i += 4)
        *reinterpret_cast<f32x4_t *>(&s_o[wave][row][ND * (4 * g + reg) + i]) =
            f32x4_t{o[qb][i][reg], o[qb][i + 1][reg], o[qb][i + 2][reg], o[qb][i + 3][reg]};
    if (g == 0) {
      s_ml[wave][row][0] = thr[qb] == -INFINITY ? -INFINITY : -ncm[qb];
      s_ml[wave][row][1] = l;
    }
  }
  __syncthreads();
  // A block whose steps lie in one run is finished here.
  const int32_t w0 = wg_of(block_at), w1 = wg_of(block_at + seq.steps - 1), live = min(QN, rows - row0);
  auto write_row = [&](int row, int d, f32x4_t x, float l) __attribute__((always_inline)) {
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int32_t rr = row0 + row, tok = rr / p.G;
    *reinterpret_cast<u32x2_t *>(p.out + (int64_t)(seq.start + tok) * p.o_ts +
                                 (int64_t)(kvh * p.G + rr - tok * p.G) * p.o_hs + d) =
        u32x2_t{as_u32(half2_t{(half_t)(x[0] * inv), (half_t)(x[1] * inv)}),
                as_u32(half2_t{(half_t)(x[2] * inv), (half_t)(x[3] * inv)})};
  };
  // A run holds at most two blocks in part: one that began before it (slot 0),
  // one that begins in it and goes on behind it (slot 1).
  auto partial_slot = [&](int32_t w) { return ((int64_t)w * 2 + (w == w0 ? 1 : 0)) * p.Hk + kvh; };
  const int64_t mine = partial_slot(wg) * QN;
  for (int idx = tid; idx < live * (D / 4); idx += NT) {
    const int row = idx / (D / 4), d = 4 * (idx % (D / 4));
    float mx = s_ml[0][row][0];
#pragma unroll
    for (int w = 1; w < NW; ++w) mx = fmaxf(mx, s_ml[w][row][0]);
    float l = 0.0f;
    f32x4_t x = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = s_ml[w][row][0], fw = mw == -INFINITY ? 0.0f : fast_exp2(mw - mx);
      l += s_ml[w][row][1] * fw;
      x += *reinterpret_cast<const f32x4_t *>(&s_o[w][row][d]) * fw;
    }
    if (w0 == w1) {
      write_row(row, d, x, l);
    } else {
      // (agent scope: the other workgroups of the block may run on other XCDs)
      uint64_t *dst = reinterpret_cast<uint64_t *>(p.ws_o + (mine + row) * D + d);
      __hip_atomic_store(dst, __builtin_bit_cast(uint64_t, u32x2_t{__float_as_uint(x[0]), __float_as_uint(x[1])}),
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(dst + 1, __builtin_bit_cast(uint64_t, u32x2_t{__float_as_uint(x[2]), __float_as_uint(x[3])}),
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (d == 0)
        __hip_atomic_store(reinterpret_cast<uint64_t *>(p.ws_ml + 2 * (mine + row)),
                           __builtin_bit_cast(uint64_t, u32x2_t{__float_as_uint(mx), __float_as_uint(l)}),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (w0 != w1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's partial stores are complete
    __syncthreads();
    if (tid == 0) {
      uint32_t *cnt = p.ws_cnt + (int64_t)(seq_blocks + block) * p.Hk + kvh;
      const uint32_t n = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
      s_last = n == (uint32_t)(w1 - w0 + 1);
      if (s_last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (s_last) {
      // Weights of the partials, row by row (a wave per row), in s_o; the row's
      // sum in s_ml. Then each thread adds four dims of a row over them.
      auto load2 = [&](const float *src) __attribute__((always_inline)) {
        const u32x2_t u = __builtin_bit_cast(
            u32x2_t, __hip_atomic_load(reinterpret_cast<const uint64_t *>(src), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT));
        return float2{__uint_as_float(u[0]), __uint_as_float(u[1])};
      };
      const int32_t parts = w1 - w0 + 1;
      float *wgt = &s_o[0][0][0];
      constexpr int WS = NW * OS;  // weights of a row
      for (int row = wave; row < live; row += NW) {
        float mx = -INFINITY, l = 0.0f;
        for (int32_t i = lane; i < parts; i += 64) {
          const float2 ml = load2(p.ws_ml + 2 * (partial_slot(w0 + i) * QN + row));
          wgt[row * WS + i] = ml.x;
          mx = fmaxf(mx, ml.x);
        }
        mx = wave_max(mx);
        for (int32_t i = lane; i < parts; i += 64) {
          const float m = wgt[row * WS + i], f = m == -INFINITY ? 0.0f : fast_exp2(m - mx);
          wgt[row * WS + i] = f;
          l += f * load2(p.ws_ml + 2 * (partial_slot(w0 + i) * QN + row)).y;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) l += shfl_xor(l, off);
        if (lane == 0) s_ml[0][row][1] = l;
      }
      __syncthreads();
      for (int idx = tid; idx < live * (D / 4); idx += NT) {
        const int row = idx / (D / 4), d = 4 * (idx % (D / 4));
        f32x4_t x = {};
        for (int32_t i0 = 0; i0 < parts; i0 += 8) {
          float2 y[8][2];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float *src = p.ws_o + (partial_slot(w0 + min(i0 + k, parts - 1)) * QN + row) * D + d;
            y[k][0] = load2(src);
            y[k][1] = load2(src + 2);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float f = i0 + k < parts ? wgt[row * WS + i0 + k] : 0.0f;
            x += f32x4_t{y[k][0].x, y[k][0].y, y[k][1].x, y[k][1].y} * f;
          }
        }
        write_row(row, d, x, s_ml[0][row][1]);
      }
    }
  }
  __syncthreads();  // s_o and s_ml are free for the next block
  }
}

// Query rows per block: 16 where a sequence has no more than that.
struct PackedPlan {
  int32_t qn, wgs;
  int64_t blocks;  // at most this many
};

static PackedPlan packed_plan(const memopt_packed_desc &d) {
  PackedPlan pl;
  const int64_t G = d.num_heads / d.num_kv_heads, most = (int64_t)std::min(d.max_query_len, d.tokens) * G;
  pl.qn = most <= 16 ? 16 : 32;
  // sum over the sequences of ceil(rows / qn)
  pl.blocks = (d.tokens * G + (int64_t)(pl.qn - 1) * std::min(d.batch, d.tokens)) / pl.qn;
  const int64_t resident = pl.qn == 16 && (d.kv_format == MEMOPT_KV_INT4 || d.head_dim == 64) ? 3 : 2;
  pl.wgs = (int32_t)std::max<int64_t>(1, std::min<int64_t>(resident * compute_units() / d.num_kv_heads,
                                                           max_workgroups(d.head_dim)));
  return pl;
}

// Steps (32 tokens) that a block can need.
static int64_t packed_steps(const memopt_packed_desc &d) {
  return ((int64_t)d.max_blocks_per_seq * d.block_size + 31) / 32;
}

struct PackedWorkspace {
  int64_t counters, ml, total;  // bytes of the counters, offset of the (m, l) pairs
};
static PackedWorkspace packed_workspace(const memopt_packed_desc &d, const PackedPlan &pl) {
  PackedWorkspace w;
  w.counters = (pl.blocks * d.num_kv_heads * 4 + 255) / 256 * 256;
  const int64_t rows = 2LL * pl.wgs * d.num_kv_heads * pl.qn;
  w.ml = w.counters + rows * d.head_dim * 4;
  w.total = w.ml + rows * 8;
  return w;
}

static int validate_packed(const memopt_packed_desc &d) {
  MEMOPT_REQUIRE(d.tokens >= 0 && d.batch >= 0 && d.max_query_len >= 0, MEMOPT_ERR_INVALID,
                 "packed_attention: negative size");
  MEMOPT_REQUIRE(d.num_heads > 0 && d.num_kv_heads > 0 && d.num_heads % d.num_kv_heads == 0, MEMOPT_ERR_INVALID,
                 "packed_attention: num_heads must be a positive multiple of num_kv_heads");
  MEMOPT_REQUIRE(d.kv_format == MEMOPT_KV_FP16 || d.kv_format == MEMOPT_KV_INT4, MEMOPT_ERR_UNSUPPORTED,
                 "packed_attention: the cache must be an fp16 pool or INT4 pages");
  MEMOPT_REQUIRE(d.head_dim == 64 || d.head_dim == 128, MEMOPT_ERR_UNSUPPORTED,
                 "packed_attention: head_dim must be 64 or 128");
  MEMOPT_REQUIRE(d.num_kv_blocks > 0 && d.max_blocks_per_seq > 0 && d.block_size > 0, MEMOPT_ERR_INVALID,
                 "packed_attention: empty cache or block table");
  MEMOPT_REQUIRE(d.kv_format == MEMOPT_KV_FP16 ? d.block_size % 16 == 0 : d.block_size == 16, MEMOPT_ERR_UNSUPPORTED,
                 "packed_attention: pages must hold 16 tokens (fp16 pools: a multiple of 16)");
  auto aligned = [](const void *x, int64_t ts, int64_t hs) {
    return ((uintptr_t)x & 15) == 0 && ts % 8 == 0 && hs % 8 == 0;
  };
  MEMOPT_REQUIRE(aligned(d.query, d.q_token_stride, d.q_head_stride) &&
                     aligned(d.out, d.o_token_stride, d.o_head_stride) && aligned(d.key_cache, 0, 0) &&
                     aligned(d.value_cache, 0, 0) && aligned(d.workspace, 0, 0),
                 MEMOPT_ERR_INVALID, "packed_attention: rows, caches and workspace must be 16-byte aligned");
  return MEMOPT_OK;
}

template <int D, int FMT>
static void launch_packed(const PackedParams &p, int qn, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)p.wgs * p.Hk));
  if (qn == 16) hipLaunchKernelGGL((packed_kernel<D, FMT, 1>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((packed_kernel<D, FMT, 2>), grid, dim3(256), 0, stream, p);
}

}  // namespace memopt

using namespace memopt;

extern "C" int memopt_packed_workspace_size(const memopt_packed_desc *desc, int64_t *bytes, int64_t *zeroed) {
  MEMOPT_REQUIRE(desc && bytes && zeroed, MEMOPT_ERR_INVALID, "packed_workspace_size: null pointer");
  *bytes = *zeroed = 0;
  int rc = validate_packed(*desc);
  if (rc != MEMOPT_OK || desc->tokens == 0 || desc->batch == 0 || desc->max_query_len == 0) return rc;
  const PackedWorkspace w = packed_workspace(*desc, packed_plan(*desc));
  *bytes = w.total;
  *zeroed = w.counters;
  return MEMOPT_OK;
}

extern "C" int memopt_packed_attention(const memopt_packed_desc *desc, void *stream) {
  MEMOPT_REQUIRE(desc, MEMOPT_ERR_INVALID, "packed_attention: null descriptor");
  const memopt_packed_desc &d = *desc;
  int rc = validate_packed(d);
  if (rc != MEMOPT_OK || d.tokens == 0 || d.batch == 0 || d.max_query_len == 0) return rc;
  MEMOPT_REQUIRE(d.query && d.out && d.key_cache && (d.value_cache || d.kv_format == MEMOPT_KV_INT4) &&
                     d.block_tables && d.context_lens && d.query_starts,
                 MEMOPT_ERR_INVALID, "packed_attention: null pointer");
  const PackedPlan pl = packed_plan(d);
  const PackedWorkspace w = packed_workspace(d, pl);
  MEMOPT_REQUIRE(d.workspace && d.workspace_bytes >= w.total, MEMOPT_ERR_INVALID,
                 "packed_attention: workspace needs " + std::to_string(w.total) + " bytes");
  MEMOPT_REQUIRE((int64_t)d.tokens * d.num_heads < (1LL << 31) && pl.blocks * packed_steps(d) < (1LL << 31),
                 MEMOPT_ERR_UNSUPPORTED, "packed_attention: too many (row, page) pairs for one call");
  PackedParams p = {};
  p.q = (const half_t *)d.query;
  p.out = (half_t *)d.out;
  p.q_ts = d.q_token_stride;
  p.q_hs = d.q_head_stride;
  p.o_ts = d.o_token_stride;
  p.o_hs = d.o_head_stride;
  p.cu = d.query_starts;
  p.ctx = d.context_lens;
  p.bt = d.block_tables;
  p.T = d.tokens;
  p.B = d.batch;
  p.Hq = d.num_heads;
  p.Hk = d.num_kv_heads;
  p.G = d.num_heads / d.num_kv_heads;
  p.M = d.max_blocks_per_seq;
  p.bs = d.block_size;
  p.nb = d.num_kv_blocks;
  p.k = (const uint8_t *)d.key_cache;
  p.v = (const uint8_t *)d.value_cache;
  if (d.kv_format == MEMOPT_KV_INT4) {
    p.kv_hs = Int4Page(d.head_dim).block;
    p.kv_ps = d.num_kv_heads * p.kv_hs;
  } else {
    p.kv_hs = 2 * d.head_dim;
    p.kv_ts = d.num_kv_heads * p.kv_hs;
    p.kv_ps = d.block_size * p.kv_ts;
  }
  p.W = std::min(effective_window(d.window_size, d.max_seq_len), 1 << 30);  // (position - W stays in 32 bits)
  p.sinks = std::max(0, d.num_sink_tokens);
  p.qk_scale_log2 = 1.4426950408889634f / sqrtf((float)d.head_dim);
  p.wgs = pl.wgs;
  p.blocks = (int32_t)pl.blocks;
  p.ws_cnt = (uint32_t *)d.workspace;
  p.ws_o = (float *)((uint8_t *)d.workspace + w.counters);
  p.ws_ml = (float *)((uint8_t *)d.workspace + w.ml);
  hipStream_t s = (hipStream_t)stream;
  if (d.head_dim == 128) {
    if (d.kv_format == MEMOPT_KV_INT4) launch_packed<128, MEMOPT_KV_INT4>(p, pl.qn, s);
    else launch_packed<128, MEMOPT_KV_FP16>(p, pl.qn, s);
  } else {
    if (d.kv_format == MEMOPT_KV_INT4) launch_packed<64, MEMOPT_KV_INT4>(p, pl.qn, s);
    else launch_packed<64, MEMOPT_KV_FP16>(p, pl.qn, s);
  }
  return check_launch("packed_attention");
}
