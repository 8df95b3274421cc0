// latent.hip — attention over a paged cache that holds one vector per token
// for all heads (gfx950 matrix cores), and the writer of that cache.
//
// A cached row c_j has R latent elements and P rotary ones. With queries that
// carry the key projection already (q = [W_k^T q_nope, q_rope], R + P wide):
//   o_rh = sum_j softmax_j(scale q_rh . c_j) c_j[0 .. R)
// over the keys that packed_attention would show row r. So all heads share
// keys and values, the values are part of the keys, and a sequence's rows are
// its tokens times its heads.
//
// A tile of 64 rows c_j is read once into LDS and used twice: as 32 x 16 key
// operands (rows) and, through transposed reads, as value operands (columns).
// Rows of queries are the columns of both products, so a row's softmax stays
// in its lane, and the weights leave one product in the layout in which the
// other takes them. One pass with a running maximum and sum.
//
// Measured (rank 512 + 64, bf16): 32 single tokens of 16 heads over up to 8192
// tokens: 60 us with the merge's 6, 3.9 TB/s of rows read once (the copies
// without the arithmetic: 41-48). 16 single tokens of 128 heads: 63-66 us with
// the merge's 9: each 64-row tile reads all keys, so a head count of 128 reads them
// twice. Three chunks of 256 tokens, 16 heads, beside nine single tokens: 171-195
// us with the merge's 13, 0.71 PFLOP/s: of a tile's 6400 clocks the first
// product takes 2900 (1152 of matrix instructions, the rest the issue of
// copies and operand reads), the softmax 500, the second product 1850 (1024),
// barriers and the next tile's pages 1100. write_latent: a launch (2 us) up to
// some 2048 tokens, 12.7 us for 32768 (150 MB, partly from the last-level cache).
#include <algorithm>
#include <cmath>

#include "lds_dma.hpp"
#include "tiles.hpp"

namespace memopt {

typedef float f32x2m_t __attribute__((ext_vector_type(2)));

struct LatentParams {
  const uint16_t *q, *c;
  uint16_t *out;
  int64_t q_ts, q_hs, o_ts, o_hs;
  const int32_t *bt, *ctx, *starts;
  int64_t nb, page_bytes;
  int32_t T, B, H, M, W, sinks;
  int32_t max_keys;  // tokens that are looked at
  int32_t max_n;     // query tokens of a sequence
  int32_t span;      // tokens that a tile of rows can touch
  Divisor by_h, by_chunks;  // by_chunks: 16-token chunks of a page
  float scale_log2;
  int32_t wgs;
  float *ws_o;    // [wgs][2][rows][R]
  float2 *ws_ml;  // [wgs][2][rows]
};

// The call's work is a list of steps: for each sequence, for each tile of its
// rows, its key tiles. Workgroup w takes steps [w run, (w + 1) run), so that
// all end together whatever the lengths; a tile of rows whose steps fall to
// more than one workgroup leaves partial sums, merged by the second launch.
static constexpr int kLatentKeys = 64;

struct LatentSeq {
  int32_t start, rows, pos0, len;
  int32_t tiles, steps;  // tiles of rows; steps of each
};
template <int ROWS>
__device__ __forceinline__ LatentSeq latent_seq(const LatentParams &p, int32_t b) {
  const Rows r = rows_of(p.starts, p.T, b);
  const int32_t ctx = p.ctx[b], n = min(r.n, p.max_n);
  LatentSeq s = {r.start, n * p.H, ctx - r.n, max(0, min(ctx, p.max_keys)), 0, 0};
  s.tiles = (s.rows + ROWS - 1) / ROWS;
  const int32_t all = (s.len + kLatentKeys - 1) / kLatentKeys;
  const int32_t sink = (min(p.sinks, s.len) + kLatentKeys - 1) / kLatentKeys;
  s.steps = max(1, min(all, sink + (p.W + p.span + kLatentKeys) / kLatentKeys + 1));
  return s;
}
// The same for a wave-uniform b, in scalar registers.
template <int ROWS>
__device__ __forceinline__ LatentSeq uniform_seq(const LatentParams &p, int32_t b) {
  LatentSeq s = latent_seq<ROWS>(p, b);
  for (int32_t *x : {&s.start, &s.rows, &s.pos0, &s.len, &s.tiles, &s.steps}) *x = __builtin_amdgcn_readfirstlane(*x);
  return s;
}

// Where step `at` of the list lies; total: all steps. Every lane returns the same.
struct LatentPlace {
  int32_t b;
  uint32_t before;  // steps of the sequences before b
  uint32_t total, units_before;
};
template <int ROWS, bool BY_UNIT>
__device__ __forceinline__ LatentPlace latent_place(const LatentParams &p, uint32_t at, bool only_total) {
  const int lane = threadIdx.x & 63;
  LatentPlace r = {-1, 0, 0, 0};
  uint32_t sum = 0, units = 0;
  for (int32_t b0 = 0; b0 < p.B; b0 += 64) {
    const int32_t b = b0 + lane;
    uint32_t n = 0, u = 0;
    if (b < p.B) {
      const LatentSeq s = latent_seq<ROWS>(p, b);
      u = (uint32_t)s.tiles;
      n = u * (uint32_t)s.steps;
    }
    const uint32_t end = wave_scan(n), uend = wave_scan(u);
    const bool here = BY_UNIT ? units + uend > at : sum + end > at;
    const uint64_t m = only_total ? 0 : __ballot(here);
    if (r.b < 0 && m) {
      const int src = __builtin_ctzll(m);
      r.b = b0 + src;
      r.before = sum + __builtin_amdgcn_readlane(end - n, src);
      r.units_before = units + __builtin_amdgcn_readlane(uend - u, src);
      if (!BY_UNIT) return r;
    }
    sum += __builtin_amdgcn_readlane(end, 63);
    units += __builtin_amdgcn_readlane(uend, 63);
  }
  r.total = sum;
  return r;
}
__device__ __forceinline__ uint32_t latent_run(uint32_t total, int32_t wgs) {
  return max(1u, (total + (uint32_t)wgs - 1) / (uint32_t)wgs);
}

// Two waves share 32 rows: in the first product each takes 32 of a tile's keys,
// in the second half of the latent's columns, over all keys, so that a wave
// holds (R + P) / 4 operand and R / 4 accumulator registers (272 at 512 +
// 64; a wave with whole rows would need 400 and spills). Between the products
// they exchange their keys' maxima and weights through LDS. RW such pairs.
template <int R, int P, int RW>
struct LatentLds {
  static constexpr int tiles = 2 * 4 * 16 * 2 * (R + P);   // two tiles of 64 keys
  static constexpr int weights = tiles, tops = weights + RW * 2 * 2048, bytes = tops + RW * 2 * 128;
};
template <class E, int R, int P, int RW>
__global__ __launch_bounds__(RW * 128) __attribute__((amdgpu_waves_per_eu(1, 1))) void latent_kernel(const LatentParams p) {
  constexpr int W = R + P, RB = 2 * W, NCH = W / 16, NDB = R / 64, NW = 2 * RW, ROWS = 32 * RW;
  constexpr int CB = 16 * RB, NCOPY = CB / 1024, CPW = 4 / NW;  // a 16-token chunk's bytes and copies; chunks per wave
  constexpr int BUF = 4 * CB;
  using L = LatentLds<R, P, RW>;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, n = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave / 2, kw = wave % 2;
  // Workgroup i runs on XCD i % 8: an XCD takes neighbouring runs, whose tiles of rows read the same keys.
  const uint32_t w = (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
  const uint32_t total = latent_place<ROWS, false>(p, 0, true).total, run = latent_run(total, p.wgs);
  const uint32_t begin = w * run;
  uint32_t end = min(total, begin + run);  // of the steps that are left
  if (begin >= end) return;
  // A run's tiles of rows from the last back: its first keys, then others' last ones. Workgroups that begin together
  // so meet the same keys together, in their XCD's L2.
  const LatentPlace place = latent_place<ROWS, false>(p, end - 1, false);
  if (place.b < 0) return;
  int32_t b = __builtin_amdgcn_readfirstlane(place.b);
  uint32_t before = __builtin_amdgcn_readfirstlane(place.before);

  // LDS rows are the 64 keys; their 16-byte pieces are swizzled by bits of the
  // row, within groups of four, so that neither the reads of one piece of
  // eight rows nor those of 32 bytes of four rows meet a bank twice (rows are
  // 32 banks apart where R + P is an odd multiple of 64).
  auto swz = [](int row) { return 2 * ((row >> 1) & 1) + ((row >> 2) & 1); };
  // (copies of the chunk's second eight rows, where they begin a copy, differ from those of the first by an offset)
  constexpr int NOFF = NCOPY % 2 ? NCOPY : NCOPY / 2, PAIRS = (NOFF + 1) / 2;
  uint32_t off[NOFF];
#pragma unroll
  for (int c = 0; c < NOFF; ++c) {
    const int piece = c * 64 + lane, row = piece / (RB / 16), j = piece % (RB / 16);
    off[c] = row * RB + 16 * (j ^ swz(row)) - c % 2 * 1024;  // (of a pair, the second)
  }
  uint32_t ka[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) ka[c] = n * RB + 16 * ((2 * c + hl) ^ swz(n));
  const int i16 = lane & 15, vrow = 4 * hl + (i16 >> 2);
  const uint32_t va = vrow * RB + 16 * ((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ swz(vrow)) + 8 * (i16 & 1) + 64 * NDB * kw;
  u32x4p_t *const s_weights = reinterpret_cast<u32x4p_t *>(lds + L::weights) + rw * 256 + lane;  // [half][register quad][lane]
  float *const s_tops = reinterpret_cast<float *>(lds + L::tops) + rw * 64;                      // [half][row]

  while (begin < end) {
    LatentSeq s = uniform_seq<ROWS>(p, b);
    while (before >= end) {
      if (--b < 0) return;  // (sequences that overlap: their steps may pass 32 bits)
      s = uniform_seq<ROWS>(p, b);
      before -= (uint32_t)s.tiles * (uint32_t)s.steps;
    }
    const int32_t rt = (int32_t)((end - 1 - before) / (uint32_t)s.steps);
    const uint32_t unit = before + (uint32_t)rt * (uint32_t)s.steps, at = max(begin, unit);
    const int32_t first_step = (int32_t)(at - unit), last_step = (int32_t)(end - unit);
    const int32_t q0 = ROWS * rt, qw0 = q0 + 32 * rw;
    auto pos_of = [&](int32_t row) { return s.pos0 + p.by_h(min(row, s.rows - 1)); };

    // Key tiles of the tile of rows: sinks, then the window.
    const int32_t hi = max(0, min(s.len, pos_of(q0 + ROWS - 1) + 1));
    const int32_t sink_tiles = (min(p.sinks, hi) + kLatentKeys - 1) / kLatentKeys;
    const int32_t t_first = max(max(0, pos_of(q0) - p.W + 1) / kLatentKeys, sink_tiles);
    const int32_t n_tiles = sink_tiles + max(0, (hi + kLatentKeys - 1) / kLatentKeys - t_first);
    const int32_t i0 = min(first_step, n_tiles), i1 = min(last_step, n_tiles);
    auto tile_base = [&](int32_t it) { return (it < sink_tiles ? it : t_first + (it - sink_tiles)) * kLatentKeys; };

    // Block-table entries of the 64 chunks of 16 tiles from `it` on, one a lane; -1 behind the context or the last tile.
    // (Scalar loads would be waited for with every LDS read: 2000 clocks and more a tile.)
    auto entries_of = [&](int32_t it) __attribute__((always_inline)) {
      const int32_t t = it + (lane >> 2), key = tile_base(t) + 16 * (lane & 3);
      return t < i1 && key < s.len ? p.bt[(int64_t)b * p.M + p.by_chunks(key >> 4)] : -1;
    };
    int32_t entries = entries_of(i0), entries_next = -1;

    u32x4p_t qf[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) qf[c] = (u32x4p_t){};
    if (qw0 + n < s.rows) {
      const int32_t tok = p.by_h(qw0 + n);
      const uint16_t *src = p.q + (int64_t)(s.start + tok) * p.q_ts + (int64_t)(qw0 + n - tok * p.H) * p.q_hs + 8 * hl;
#pragma unroll
      for (int c = 0; c < NCH; ++c) qf[c] = *reinterpret_cast<const u32x4p_t *>(src + 16 * c);
    }
    // Waited for here: the first product would wait for them, and with them for every copy before, in each iteration.
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __builtin_amdgcn_sched_barrier(0);

    // They live in accumulation registers, where matrix instructions take operands from; the sums, which a new maximum
    // scales, in the others. (A hint: without it some of them move about in the loop, 213 against 197 us for chunks.)
#pragma unroll
    for (int c = 0; c < NCH; ++c) asm volatile("" : "+a"(qf[c]));

    // A tile's copies are set up together (of nothing, where no tile follows) and issued in pairs between the matrix
    // instructions of the tile before: all at once they keep a wave waiting for the queue (3400 of a tile's 9000 clocks).
    // An entry that is no page, and rows behind the context, read as zeros.
    auto pages_of = [&](int32_t e) { return __ballot(e >= 0 && e < p.nb); };
    uint64_t linked = pages_of(entries);  // of the lanes
    uint32_t link_next = 0;               // bit g: chunk g is there
    __amdgpu_buffer_rsrc_t next[CPW];
    constexpr int N = NCOPY / NOFF * PAIRS * CPW;
    auto prepare = [&](int32_t it) __attribute__((always_inline)) {
      const int32_t first = 4 * ((it - i0) & 15);
      link_next = (uint32_t)(linked >> first) & 15;
#pragma unroll
      for (int i = 0; i < CPW; ++i) {
        const int g = wave * CPW + i;
        const int32_t e = __builtin_amdgcn_readlane(entries, first + g);
        const bool there = (link_next >> g) & 1;
        const int32_t key = tile_base(it) + 16 * g, chunk = key >> 4;
        const uint8_t *base = reinterpret_cast<const uint8_t *>(p.c) + (there ? (int64_t)e : 0) * p.page_bytes +
                              (int64_t)(chunk - p.by_chunks(chunk) * (int32_t)p.by_chunks.d) * CB;
        next[i] = uniform_rsrc(base, there ? max(0, min(16, s.len - key)) * RB : 0);
      }
    };
    auto issue = [&](int buf, int from, int to) __attribute__((always_inline)) {  // pairs of copies [from, to) of N
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (k < from || k >= to) continue;
        const int i = k * CPW / N, half = k / PAIRS % (NCOPY / NOFF), c = 2 * (k % PAIRS);
        const uint32_t to_lds = lds_u32(lds) + buf * BUF + (wave * CPW + i) * CB + (half * NOFF + c) * 1024;
        if (c + 1 < NOFF) lds_dma<0, 2>(next[i], to_lds, off + c, half * 8 * RB);
        else lds_dma<0, 1>(next[i], to_lds, off + c, half * 8 * RB);
      }
    };

    f32x16_t o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[db] = (f32x16_t){};
    // x = scale_log2 s + ncm is the exp2 argument; a new maximum lands at kTop
    // and the next rescale comes past kTop + 8 (prompt.hip).
    constexpr float kTop = E::kTop;
    float ncm = 0.0f, thr = -INFINITY, lsum = 0.0f;
    bool odd = false;  // a tile of this part held inf or NaN that was made finite
    const bool any = qw0 < s.rows;
    const int32_t pos_first = pos_of(qw0), pos_last = pos_of(qw0 + 31);
    // Whether all this wave's rows see the 32 keys from k0 on; whether any sees one.
    auto full = [&](int32_t k0, uint32_t link) {
      return qw0 + 31 < s.rows && k0 + 31 <= pos_first && k0 + 32 <= s.len && link == 3u &&
             (k0 > pos_last - p.W || k0 + 32 <= p.sinks);
    };
    auto seen = [&](int32_t k0) {
      return any && k0 <= pos_last && k0 < s.len && (k0 + 32 > pos_first - p.W + 1 || k0 < p.sinks);
    };
    auto lane_row = [&]() { return qw0 + n; };

    // Scores of this wave's 32 keys, in log2 units, hidden ones -inf.
    constexpr int NSC = (2 * N + 2) / 3;  // copies beside the first product; the others go beside the second
    auto scores = [&](const uint8_t *kt, int32_t k0, uint32_t link, int next_buf, f32x16_t &x) __attribute__((always_inline)) {
      x = (f32x16_t){};
      // Operands are read a group of products ahead: a wave has its SIMD to itself and nothing else hides an LDS read.
      constexpr int GR = 4, NG = (NCH + GR - 1) / GR;
      u32x4p_t f[2][GR];
      auto read = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < GR; ++i)
          if (g * GR + i < NCH)
            f[g & 1][i] = *reinterpret_cast<const u32x4p_t *>(kt + ka[i & 1] + 64 * ((g * GR + i) >> 1));
      };
      read(0);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        __builtin_amdgcn_sched_barrier(0);
        if (g + 1 < NG) read(g + 1);
        __builtin_amdgcn_sched_barrier(0);
        issue(next_buf, NSC * g / NG, NSC * (g + 1) / NG);
#pragma unroll
        for (int i = 0; i < GR; ++i)
          if (g * GR + i < NCH) x = E::mfma(f[g & 1][i], qf[g * GR + i], x);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], p.scale_log2, ncm);
      if (full(k0, link)) return;
      const int32_t row = lane_row(), qp = pos_of(row), key0 = k0 + 4 * hl;
      const int32_t last = row < s.rows ? min(qp, s.len - 1) - key0 : -1;
      const int32_t first = qp - p.W + 1 - key0, sink = p.sinks - key0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int32_t stop = (link >> half) & 1 ? last : -1;
#pragma unroll
        for (int r = 8 * half; r < 8 * half + 8; ++r) {
          const int32_t k = 8 * (r >> 2) + (r & 3);
          x[r] = (k <= stop) & ((k >= first) | (k < sink)) ? x[r] : -INFINITY;
        }
      }
    };
    // A maximum t of the pair's 64 keys: both waves come to the same reference.
    auto raise_max = [&](float t, f32x16_t &x) __attribute__((always_inline)) {
      if (!__any(t > thr)) return;
      const bool start = thr == -INFINITY, found = t > -INFINITY;
      const float shift = start ? (found ? t - kTop : 0.0f) : fmaxf(t - kTop, 0.0f);
      if (__any(!start && shift > 0.0f)) {
        const float alpha = start ? 1.0f : fast_exp2(-shift);  // (nothing summed before the start)
        lsum *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] -= shift;
      ncm -= shift;
      thr = (start && !found) ? thr : kTop + 8.0f;
    };
    // Values of 16 keys and 32 columns, transposed by the read.
    auto values = [&](const uint8_t *kt, int db, int i) __attribute__((always_inline)) {
      const uint8_t *src = kt + va + 64 * db + 16 * i * RB;
      const u32x2p_t a = v_read(src, 0), b8 = v_read(src + 8 * RB, 0);
      return u32x4p_t{a[0], a[1], b8[0], b8[1]};
    };
    // `first`: the values of the first 32 columns, read before the weights were there.
    auto add_values = [&](const uint8_t *kt, const u32x4p_t (&pb)[4], const u32x4p_t (&first)[4],
                          int next_buf) __attribute__((always_inline)) {
      constexpr int G = (3 * NDB + 3) / 4;  // (none in the last quarter: they have to arrive)
      u32x4p_t v[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[0][i] = first[i];
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (db + 1 < NDB) v[(db + 1) & 1][i] = values(kt, db + 1, i);
        __builtin_amdgcn_sched_barrier(0);
        if (db < G) issue(next_buf, NSC + (N - NSC) * db / G, NSC + (N - NSC) * (db + 1) / G);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[db] = E::mfma(v[db & 1][i], pb[i], o[db]);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // A weight of 0 must not meet an inf or NaN. Where a tile has a token that
    // some row of the workgroup does not see, such values become finite in LDS
    // (after all scores were taken), and rows that do see one get it at the end.
    const int32_t group_first = pos_of(q0), group_last = pos_of(q0 + ROWS - 1);
    auto hides = [&](int32_t tb) {
      return min(tb + kLatentKeys, s.len) - 1 > group_first || (tb <= group_last - p.W && tb + kLatentKeys > p.sinks);
    };
    auto tame_tile = [&](uint8_t *kt) __attribute__((always_inline)) {
      uint32_t changed = 0;
#pragma unroll 1
      for (int i = threadIdx.x; i < kLatentKeys * (R / 8); i += 64 * NW) {
        const int row = i / (R / 8), j = i % (R / 8);
        u32x4p_t *const at = reinterpret_cast<u32x4p_t *>(kt + row * RB + 16 * (j ^ swz(row)));
        u32x4p_t v = *at;
        uint32_t odd = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = tame<E>(v[k], odd);
        if (odd) *at = v;
        changed |= odd;
      }
      return changed;
    };

    if (i0 < i1) {
      prepare(i0);
      issue(0, 0, N);
    }
    for (int32_t it = i0; it < i1; ++it) {
      const int buf = (it - i0) & 1;
      // This wave's copies of the tile have arrived; the barrier says so for all.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      const uint32_t link = link_next;
      if (((it + 1 - i0) & 15) == 0) {
        entries = entries_next;
        linked = pages_of(entries);
      }
      prepare(it + 1);
      if (((it + 2 - i0) & 15) == 0) entries_next = entries_of(it + 2);
      const int32_t tb = tile_base(it), k0 = tb + 32 * kw;
      const uint8_t *const kt = lds + buf * BUF;
      const bool some = seen(tb) || seen(tb + 32);  // (the same for both waves of the pair)
      f32x16_t x;
      if (some) {
        scores(kt + 2 * kw * CB, k0, (link >> (2 * kw)) & 3, buf ^ 1, x);
        float t = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) t = fmaxf(t, x[r]);
        t = both_halves_max(t);
        if (hl == 0) s_tops[32 * kw + n] = t;
      } else {
        issue(buf ^ 1, 0, N);
      }
      __syncthreads();
      u32x4p_t pb[4], first[4];
      if (some) {
        raise_max(fmaxf(s_tops[n], s_tops[32 + n]), x);
        // Weights enter the second product in 16 bits, and so the row's sum. With what the rounding leaves as a second
        // operand the result's error would be its own rounding alone (bf16 1.65e-3 for 1.91e-3, fp16 2.07e-4 for
        // 2.27e-4 of its norm), for 64 instead of 60 us (32 single tokens), and 64-row tiles have no LDS for it.
        u32x4p_t mine[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[i >> 2][i & 3] = E::pack(fast_exp2(x[2 * i]), fast_exp2(x[2 * i + 1]));
#pragma unroll
        for (int i = 0; i < 8; ++i) lsum = E::dot2(mine[i >> 2][i & 3], E::kOnes, lsum);
#pragma unroll
        for (int i = 0; i < 2; ++i) s_weights[128 * kw + 64 * i] = mine[i];
      }
      if (hides(tb)) odd |= __syncthreads_or((int)tame_tile(lds + buf * BUF)) != 0;
      if (some) {
#pragma unroll
        for (int i = 0; i < 4; ++i) first[i] = values(kt, 0, i);
      }
      __syncthreads();
      if (some) {
#pragma unroll
        for (int i = 0; i < 4; ++i) pb[i] = s_weights[64 * i];
        add_values(kt, pb, first, buf ^ 1);
      }
      __syncthreads();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the last tile's copies of nothing)

    // The pair's row sums.
    float l = xor32_sum(lsum);
    if (hl == 0) s_tops[32 * kw + n] = l;
    __syncthreads();
    l = s_tops[n] + s_tops[32 + n];
    // (a part without a maximum is left out of the merge, unless all it has is NaN)
    const float m = thr == -INFINITY && l == 0.0f ? -INFINITY : -ncm;
    const int32_t row = lane_row();
    if (first_step == 0 && last_step == s.steps) {
      if (row < s.rows) {
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        const int32_t tok = p.by_h(row);
        uint16_t *dst = p.out + (int64_t)(s.start + tok) * p.o_ts + (int64_t)(row - tok * p.H) * p.o_hs + 4 * hl + 32 * NDB * kw;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<u32x2p_t *>(dst + 32 * db + 8 * g) =
                u32x2p_t{E::pack(o[db][4 * g] * inv, o[db][4 * g + 1] * inv),
                         E::pack(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv)};
      }
    } else if (row < s.rows) {
      const int64_t slot = ((int64_t)w * 2 + (at == begin ? 0 : 1)) * ROWS + 32 * rw + n;
      if (hl == 0 && kw == 0) p.ws_ml[slot] = float2{m, l};
      float *dst = p.ws_o + slot * R + 4 * hl + 32 * NDB * kw;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4p_t *>(dst + 32 * db + 8 * g) =
              f32x4p_t{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
    }
    if (odd && row < s.rows) {
      // Rows that see an inf or NaN that was made finite have it in that column whatever its weight.
      const int32_t qp = pos_of(row), tok = p.by_h(row);
      const bool direct = first_step == 0 && last_step == s.steps;
      uint16_t *const out = p.out + (int64_t)(s.start + tok) * p.o_ts + (int64_t)(row - tok * p.H) * p.o_hs;
      float *const part = p.ws_o + (((int64_t)w * 2 + (at == begin ? 0 : 1)) * ROWS + 32 * rw + n) * R;
#pragma unroll 1
      for (int32_t it = i0; it < i1; ++it) {
        const int32_t tb = tile_base(it);
        if (!hides(tb)) continue;
#pragma unroll 1
        for (int32_t key = tb; key < min(tb + kLatentKeys, s.len); ++key) {
          const int32_t chunk = key >> 4, e = p.bt[(int64_t)b * p.M + p.by_chunks(chunk)];
          if (e < 0 || e >= p.nb || key > qp || (key >= p.sinks && key <= qp - p.W)) continue;
          const uint16_t *src = reinterpret_cast<const uint16_t *>(
              reinterpret_cast<const uint8_t *>(p.c) + (int64_t)e * p.page_bytes +
              (int64_t)(chunk - p.by_chunks(chunk) * (int32_t)p.by_chunks.d) * CB + (key & 15) * RB);
#pragma unroll 1
          for (int i = 0; i < 16 * NDB; ++i) {
            const int d = 32 * NDB * kw + 8 * (i >> 2) + 4 * hl + (i & 3);
            const uint16_t bits = src[d];
            if ((bits & E::kExponent) != E::kExponent) continue;
            if (direct) out[d] = (uint16_t)E::pack(E::value(out[d]) + E::value(bits), 0.0f);
            else part[d] += E::value(bits);
          }
        }
      }
    }
    end = at;
    __syncthreads();  // the space is free for the next tiles
  }
}

// Rows whose steps fell to more than one workgroup: a wave per row.
template <class E, int R, int ROWS>
__global__ __launch_bounds__(256) void latent_merge_kernel(const LatentParams p) {
  constexpr int PER = R / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t unit = blockIdx.x / (ROWS / 4);
  const int32_t r = (int32_t)(blockIdx.x % (ROWS / 4)) * 4 + wave;
  const LatentPlace place = latent_place<ROWS, true>(p, unit, false);
  if (place.b < 0) return;
  const LatentSeq s = uniform_seq<ROWS>(p, place.b);
  const int32_t rt = (int32_t)(unit - place.units_before), row = rt * ROWS + r;
  if (row >= s.rows) return;
  const uint32_t run = latent_run(place.total, p.wgs), s0 = place.before + (uint32_t)rt * (uint32_t)s.steps;
  const uint32_t w0 = s0 / run, w1 = (s0 + (uint32_t)s.steps - 1) / run;
  if (w0 == w1) return;
  // The first of them began the unit behind its run's begin, or with it.
  auto slot_of = [&](uint32_t w) { return ((int64_t)w * 2 + (w == w0 && s0 != w * run ? 1 : 0)) * ROWS + r; };
  // Maxima and sums 64 parts at a time, one per lane; then the parts' rows, four reads in flight.
  const uint32_t parts = w1 - w0 + 1;
  float top = -INFINITY, l = 0.0f, acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
  for (uint32_t i0 = 0; i0 < parts; i0 += 64)
    top = fmaxf(top, i0 + lane < parts ? p.ws_ml[slot_of(w0 + i0 + lane)].x : -INFINITY);
  top = wave_max(top);
  for (uint32_t i0 = 0; i0 < parts; i0 += 64) {
    const float2 ml = i0 + lane < parts ? p.ws_ml[slot_of(w0 + i0 + lane)] : float2{-INFINITY, 0.0f};
    // A part of a maximum of -inf saw nothing, and its row may hold anything. Every other part counts, also where its
    // factor is 0: 0 times the NaN or inf that it may hold is the row's NaN.
    const bool seen = ml.x != -INFINITY;
    const uint64_t parts_seen = __ballot(seen);
    const float f = seen ? fast_exp2(ml.x - top) : 0.0f;
    l += seen ? ml.y * f : 0.0f;
    const uint32_t n = min(64u, parts - i0);
    for (uint32_t i = 0; i < n; i += 4) {
      f32x4p_t v[4][PER / 4 ? PER / 4 : 1];
      f32x2m_t v2[4];
      float g[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t j = min(i + k, n - 1);
        g[k] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), j));
        const float *src = p.ws_o + slot_of(w0 + i0 + j) * R + lane * PER;
        if constexpr (PER == 2) v2[k] = *reinterpret_cast<const f32x2m_t *>(src);
        else
#pragma unroll
          for (int x = 0; x < PER / 4; ++x) v[k][x] = *reinterpret_cast<const f32x4p_t *>(src + 4 * x);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (i + k >= n || !((parts_seen >> (i + k)) & 1)) continue;
#pragma unroll
        for (int x = 0; x < PER; ++x) {
          if constexpr (PER == 2) acc[x] = fmaf(v2[k][x], g[k], acc[x]);
          else acc[x] = fmaf(v[k][x / 4][x & 3], g[k], acc[x]);
        }
      }
    }
  }
  l += xor1(l);
  l += xor2(l);
  l += half_mirror(l);
  l += dpp_f32<0x140>(l);
  l = xor32_sum(xor16_sum(l));
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  const int32_t tok = p.by_h(row);
  uint32_t *dst = reinterpret_cast<uint32_t *>(p.out + (int64_t)(s.start + tok) * p.o_ts + (int64_t)(row - tok * p.H) * p.o_hs +
                                               lane * PER);
#pragma unroll
  for (int i = 0; i < PER / 2; ++i) dst[i] = E::pack(acc[2 * i] * inv, acc[2 * i + 1] * inv);
}

// Rows into their slots, 16 bytes a thread.
struct WriteLatentParams {
  const uint16_t *latents, *rope;
  uint16_t *cache;
  int64_t l_ts, r_ts, slots_in_cache;
  const int32_t *slots;
  int32_t T, R, P;
  Divisor by_pieces;
};
__global__ __launch_bounds__(256) void write_latent_kernel(const WriteLatentParams p) {
  const int32_t pieces = (p.R + p.P) / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)p.T * pieces; i += (int64_t)gridDim.x * 256) {
    const int32_t t = p.by_pieces((int32_t)i), j = 8 * ((int32_t)i - t * pieces);
    const int32_t slot = p.slots[t];
    if (slot < 0 || slot >= p.slots_in_cache) continue;
    const uint16_t *src = j < p.R ? p.latents + t * p.l_ts + j : p.rope + t * p.r_ts + (j - p.R);
    *reinterpret_cast<u32x4p_t *>(p.cache + (int64_t)slot * (p.R + p.P) + j) = *reinterpret_cast<const u32x4p_t *>(src);
  }
}

struct LatentPlan {
  int rows;  // query rows of a tile
  int32_t wgs;
  int64_t ml, total;  // offset of ws_ml; bytes
};
static int64_t latent_keys(const memopt_latent_desc &d) {
  return std::min<int64_t>((int64_t)d.max_blocks_per_seq * d.block_size, std::max(0, d.max_seq_len));
}
static LatentPlan latent_plan(const memopt_latent_desc &d) {
  LatentPlan pl = {};
  const int64_t most = (int64_t)std::min(d.max_query_len, d.tokens) * d.num_heads;
  // Tiles of 32 rows leave room for two workgroups on a compute unit at rank 128 (single tokens of 8 to 32 heads take 0.71
  // to 0.95 of the time with 64) and at 256 + 32 (0.90 to 1.0 in batches, 1.4 for four sequences of 8192); elsewhere
  // both take about the same (0.97 to 1.08), and 32 rows half the workspace. By the longest query of the call: the
  // lengths are on the device.
  pl.rows = most <= 32 ? 32 : 64;
  // As many workgroups as are resident at once: the key tiles take 144 KiB of LDS at 576 elements.
  const int per_cu = std::max(1, std::min(2, 163840 / (8 * 16 * 2 * (d.rank + d.rope_dim) + pl.rows / 32 * 4352)));
  const int64_t tiles = std::max<int64_t>(1, (latent_keys(d) + kLatentKeys - 1) / kLatentKeys);
  const int64_t units = ((int64_t)d.tokens * d.num_heads + (int64_t)pl.rows * std::min(d.batch, d.tokens)) / pl.rows;
  const int64_t wgs = std::min<int64_t>((int64_t)compute_units() * per_cu, units * tiles);
  pl.wgs = (int32_t)std::max<int64_t>(8, (wgs + 7) / 8 * 8);
  pl.ml = (int64_t)pl.wgs * 2 * pl.rows * d.rank * 4;
  pl.total = pl.ml + (int64_t)pl.wgs * 2 * pl.rows * 8;
  return pl;
}

static int validate_latent(const memopt_latent_desc &d) {
  MEMOPT_REQUIRE(d.dtype == MEMOPT_FP16 || d.dtype == MEMOPT_BF16, MEMOPT_ERR_INVALID,
                 "latent_attention: dtype must be fp16 or bf16");
  MEMOPT_REQUIRE(d.tokens >= 0 && d.batch >= 0 && d.max_query_len >= 0, MEMOPT_ERR_INVALID,
                 "latent_attention: negative size");
  MEMOPT_REQUIRE(d.num_heads > 0 && d.num_kv_blocks > 0 && d.max_blocks_per_seq > 0 && d.block_size > 0, MEMOPT_ERR_INVALID,
                 "latent_attention: no heads, or an empty cache or block table");
  MEMOPT_REQUIRE((d.rank == 128 || d.rank == 256 || d.rank == 512) && (d.rope_dim == 32 || d.rope_dim == 64),
                 MEMOPT_ERR_UNSUPPORTED, "latent_attention: rank must be 128, 256 or 512, rope_dim 32 or 64");
  MEMOPT_REQUIRE(d.block_size % 16 == 0, MEMOPT_ERR_UNSUPPORTED, "latent_attention: pages must hold a multiple of 16 tokens");
  MEMOPT_REQUIRE((int64_t)d.max_blocks_per_seq * d.block_size <= 1 << 30, MEMOPT_ERR_UNSUPPORTED,
                 "latent_attention: block tables of up to 2^30 tokens");
  auto aligned = [](const void *x, int64_t ts, int64_t hs) {
    return ((uintptr_t)x & 15) == 0 && ts % 8 == 0 && hs % 8 == 0;
  };
  MEMOPT_REQUIRE(aligned(d.query, d.q_token_stride, d.q_head_stride) && aligned(d.out, d.o_token_stride, d.o_head_stride) &&
                     aligned(d.cache, 0, 0) && aligned(d.workspace, 0, 0),
                 MEMOPT_ERR_INVALID, "latent_attention: rows, cache and workspace must be 16-byte aligned");
  // (steps and row tiles are counted in 32 bits; a launch holds 2^32 - 1 threads)
  const int64_t tiles = latent_keys(d) / kLatentKeys + 1, rows = (int64_t)d.tokens * d.num_heads;
  MEMOPT_REQUIRE(rows <= INT32_MAX - 255 && (rows / 32 + std::min(d.batch, d.tokens)) * tiles < (1LL << 31) &&
                     (rows / 32 + std::min(d.batch, d.tokens)) * 32 < (1LL << 24),
                 MEMOPT_ERR_UNSUPPORTED, "latent_attention: too many (row, token) tiles for one call");
  return MEMOPT_OK;
}

template <class E, int R, int P, int RW>
static int launch_latent(const LatentParams &p, int64_t units, hipStream_t s) {
  constexpr int bytes = LatentLds<R, P, RW>::bytes;
  const hipError_t set = allow_lds<&latent_kernel<E, R, P, RW>>(bytes);
  MEMOPT_REQUIRE(set == hipSuccess, MEMOPT_ERR_HIP, std::string("latent_attention: ") + hipGetErrorString(set));
  hipLaunchKernelGGL((latent_kernel<E, R, P, RW>), dim3((unsigned)p.wgs), dim3(128 * RW), bytes, s, p);
  int rc = check_launch("latent_attention");
  if (rc != MEMOPT_OK) return rc;
  hipLaunchKernelGGL((latent_merge_kernel<E, R, 32 * RW>), dim3((unsigned)(units * 8 * RW)), dim3(256), 0, s, p);
  return check_launch("latent_attention(merge)");
}
template <class E, int R, int P>
static int launch_latent(const LatentParams &p, int rows, int64_t units, hipStream_t s) {
  return rows == 32 ? launch_latent<E, R, P, 1>(p, units, s) : launch_latent<E, R, P, 2>(p, units, s);
}
template <class E>
static int launch_latent(const LatentParams &p, const memopt_latent_desc &d, int rows, int64_t units, hipStream_t s) {
  if (d.rope_dim == 64) {
    if (d.rank == 512) return launch_latent<E, 512, 64>(p, rows, units, s);
    if (d.rank == 256) return launch_latent<E, 256, 64>(p, rows, units, s);
    return launch_latent<E, 128, 64>(p, rows, units, s);
  }
  if (d.rank == 512) return launch_latent<E, 512, 32>(p, rows, units, s);
  if (d.rank == 256) return launch_latent<E, 256, 32>(p, rows, units, s);
  return launch_latent<E, 128, 32>(p, rows, units, s);
}

}  // namespace memopt

using namespace memopt;

extern "C" int memopt_latent_workspace_size(const memopt_latent_desc *desc, int64_t *bytes) {
  MEMOPT_REQUIRE(desc && bytes, MEMOPT_ERR_INVALID, "latent_workspace_size: null pointer");
  *bytes = 0;
  int rc = validate_latent(*desc);
  if (rc != MEMOPT_OK || desc->tokens == 0 || desc->batch == 0 || desc->max_query_len == 0) return rc;
  *bytes = latent_plan(*desc).total;
  return MEMOPT_OK;
}

extern "C" int memopt_latent_attention(const memopt_latent_desc *desc, void *stream) {
  MEMOPT_REQUIRE(desc, MEMOPT_ERR_INVALID, "latent_attention: null descriptor");
  const memopt_latent_desc &d = *desc;
  int rc = validate_latent(d);
  if (rc != MEMOPT_OK || d.tokens == 0 || d.batch == 0 || d.max_query_len == 0) return rc;
  MEMOPT_REQUIRE(d.query && d.cache && d.out && d.block_tables && d.context_lens && d.query_starts, MEMOPT_ERR_INVALID,
                 "latent_attention: null pointer");
  const LatentPlan pl = latent_plan(d);
  MEMOPT_REQUIRE(d.workspace && d.workspace_bytes >= pl.total, MEMOPT_ERR_INVALID,
                 "latent_attention: workspace needs " + std::to_string(pl.total) + " bytes");
  LatentParams p = {};
  p.q = (const uint16_t *)d.query;
  p.c = (const uint16_t *)d.cache;
  p.out = (uint16_t *)d.out;
  p.q_ts = d.q_token_stride;
  p.q_hs = d.q_head_stride;
  p.o_ts = d.o_token_stride;
  p.o_hs = d.o_head_stride;
  p.bt = d.block_tables;
  p.ctx = d.context_lens;
  p.starts = d.query_starts;
  p.nb = d.num_kv_blocks;
  p.page_bytes = (int64_t)d.block_size * (d.rank + d.rope_dim) * 2;
  p.T = d.tokens;
  p.B = d.batch;
  p.H = d.num_heads;
  p.M = d.max_blocks_per_seq;
  p.W = std::min(effective_window(d.window_size, d.max_seq_len), 1 << 30);  // (position - W stays in 32 bits)
  p.sinks = std::max(0, d.num_sink_tokens);
  p.max_keys = (int32_t)latent_keys(d);
  p.max_n = std::min(d.max_query_len, d.tokens);
  p.span = (pl.rows - 1) / d.num_heads + 2;
  p.by_h = Divisor::of((uint32_t)d.num_heads);
  p.by_chunks = Divisor::of((uint32_t)d.block_size / 16);
  p.scale_log2 = 1.4426950408889634f * d.scale;
  p.wgs = pl.wgs;
  p.ws_o = (float *)d.workspace;
  p.ws_ml = (float2 *)((uint8_t *)d.workspace + pl.ml);
  const int64_t units = ((int64_t)d.tokens * d.num_heads + (int64_t)pl.rows * std::min(d.batch, d.tokens)) / pl.rows;
  hipStream_t s = (hipStream_t)stream;
  return d.dtype == MEMOPT_FP16 ? launch_latent<Fp16>(p, d, pl.rows, units, s) : launch_latent<Bf16>(p, d, pl.rows, units, s);
}

extern "C" int memopt_write_latent(const void *latents, int64_t latent_stride, const void *rope_keys, int64_t rope_stride,
                                   int32_t num_tokens, int32_t rank, int32_t rope_dim, const int32_t *slots, void *cache,
                                   int64_t num_slots, void *stream) {
  MEMOPT_REQUIRE(num_tokens >= 0 && num_slots >= 0, MEMOPT_ERR_INVALID, "write_latent: negative size");
  MEMOPT_REQUIRE(rank > 0 && rope_dim >= 0 && rank % 8 == 0 && rope_dim % 8 == 0 && rank <= 65536 && rope_dim <= 65536,
                 MEMOPT_ERR_UNSUPPORTED, "write_latent: rank and rope_dim must be multiples of 8");
  if (num_tokens == 0) return MEMOPT_OK;
  MEMOPT_REQUIRE(latents && (rope_keys || rope_dim == 0) && slots && cache, MEMOPT_ERR_INVALID, "write_latent: null pointer");
  MEMOPT_REQUIRE((((uintptr_t)latents | (uintptr_t)rope_keys | (uintptr_t)cache) & 15) == 0 && latent_stride % 8 == 0 &&
                     rope_stride % 8 == 0,
                 MEMOPT_ERR_INVALID, "write_latent: rows must be 16-byte aligned");
  const int64_t pieces = (int64_t)num_tokens * ((rank + rope_dim) / 8);
  MEMOPT_REQUIRE(pieces <= INT32_MAX, MEMOPT_ERR_UNSUPPORTED, "write_latent: too many tokens for one call");
  const WriteLatentParams p = {(const uint16_t *)latents, (const uint16_t *)rope_keys, (uint16_t *)cache, latent_stride,
                               rope_stride, num_slots, slots, num_tokens, rank, rope_dim,
                               Divisor::of((uint32_t)(rank + rope_dim) / 8)};
  const int64_t wgs = std::min<int64_t>((pieces + 255) / 256, 16LL * compute_units());
  hipLaunchKernelGGL(write_latent_kernel, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, p);
  return check_launch("write_latent");
}
