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
// Long chunks: enough of them to fill the GPU with 128-row tiles attend from a
// staged copy of what they see instead (stage_kernel here, then the tiles of
// prompt.hip): a block of 32 rows unpacks each page once more, and from 512
// rows on that costs more than writing the copy. What follows is the rest.
//
// Work: QN = 8, 16 or 32 rows of one (sequence, key head) are a block; a wave takes
// two 16-token chunks (32 tokens) of a block's visible ones per step. The steps
// of all blocks of a key head form one list, which is dealt to its workgroups
// of 4 waves in runs that are equal but for a few steps around block ends,
// whatever the sequences' lengths (by sequence and split, a batch of 2700 to
// 8192 tokens ran as long as its longest part). A block whose steps fall to
// one workgroup is finished there; else each leaves partial sums, and the last
// to arrive adds them up. Layout, as in direct.hip:
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
//  * V enters as exact codes, too: the products of a scale group take the
//    weights times that group's scale per token. So a page's only rounding to
//    16 bits is that of weight times scale, and up to 128 rows what that loses
//    is a second operand (HALVES, REST).
//
// Bound by the stream of pages and 7 us around it: a copy of the kernel without
// its arithmetic took 41.5 us where it took 46.7 (32 sequences of 2700 to 8192
// tokens, 32 query over 8 key heads; 44.6 now, 4.4 TB/s of pages), one without
// the copies 37; one sequence of 131072 tokens 30 and 29 of 34.5 (34.2 now, 4.2
// TB/s). A large copy reaches 5.1 on the card. One sequence of 1024: 6.8 us, a
// chain of the list of sequences, the table, two steps, the waves' merge, the
// arrival and the workgroups' merge.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention.hpp"
#include "lds_dma.hpp"
#include "packed.hpp"
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
  int32_t T, B, Hq, Hk, G, M, bs;
  Divisor by_g;                  // rows to tokens
  int32_t span;                  // positions that a block of rows can spread over, less one
  int64_t nb;
  const uint8_t *k, *v;          // INT4 pages: k = the page buffer
  int64_t kv_ps, kv_hs, kv_ts;   // bytes
  int32_t W, sinks;
  float qk_scale_log2;
  int32_t wgs, blocks;           // workgroups per key head; blocks that ws_cnt has counters for
  uint32_t *ws_cnt;              // [blocks * Hk] arrivals; zero between calls
  float *ws_o, *ws_ml;           // [2 * wgs * Hk][QN][D], [2 * wgs * Hk][QN][2]: see partial_slot
  Staged st;                     // sequences that attend from a staged copy instead
};

// Workgroups per key head, so partial sums of a block, at most. (Reached with one
// or two key heads on 256 CUs, where it leaves room for more workgroups.)
static constexpr int kMaxParts = 256;

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
__device__ __forceinline__ Seq sequence(const PackedParams &p, const int32_t *__restrict__ starts,
                                        const int32_t *__restrict__ ctxs, int32_t b) {
  Seq q;
  const Rows rows = rows_of(starts, p.T, b);
  q.start = rows.start;
  q.n = rows.n;
  q.ctx = ctxs[b];
  q.kv_lim = (int32_t)min((int64_t)q.ctx, (int64_t)p.M * p.bs);
  q.blocks = is_staged(p.st, q.n, p.G) ? 0 : (q.n * p.G + QN - 1) / QN;
  const int32_t pos0 = q.ctx - q.n;
  int32_t n = visible_chunks(p, q.kv_lim, pos0, q.ctx - 1).n;
  if (q.blocks > 1) n = min(n, ((min(p.sinks, max(q.kv_lim, 0)) + 15) >> 4) + ((p.W + p.span) >> 4) + 2);
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
  uint32_t w[4][D / 64];  // [p_i][group]
  u32x4_t sc[D / 64];     // of a group: pair (p_i, p_i + 8) in word i
};
template <int D>
struct PackedV<D, MEMOPT_KV_FP16> {
  uint32_t w[8][D / 32];  // token e: D / 16 halves
};

// A block of BLK bytes (1 or 2 KiB and a tail) into LDS at m0v, 16 bytes per
// lane (lane16 = 16 * lane), not waited for: the compiler does not track it.
// The immediate offsets count for both addresses, the s_nop are the wait states
// between a write of m0 or of the descriptor and its use, as in lds_dma.hpp, and the tail's lanes are
// chosen in here (a branch around them costs six scalar instructions). STREAM:
// data read once per launch (kStreamLoad).
#define MEMOPT_COPY(OFF, NT) "buffer_load_dwordx4 %1, %2, 0 offen offset:" OFF NT " lds\n\t"
#define MEMOPT_COPY_TAIL(LANES, OFF, NT) \
  "s_mov_b64 %0, exec\n\ts_and_b64 exec, exec, " LANES "\n\t" MEMOPT_COPY(OFF, NT) "s_mov_b64 exec, %0"
template <bool STREAM, int BLK>
__device__ __forceinline__ void block_copy(__amdgpu_buffer_rsrc_t r, uint32_t m0v, uint32_t lane16) {
  static_assert(BLK == 2048 + 8 * 16 || BLK == 1024 + 4 * 16, "tails of 8 and 4 lanes");
  uint64_t lanes;
#define MEMOPT_COPY_ASM(TEXT) \
  asm volatile("s_nop 4\n\t" TEXT : "=&s"(lanes) : "v"(lane16), "s"(r), "{m0}"(m0v) : "memory", "scc")
  if constexpr (BLK == 2176 && STREAM)
    MEMOPT_COPY_ASM(MEMOPT_COPY("0", " nt") MEMOPT_COPY("1024", " nt") MEMOPT_COPY_TAIL("0xff", "2048", " nt"));
  else if constexpr (BLK == 2176)
    MEMOPT_COPY_ASM(MEMOPT_COPY("0", "") MEMOPT_COPY("1024", "") MEMOPT_COPY_TAIL("0xff", "2048", ""));
  else if constexpr (STREAM)
    MEMOPT_COPY_ASM(MEMOPT_COPY("0", " nt") MEMOPT_COPY_TAIL("0xf", "1024", " nt"));
  else
    MEMOPT_COPY_ASM(MEMOPT_COPY("0", "") MEMOPT_COPY_TAIL("0xf", "1024", ""));
#undef MEMOPT_COPY_ASM
}
#undef MEMOPT_COPY
#undef MEMOPT_COPY_TAIL

template <typename T>
__device__ __forceinline__ T lds_at(uint32_t a) {
  return *(const __attribute__((address_space(3))) T *)(uintptr_t)a;
}

// Workgroups per CU that the kernels' registers and LDS are meant for.
__host__ __device__ static constexpr int resident(int NW, int QN) { return QN == 32 ? 2 : NW == 4 ? 3 : 1; }

// Where the rest of the weights is a second operand (see REST below): for no
// row, for all, or for those of sequences with up to kRestRows rows.
enum Rest { kNoRest, kAllRest, kShortRest };
static constexpr int kRestRows = 128;

template <int D, int FMT, int QN, int NW, Rest REST>
__global__ __launch_bounds__(64 * NW, NW * resident(NW, QN) / 4) void packed_kernel(
    const PackedParams p, const int32_t *__restrict__ starts, const int32_t *__restrict__ ctxs,
    const int32_t *__restrict__ tables) {
  constexpr int NT = 64 * NW, KK = D / 32, ND = D / 16, QB = QN == 32 ? 2 : 1;
  constexpr bool PAGES = FMT == MEMOPT_KV_INT4;
  constexpr int NG = PAGES ? D / 64 : 1;  // score sums per (row, token)
  // Over pages, in sequences of up to 128 rows: a weight enters the second product
  // as the sum of two 16-bit operands, itself and what its rounding lost. One
  // rounding of a weight that makes up much of a row is an error of that whole
  // row: up to 4.8e-4 of the output's norm, where two operands leave the output's
  // own 2e-4. Up to 8 rows, the rest takes the other 8 columns of the same
  // instructions (HALVES: columns n and n + 8 are the same row); else
  // instructions of its own (REST), by sequence where a batch has longer ones, so
  // that what a request gets does not hang on its neighbours. (131072 tokens, 5
  // rows: 33.1 us without, 34.2 in columns, 37.7 as instructions; 8 sequences of
  // 4096 tokens and 64 rows 34.3 without, 38.8 with, of 256 rows 73 and 89: there
  // errors average out, to 3.0e-4. 12 single tokens of 4 rows beside 4 chunks of
  // 512 tokens: 2.9e-4 and 18.2 us without, 2.1e-4 and 20.4 with.)
  constexpr bool HALVES = QN == 8;
  constexpr int OS = D + 4;               // row stride of s_o: 16 rows of D floats would share a bank
  // Pages stream through a ring of raw blocks per wave (see copy_step), which
  // the merge of the waves takes over when the steps are done.
  constexpr int BLK = 16 * D + 64 * (D / 64), STG = 2 * BLK, NS = 2;
  constexpr int OBYTES = NW * QN * OS * 4, RBYTES = PAGES ? NW * NS * STG : 0, MBYTES = NT * 24;
  __shared__ __attribute__((aligned(16))) uint8_t smem[std::max({OBYTES, RBYTES, MBYTES})];
  float(*const s_o)[QN][OS] = reinterpret_cast<float(*)[QN][OS]>(smem);
  __shared__ float s_ml[NW][QN][2];
  __shared__ int s_last;

  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t kvh = blockIdx.x % p.Hk, wg = blockIdx.x / p.Hk;

  // The list's length; then the sequence that holds this workgroup's first
  // place. Lane i takes sequence b0 + i; up to 64 sequences are counted once.
  uint32_t sum = 0, blocks_sum = 0, c = 0, nb = 0, c_to = 0, nb_to = 0;  // places, blocks; up to this lane's end
  Seq lane_seq = {};
  auto count = [&](int32_t b0) __attribute__((always_inline)) {
    c = nb = 0;
    if (b0 + lane < p.B) {
      lane_seq = sequence<QN>(p, starts, ctxs, b0 + lane);
      nb = lane_seq.blocks;
      c = nb * (uint32_t)lane_seq.steps;
    }
    c_to = wave_scan(c);
    nb_to = wave_scan(nb);
  };
  for (int32_t b0 = 0; b0 < p.B; b0 += 64) {
    count(b0);
    sum = __builtin_elementwise_add_sat(sum, (uint32_t)__builtin_amdgcn_readlane((int)c_to, 63));
    blocks_sum = __builtin_elementwise_add_sat(blocks_sum, (uint32_t)__builtin_amdgcn_readlane((int)nb_to, 63));
  }
  // (past 2^31 only where sequences overlap: nothing is computed then)
  const int32_t total = (int32_t)sum;
  // Runs of one step per wave at least: shorter ones cost more to merge than they save.
  const int32_t wgs = min(p.wgs, max(1, total / NW));
  if (total <= 0 || wg >= wgs) return;
  const int32_t run = total / wgs, longer = total - run * wgs;  // the first `longer` runs have one place more
  auto start_of = [&](int32_t w) { return w * run + min(w, longer); };
  const int32_t first = start_of(wg), next = start_of(wg + 1);
  int32_t at = first;
  auto wg_of = [&](int32_t x) {
    const int32_t edge = longer * (run + 1);
    const bool head = x < edge;
    return (head ? 0 : longer) + (head ? x : x - edge) / (head ? run + 1 : run);
  };
  // A run that would begin within `snap` places of a block's end begins there: a
  // block in two workgroups costs a start and a merge more, about as long as
  // that many steps of one; the more, the fewer workgroups there are for each
  // block. (Us with 0, 8 and 16, 32 query over 8 key heads, 96 workgroups: 64
  // sequences of 300 tokens 22.3, 13.1, 13.0; 64 of 1000 28.1, 26.4, 22.5; 128 of
  // 100 to 3000 57.7, 53.9, 51.0; 32 of 2700 to 8192 45.6, 42.2, 42.6; 8 of 100 to
  // 2000 17.4, 12.3, 13.6; 4 of 1000 11.2, 11.3, 12.7.)
  const int32_t snap = blocks_sum <= 1 ? 0 : 2 * blocks_sum >= (uint32_t)wgs ? 16 : 8;
  int32_t seq_at = 0, seq_blocks = 0, b = 0;  // places and blocks before sequence b
  Seq seq = {};
  for (int32_t b0 = 0; b0 < p.B; b0 += 64) {
    if (p.B > 64) count(b0);
    const int32_t sum64 = __builtin_amdgcn_readlane((int)c_to, 63);
    if (at < seq_at + sum64) {
      const int src = __builtin_ctzll(__ballot(at < seq_at + (int32_t)c_to));
      auto from = [&](int32_t v) { return __builtin_amdgcn_readlane(v, src); };
      b = b0 + src;
      seq_at += from((int32_t)(c_to - c));
      seq_blocks += from((int32_t)(nb_to - nb));
      seq = {from(lane_seq.start), from(lane_seq.n),      from(lane_seq.ctx),
             from(lane_seq.kv_lim), from(lane_seq.blocks), from(lane_seq.steps)};
      break;
    }
    seq_at += sum64;
    seq_blocks += __builtin_amdgcn_readlane((int)nb_to, 63);
  }

  // Block by block of this workgroup's run.
  for (;;) {
    int32_t block, block_at, w0, w1;
    do {
      while (at >= seq_at + seq.blocks * seq.steps) {  // (sequences without rows take no place)
        seq_at += seq.blocks * seq.steps;
        seq_blocks += seq.blocks;
        seq = sequence<QN>(p, starts, ctxs, ++b);
      }
      block = seq.blocks == 1 ? 0 : (at - seq_at) / seq.steps;
      block_at = seq_at + block * seq.steps;
      at = block_at + seq.steps;
      const int32_t s = min(snap, seq.steps >> 1), x0 = block_at + s, x1 = at - max(s, 1);
      w0 = x0 >= first && x0 < next ? wg : wg_of(x0);
      w1 = x1 >= first && x1 < next ? wg : wg_of(x1);
    } while (wg > w1 && at < total);  // (a run that begins behind its first place)
    if (wg < w0 || wg > w1) return;
    if (seq_blocks + block >= p.blocks) return;  // sequences overlap: past the counters
    const int32_t row0 = block * QN, rows = seq.n * p.G, ctx = seq.ctx, kv_lim = seq.kv_lim;
    const int32_t pos0 = ctx - seq.n;  // position of the sequence's first query
    const int32_t pos_lo = pos0 + p.by_g(row0), pos_hi = pos0 + p.by_g(min(row0 + QN, rows) - 1);
    const Visible vis = visible_chunks(p, kv_lim, pos_lo, pos_hi);
    const int32_t sc = vis.sc, wc0 = vis.wc0, n_vis = vis.n;
    const int32_t begin = wg == w0 ? 0 : first - block_at;
    const int32_t end = min(wg == w1 ? seq.steps : next - block_at, (n_vis + 1) >> 1);

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

    // Chunk i of the visible list is logical chunk i, or i + skip behind the
    // sinks. A step is the chunks 2 i and 2 i + 1; those of steps [full0, full1)
    // lie where every row sees all their tokens, so they need no mask once both
    // pages are there.
    const int32_t *btrow = tables + (int64_t)b * p.M;
    const int32_t cpp = PAGES ? 1 : p.bs >> 4;
    const int32_t nb32 = (int32_t)min(p.nb, (int64_t)INT32_MAX);
    const int32_t skip = wc0 - sc;
    auto logical = [&](int32_t i) { return i + (i < sc ? 0 : skip); };
    const int32_t full0 = (max(skip > 0 ? sc : 0, ((max(0, pos_hi - p.W + 1) + 15) >> 4) - skip) + 1) >> 1;
    const int32_t full1 = ((max(0, min(kv_lim, pos_lo + 1)) >> 4) - skip) >> 1;
    // This wave's steps are begin + wave + j NW, j < mine. Their block-table
    // entries are looked up 32 steps at a time, lane l for chunk l % 2 of step
    // at0 + l / 2: byte offset of the chunk (chunk 0 of page 0 if its page is not
    // there), whether it is there, and whether the step needs no mask. (Entry
    // by entry, in scalar loads, they took half as many scalar instructions
    // per step as it has vector ones, and every wait for LDS waited for them.)
    const int32_t mine = max(0, end - begin - wave + NW - 1) / NW;
    int32_t at0 = 0;
    uint32_t off_lo = 0, off_hi = 0;
    uint64_t there = 0, whole = 0;
    auto look_up = [&](int32_t j0) __attribute__((always_inline)) {
      at0 = j0;
      const int32_t i = begin + wave + (j0 + (lane >> 1)) * NW, c = 2 * i + (lane & 1), lc = logical(c);
      const bool in = i < end && c < n_vis;
      const int32_t phys = in ? btrow[cpp == 1 ? lc : lc / cpp] : -1;
      const bool ok = phys >= 0 && phys < nb32;
      int64_t x = (int64_t)(ok ? phys : 0) * p.kv_ps;
      if constexpr (!PAGES) x += (int64_t)(ok ? 16 * (lc - lc / cpp * cpp) : 0) * p.kv_ts;
      off_lo = (uint32_t)x;
      off_hi = (uint32_t)((uint64_t)x >> 32);
      there = __ballot(ok);
      whole = there & (there >> 1) & __ballot(i >= full0 && i < full1);  // (even bits count)
    };
    auto step_at = [&](int32_t j) { return begin + wave + j * NW; };
    auto offset_of = [&](int32_t j, int chunk) __attribute__((always_inline)) {
      const int32_t l = 2 * (j - at0) + chunk;
      return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)off_hi, l) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)off_lo, l));
    };

    const Int4Page f(D);
    PackedK<D, FMT> kr;
    PackedV<D, FMT> vr;
    const int p0 = 4 * (g & 1);  // this lane's score tokens: p0 + i and p0 + i + 8 of chunk g / 2
    // Pages: the two blocks of a step as they are, 1 KiB per copy, straight into
    // the wave's ring: NS steps are in flight without holding registers.
    const uint32_t ring = lds_u32(smem) + wave * NS * STG;
    const uint8_t *const kbase = p.k + (int64_t)kvh * p.kv_hs, *const vbase = p.v + (int64_t)kvh * p.kv_hs;
    auto copy_block = [&](int64_t kv, uint32_t dst) __attribute__((always_inline)) {
      const __amdgpu_buffer_rsrc_t rs =
          __builtin_amdgcn_make_buffer_rsrc((void *)(kbase + kv), (short)0, BLK, 0x00020000);
      block_copy<QB == 1, BLK>(rs, dst, 16 * lane);
    };
    auto copy_step = [&](int32_t j, int stage) __attribute__((always_inline)) {
      copy_block(offset_of(j, 0), ring + stage * STG);
      copy_block(offset_of(j, 1), ring + stage * STG + BLK);
    };
    // K of a step: lane row r is tokens r % 8 and r % 8 + 8 of chunk r / 8.
    // V: lane (r, g) holds four dims from 64 u + 4 r (fp16: [D/16 r, D/16 (r + 1))) of its score tokens.
    auto read_k = [&](int stage) __attribute__((always_inline)) {
      if constexpr (PAGES) {
        const uint32_t at = ring + stage * STG;
        const uint32_t kb = at + (r < 8 ? 0 : BLK) + (uint32_t)f.kcodes + (8 * (r & 7) + (D == 128 ? g : 2 * g)) * (D / 8);
        const uint32_t tb = at + (g < 2 ? 0 : BLK);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          // (D = 128: lane group 4 j + g of the page, 16 dims of scale group j; D = 64: groups 2 g and 2 g + 1)
          const u32x4_t x = lds_at<u32x4_t>(kb + 4 * j * (D / 8));
#pragma unroll
          for (int w = 0; w < 4; ++w) kr.w[4 * j + w] = x[w];
          kr.sc[j] = lds_at<u32x4_t>(tb + (uint32_t)f.kscales + 2 * (16 * j + 2 * p0));
        }
      }
    };
    auto read_v = [&](int stage) __attribute__((always_inline)) {
      if constexpr (PAGES) {
        const uint32_t tb = ring + stage * STG + (g < 2 ? 0 : BLK);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int u = 0; u < D / 64; ++u)
            vr.w[i][u] = lds_at<uint32_t>(tb + (uint32_t)f.vcodes + 8 * (p0 + i) * (D / 8) + 64 * u + 4 * r);
        }
#pragma unroll
        for (int u = 0; u < D / 64; ++u)
          vr.sc[u] = lds_at<u32x4_t>(tb + (uint32_t)f.vscales + 2 * (16 * u + 2 * p0));
      }
    };
    // fp16 pools: the same from global memory into registers.
    auto load_k = [&](int32_t j) __attribute__((always_inline)) {
      if constexpr (!PAGES) {
        const int64_t xa = offset_of(j, 0), xb = offset_of(j, 1);
        const uint8_t *base = kbase + (r < 8 ? xa : xb);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
            kr.w[t][kk] = *reinterpret_cast<const u32x4_t *>(base + (int64_t)((r & 7) + 8 * t) * p.kv_ts +
                                                             2 * (32 * kk + 8 * g));
      }
    };
    auto load_v = [&](int32_t j) __attribute__((always_inline)) {
      if constexpr (!PAGES) {
        const int64_t xa = offset_of(j, 0), xb = offset_of(j, 1);
        const uint8_t *base = vbase + (g < 2 ? xa : xb);
#pragma unroll
        for (int x = 0; x < 8; ++x) {  // element 2 i + t: token p0 + i + 8 t
          const uint8_t *src = base + (int64_t)(p0 + (x >> 1) + 8 * (x & 1)) * p.kv_ts + (D / 8) * r;
          if constexpr (D == 128) {
            const u32x4_t y = *reinterpret_cast<const u32x4_t *>(src);
#pragma unroll
            for (int j = 0; j < 4; ++j) vr.w[x][j] = y[j];
          } else {
            const u32x2_t y = *reinterpret_cast<const u32x2_t *>(src);
            vr.w[x][0] = y[0];
            vr.w[x][1] = y[1];
          }
        }
      }
    };

    // (w & mask) | bits as one v_and_or_b32: the constants are hidden from the
    // compiler, which would make two instructions of them. (As inline assembly,
    // the instruction escapes the compiler's wait states: one that overwrote
    // the start of a sum while its matrix instruction still read it gave NaN.)
    uint32_t m_lo = 0x000F000Fu, m_hi = 0x00F000F0u, e1024 = 0x64006400u, e64 = 0x54005400u;
    asm("" : "+s"(m_lo), "+s"(m_hi));
    asm("" : "+v"(e1024), "+v"(e64));
    const half2_t b1032 = {(half_t)1032.0f, (half_t)1032.0f}, b72 = {(half_t)72.0f, (half_t)72.0f};
    // The eight codes of a word, less 8, in nibble-unpack order (exact).
    auto codes = [&](uint32_t w) __attribute__((always_inline)) {
      const uint32_t w8 = w >> 8;
      return u32x4_t{as_u32(as_half2((w & m_lo) | e1024) - b1032), as_u32(as_half2((w & m_hi) | e64) - b72),
                     as_u32(as_half2((w8 & m_lo) | e1024) - b1032), as_u32(as_half2((w8 & m_hi) | e64) - b72)};
    };
    // The same without the subtractions, so plus 1032 in the even pairs and 72
    // in the odd ones: K's sums start at minus those times the sums of q
    // (kstart). Their 32-bit roundings grow to about 2^-24 * 1032 of the sum of
    // |q| * scale, a tenth of what rounding K to fp16 would cost, and far below
    // the rounding of the probabilities.
    auto biased = [&](uint32_t w) __attribute__((always_inline)) {
      const uint32_t w8 = w >> 8;
      return u32x4_t{(w & m_lo) | e1024, (w & m_hi) | e64, (w8 & m_lo) | e1024, (w8 & m_hi) | e64};
    };
    const half2_t ones = {(half_t)1.0f, (half_t)1.0f};
    const uint32_t second_half = r < 8 ? 0u : ~0u;
    h8_t qf[QB][KK];
    f32x4_t kstart[QB][NG];
    int32_t row_pos[QB];
    // Q as the B operand: column r = row, k-group g; dims of product kk as the K
    // operand holds them (pages: 16 g + 8 (kk % 2) of scale group kk / 2, in
    // nibble-unpack order; fp16: 32 kk + 8 g). Loaded ahead of the first pages,
    // used behind their copies.
    auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int32_t row = row0 + 16 * qb + (HALVES ? r & 7 : r), tok = p.by_g(row);
        row_pos[qb] = pos0 + tok;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) qf[qb][kk] = (h8_t){};
        if (row < rows) {
          const half_t *src = p.q + (int64_t)(seq.start + tok) * p.q_ts +
                              (int64_t)(kvh * p.G + row - tok * p.G) * p.q_hs + (PAGES ? 16 * g : 8 * g);
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
            qf[qb][kk] = __builtin_bit_cast(
                h8_t, *reinterpret_cast<const u32x4_t *>(src + (PAGES ? 64 * (kk >> 1) + 8 * (kk & 1) : 32 * kk)));
        }
      }
    };
    auto prepare_q = [&]() __attribute__((always_inline)) {
      if constexpr (PAGES) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            const h8_t y = qf[qb][kk];
            qf[qb][kk] = h8_t{y[0], y[4], y[1], y[5], y[2], y[6], y[3], y[7]};
          }
      }
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          float x = 0.0f;
          if constexpr (PAGES) {
            float even = 0.0f, odd_q = 0.0f;  // operand pairs 0, 2 and 1, 3
#pragma unroll
            for (int kk = j * (KK / NG); kk < (j + 1) * (KK / NG); ++kk) {
              const u32x4_t y = __builtin_bit_cast(u32x4_t, qf[qb][kk]);
              even = __builtin_amdgcn_fdot2(as_half2(y[0]), ones, even, false);
              even = __builtin_amdgcn_fdot2(as_half2(y[2]), ones, even, false);
              odd_q = __builtin_amdgcn_fdot2(as_half2(y[1]), ones, odd_q, false);
              odd_q = __builtin_amdgcn_fdot2(as_half2(y[3]), ones, odd_q, false);
            }
            x = xor32_sum(xor16_sum(-1032.0f * even - 72.0f * odd_q));
          }
          kstart[qb][j] = f32x4_t{x, x, x, x};
        }
    };
    auto k_operand = [&](int t, int kk) __attribute__((always_inline)) {
      if constexpr (PAGES) {
        return __builtin_bit_cast(h8_t, biased(D == 128 ? kr.w[4 * (kk >> 1) + 2 * t + (kk & 1)] : kr.w[2 * kk + t]));
      } else {
        return __builtin_bit_cast(h8_t, kr.w[t][kk]);
      }
    };

    // exp2 argument of a new maximum: probabilities lie in (0, 2^15], so fp16
    // holds those down to 2^-21 of the largest as normal numbers.
    constexpr float kTop = 7.0f;
    uint32_t odd = 0;  // nonzero: a masked step held inf or NaN in V
    // One step; `between` runs when K has been used and V has not.
    auto step = [&](int32_t j, auto rest, auto between) __attribute__((always_inline)) {
      constexpr bool R = decltype(rest)::value;
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
                a, qf[qb][kk], kk % PG == 0 ? kstart[qb][kk / PG] : s[qb][kk / PG][t], 0, 0, 0);
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
            y = fmaf(y, (float)as_half2(kr.sc[0][e >> 1])[e & 1], 0.0f);  // (one mixed-precision instruction)
            if constexpr (NG == 2) y = fmaf(s[qb][1][e & 1][e >> 1], (float)as_half2(kr.sc[1][e >> 1])[e & 1], y);
          }
          x[qb][e] = fmaf(y, p.qk_scale_log2, ncm[qb]);
        }
      const int32_t bit = 2 * (j - at0);
      const bool full = (whole >> bit) & 1;  // (wave-uniform)
      const bool c_ok = (there >> (bit + (g >> 1))) & 1;
      const int32_t key0 = 16 * logical(2 * step_at(j) + (g >> 1)) + 4 * (g & 1);
      between();

      h8_t pf[QB][NG], pf_rest[QB][NG];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        u32x4_t vs[NG];
        if constexpr (PAGES) {
#pragma unroll
          for (int u = 0; u < NG; ++u) vs[u] = vr.sc[u];
        }
        if (!full) {
          const int32_t last = c_ok ? min(row_pos[qb], kv_lim - 1) - key0 : -1;
          const int32_t first_w = row_pos[qb] - p.W + 1 - key0, end_s = p.sinks - key0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int32_t c = (e >> 1) + 8 * (e & 1);
            const bool seen = (c <= last) & ((c >= first_w) | (c < end_s));
            x[qb][e] = seen ? x[qb][e] : -INFINITY;
            if constexpr (PAGES) {  // (a weight of 0 must not meet a scale that is inf or NaN)
#pragma unroll
              for (int u = 0; u < NG; ++u) vs[u][e >> 1] &= seen ? ~0u : (e & 1) ? 0x0000FFFFu : 0xFFFF0000u;
            }
          }
        }
        float t = x[qb][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) t = fmaxf(t, x[qb][e]);
        if constexpr (PAGES) {
          // The weights enter the second product times their token's scale, so
          // what the running maximum bounds is that product: x plus the log2 of
          // the largest scale here, read off its bits (2^(bits / 1024 - 15), too
          // small by 0.09 at most).
          typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
          u16x2 m = {0, 0};
#pragma unroll
          for (int i = 0; i < 4 * NG; ++i) {
            const uint32_t w = vs[i / 4][i % 4];  // (a bit cast of the vector's element itself takes its element 0)
            m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w));
          }
          t += fmaf((float)max((uint32_t)m[0], (uint32_t)m[1]), 1.0f / 1024.0f, -15.0f);
        }
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
#pragma unroll
        for (int e = 0; e < 8; ++e) x[qb][e] = fast_exp2(x[qb][e]);
        u32x4_t w;
        if constexpr (PAGES) {
#pragma unroll
          for (int e = 0; e < 8; ++e) lsum[qb] += x[qb][e];
#pragma unroll
          for (int u = 0; u < NG; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i)  // (one mixed-precision instruction for each half)
              w[i] = as_u32(half2_t{(half_t)fmaf(x[qb][2 * i], (float)as_half2(vs[u][i])[0], 0.0f),
                                    (half_t)fmaf(x[qb][2 * i + 1], (float)as_half2(vs[u][i])[1], 0.0f)});
            if constexpr (HALVES) {  // lanes n >= 8: what the rounding of their twin lost
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const half2_t twin = as_half2(w[i] & second_half);
                w[i] = as_u32(half2_t{(half_t)fmaf(x[qb][2 * i], (float)as_half2(vs[u][i])[0], -(float)twin[0]),
                                      (half_t)fmaf(x[qb][2 * i + 1], (float)as_half2(vs[u][i])[1], -(float)twin[1])});
              }
            }
            pf[qb][u] = __builtin_bit_cast(h8_t, w);
            if constexpr (R) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = as_u32(half2_t{
                    (half_t)fmaf(x[qb][2 * i], (float)as_half2(vs[u][i])[0], -(float)pf[qb][u][2 * i]),
                    (half_t)fmaf(x[qb][2 * i + 1], (float)as_half2(vs[u][i])[1], -(float)pf[qb][u][2 * i + 1])});
              pf_rest[qb][u] = __builtin_bit_cast(h8_t, w);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = as_u32(half2_t{(half_t)x[qb][2 * i], (half_t)x[qb][2 * i + 1]});
            lsum[qb] = __builtin_amdgcn_fdot2(as_half2(w[i]), ones, lsum[qb], false);
          }
          pf[qb][0] = __builtin_bit_cast(h8_t, w);
        }
      }

      // fp16: a weight of 0 must not meet an inf or NaN of V. Tokens that no row
      // of the block sees (behind the context, unlinked, outside the window)
      // become zeros; so do inf and NaN among those that only some rows see,
      // which get them back at the end (`odd`).
      if constexpr (!PAGES) {
        if (!full) {
          const int32_t last = c_ok ? min(pos_hi, kv_lim - 1) - key0 : -1;
          const int32_t first_w = pos_lo - p.W + 1 - key0, end_s = p.sinks - key0;
          const bool several = pos_lo != pos_hi;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int32_t c = (e >> 1) + 8 * (e & 1);
            const bool live = (c <= last) & ((c >= first_w) | (c < end_s));
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
              uint32_t w = live ? vr.w[e][j] : 0u;
              if (several) {
                const uint32_t f = ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;  // a full exponent carries
                odd |= f;
                w &= ~((f << 1) - (f >> 15));
              }
              vr.w[e][j] = w;
            }
          }
        }
      }
      auto pv = [&](int i, u32x4_t a) __attribute__((always_inline)) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const h8_t v = __builtin_bit_cast(h8_t, a);
          o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[qb][i / (ND / NG)], o[qb][i], 0, 0, 0);
          if constexpr (R)
            o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf_rest[qb][i / (ND / NG)], o[qb][i], 0, 0, 0);
        }
      };
      if constexpr (PAGES) {
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
          u32x4_t y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = codes(vr.w[i][u]);
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
    };

    // Wave w takes steps begin + w, begin + w + NW, ...
    if constexpr (PAGES) {
      constexpr int CPS = 2 * ((BLK + 1023) / 1024);  // copies per step
      load_q();
      look_up(0);
#pragma unroll
      for (int k = 0; k < NS; ++k)
        if (k < mine) copy_step(k, k);
      prepare_q();
      auto walk = [&](auto rest) __attribute__((always_inline)) {
        int stage = 0;
#pragma unroll 1
        for (int32_t j = 0; j < mine; ++j) {
          if (j + NS - at0 >= 32) look_up(j);
          // this step's copies are the oldest: wait until no more than the later step's are left
          static_assert(NS == 2, "one later step");
          if (j + 1 < mine) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(CPS) : "memory");
          else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          read_k(stage);
          step(j, rest, [&]() __attribute__((always_inline)) {
            read_v(stage);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the stage is filled again
            if (j + NS < mine) copy_step(j + NS, stage);
          });
          stage ^= 1;
        }
      };
      if constexpr (REST == kShortRest) {
        if (rows <= kRestRows) walk(std::true_type{});
        else walk(std::false_type{});
      } else {
        walk(std::integral_constant<bool, REST == kAllRest>{});
      }
      if constexpr (HALVES) {  // both columns of a row
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
          for (int reg = 0; reg < 4; ++reg) {
            const uint32_t v = __float_as_uint(o[0][i][reg]);
            o[0][i][reg] += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true));
          }
      }
      __syncthreads();  // every wave has read its ring: the sums take its place
    } else {
      load_q();
      look_up(0);
      if (0 < mine) {
        load_k(0);
        load_v(0);
      }
      prepare_q();
#pragma unroll 1
      for (int32_t j = 0; j < mine; ++j) {
        if (j + 1 - at0 >= 32) look_up(j);
        step(j, std::false_type{}, [&]() __attribute__((always_inline)) {
          if (j + 1 < mine) load_k(j + 1);
        });
        if (j + 1 < mine) load_v(j + 1);
      }
    }

    if constexpr (!PAGES) {
      if (__any(odd != 0)) {
        // Rows that see an inf or NaN of V have inf or NaN in its column whatever
        // its weight; a lane looks through its quarter of the dims.
#pragma unroll 1
        for (int32_t j = 0; j < mine; ++j) {
          if (j < at0 || j >= at0 + 32) look_up(j);
          if ((whole >> (2 * (j - at0))) & 1) continue;  // (its V went in as it is)
#pragma unroll 1
          for (int tk = 0; tk < 32; ++tk) {
            const int32_t t = tk & 15, key = 16 * logical(2 * step_at(j) + (tk >> 4)) + t;
            if (!((there >> (2 * (j - at0) + (tk >> 4))) & 1) || key >= kv_lim) continue;
            const half_t *row = reinterpret_cast<const half_t *>(vbase + offset_of(j, tk >> 4) + (int64_t)t * p.kv_ts);
#pragma unroll
            for (int d = 0; d < D / 4; ++d) {
              const float y = (float)row[(D / 4) * g + d];
              const bool bad = (__float_as_uint(y) & 0x7F800000u) == 0x7F800000u;
#pragma unroll
              for (int qb = 0; qb < QB; ++qb)
                if (bad && key <= row_pos[qb] && (key < p.sinks || key >= row_pos[qb] - p.W + 1))
                  o[qb][d % ND][d / ND] += y;
            }
          }
        }
      }
    }

    // Merge of the waves. Row 4 g + reg of V^T product i is dim 64 (i / 4) + 4 (4 g
    // + reg) + i % 4 over pages, D/16 (4 g + reg) + i over fp16 pools.
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const float l = xor32_sum(xor16_sum(lsum[qb]));
      const int row = 16 * qb + r;
      if (row0 + row >= rows || (HALVES && r >= 8)) continue;
#pragma unroll
      for (int reg = 0; reg < 4; ++reg)
#pragma unroll
        for (int i = 0; i < ND; i += 4)
          *reinterpret_cast<f32x4_t *>(&s_o[wave][row][PAGES ? 16 * i + 4 * (4 * g + reg) : ND * (4 * g + reg) + i]) =
              f32x4_t{o[qb][i][reg], o[qb][i + 1][reg], o[qb][i + 2][reg], o[qb][i + 3][reg]};
      if (g == 0) {
        s_ml[wave][row][0] = thr[qb] == -INFINITY ? -INFINITY : -ncm[qb];
        s_ml[wave][row][1] = l;
      }
    }
    __syncthreads();
    // A block whose steps lie in one run is finished here.
    const int32_t live = min(QN, rows - row0);
    auto write_row = [&](int row, int d, f32x4_t x, float l) __attribute__((always_inline)) {
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      const int32_t rr = row0 + row, tok = p.by_g(rr);
      *reinterpret_cast<u32x2_t *>(p.out + (int64_t)(seq.start + tok) * p.o_ts +
                                   (int64_t)(kvh * p.G + rr - tok * p.G) * p.o_hs + d) =
          u32x2_t{as_u32(half2_t{(half_t)(x[0] * inv), (half_t)(x[1] * inv)}),
                  as_u32(half2_t{(half_t)(x[2] * inv), (half_t)(x[3] * inv)})};
    };
    // A run holds at most two blocks in part: one that began before it (slot 0),
    // one that begins in it and goes on behind it (slot 1).
    auto partial_slot = [&](int32_t w) { return ((int64_t)w * 2 + (w == w0 ? 1 : 0)) * p.Hk + kvh; };
    const int64_t own_part = partial_slot(wg) * QN;
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
        uint64_t *dst = reinterpret_cast<uint64_t *>(p.ws_o + (own_part + row) * D + d);
        __hip_atomic_store(dst, __builtin_bit_cast(uint64_t, u32x2_t{__float_as_uint(x[0]), __float_as_uint(x[1])}),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(dst + 1, __builtin_bit_cast(uint64_t, u32x2_t{__float_as_uint(x[2]), __float_as_uint(x[3])}),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (d == 0)
          __hip_atomic_store(reinterpret_cast<uint64_t *>(p.ws_ml + 2 * (own_part + row)),
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
      const int32_t parts = w1 - w0 + 1;
      constexpr int R = 8;
      if (s_last) {
        auto load2 = [&](const float *src) __attribute__((always_inline)) {
          const u32x2_t u = __builtin_bit_cast(
              u32x2_t, __hip_atomic_load(reinterpret_cast<const uint64_t *>(src), __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT));
          return float2{__uint_as_float(u[0]), __uint_as_float(u[1])};
        };
        // Partial `part` of the block: its sums, row by row.
        auto row_of = [&](int32_t part, int row) { return partial_slot(w0 + min(part, parts - 1)) * QN + row; };
        // A thread takes four dims of a row and works out the partials' weights
        // itself: loads of one round trip and no wait between the waves. Where
        // there are more partials and threads than that, they are dealt to
        // several threads, whose sums meet in LDS. (The row's weights by a wave
        // first, then the sums: 8.6 us where this takes 7.2, for one sequence of
        // 1024 tokens.)
        auto merge = [&](auto few) __attribute__((always_inline)) {
          constexpr bool ONE = decltype(few)::value;  // one pass: no more partials than a thread loads at once
          const int32_t cells = live * (D / 4), groups = ONE ? 1 : max(1, NT / cells);
          f32x4_t *const sums = reinterpret_cast<f32x4_t *>(smem);
          float2 *const sums_ml = reinterpret_cast<float2 *>(smem + NT * 16);
          for (int c0 = 0; c0 < cells; c0 += NT) {  // (once where the cells fit the workgroup)
            const int cell = groups > 1 ? tid % cells : c0 + tid, part = groups > 1 ? tid / cells : 0;
            const bool on = cell < cells && part < groups;
            const int row = cell / (D / 4), d = 4 * (cell % (D / 4));
            f32x4_t x = {};
            float mx = -INFINITY, l = 0.0f;
            for (int32_t i0 = part; i0 < (ONE ? 1 : parts) && on; i0 += R * groups) {
              float2 ml[R], y[R][2];
#pragma unroll
              for (int k = 0; k < R; ++k) {  // (past the last: that one again, without weight)
                const int64_t at_k = row_of(i0 + k * groups, row);
                ml[k] = load2(p.ws_ml + 2 * at_k);
                y[k][0] = load2(p.ws_o + at_k * D + d);
                y[k][1] = load2(p.ws_o + at_k * D + d + 2);
              }
              const float before = mx;
#pragma unroll
              for (int k = 0; k < R; ++k) mx = fmaxf(mx, ml[k].x);
              const float again = before == -INFINITY ? 0.0f : fast_exp2(before - mx);
              l *= again;
              x *= again;
#pragma unroll
              for (int k = 0; k < R; ++k) {
                const bool past = i0 + k * groups >= parts;
                const float f = past || ml[k].x == -INFINITY ? 0.0f : fast_exp2(ml[k].x - mx);
                l += f * ml[k].y;
                const f32x4_t z = f32x4_t{y[k][0].x, y[k][0].y, y[k][1].x, y[k][1].y} * f;
                x += past ? f32x4_t{} : z;  // (no weight must not meet its inf again)
              }
            }
            if (groups > 1) {
              sums[tid] = x;
              sums_ml[tid] = float2{mx, l};
              __syncthreads();
              if (on && part == 0) {
                float top = mx;
                for (int k = 1; k < groups; ++k) top = fmaxf(top, sums_ml[tid + k * cells].x);
                l = 0.0f;
                x = (f32x4_t){};
                for (int k = 0; k < groups; ++k) {
                  const float2 ml = sums_ml[tid + k * cells];
                  const float f = ml.x == -INFINITY ? 0.0f : fast_exp2(ml.x - top);
                  l += f * ml.y;
                  x += sums[tid + k * cells] * f;
                }
              }
            }
            if (on && part == 0) write_row(row, d, x, l);
          }
        };
        if (parts <= R) merge(std::true_type{});
        else merge(std::false_type{});
      }
    }
    if (wg < w1 || at >= total) return;
    __syncthreads();  // s_o and s_ml are free for the next block
  }
}

// The staged copies: K and V of what the staged sequences see, as fp16 rows.
// The 64-token tiles of all of them form one list; workgroup i of a key head
// takes tiles i, i + gridDim, ..., each wave 16 tokens of them, which lie in
// one page. A wave reads a block of a page as it is (lane l: the 16 dims (D =
// 64: 8) of tokens p = l / 8 and p + 8 that start at D / 8 * (l % 8)) and writes
// V as fp16((code - 8) * scale), one rounding that the kernel above does not
// make (there V enters as codes, and the weights carry its scales), and K as
// codes with their factors.
template <int D, int FMT>
__global__ __launch_bounds__(256) void stage_kernel(const PackedParams p, const int32_t *__restrict__ starts,
                                                    const int32_t *__restrict__ ctxs,
                                                    const int32_t *__restrict__ tables) {
  constexpr bool PAGES = FMT == MEMOPT_KV_INT4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t kvh = blockIdx.x % p.Hk, wg = blockIdx.x / p.Hk, wgs = gridDim.x / p.Hk;
  const Int4Page f(D);
  int32_t item = wg, before = 0, slots = 0;
  for (int32_t b0 = 0; b0 < p.B; b0 += 64) {
    // lane i: sequence b0 + i
    bool on = false;
    int32_t n = 0, kv_lim = 0, tiles = 0;
    StagedMap m = {};
    if (b0 + lane < p.B) {
      n = rows_of(starts, p.T, b0 + lane).n;
      const int32_t ctx = ctxs[b0 + lane];
      kv_lim = (int32_t)min((int64_t)ctx, (int64_t)p.M * p.bs);
      on = is_staged(p.st, n, p.G);
      m = staged_map(kv_lim, ctx - n, p.W, p.sinks);
      if (on) tiles = (m.sink_end + max(0, (max(kv_lim, 0) + 63) / 64 * 64 - max(m.lo, m.sink_end))) / 64;
    }
    const uint64_t staged = __ballot(on);
    const int32_t incl = (int32_t)wave_scan((uint32_t)tiles), total = __builtin_amdgcn_readlane(incl, 63);
    for (; item < before + total; item += wgs) {
      const int src = __builtin_ctzll(__ballot(item < before + incl));
      const int32_t slot = slots + (int32_t)__popcll(staged & ((1ull << src) - 1));
      if (slot >= p.st.slots) return;  // sequences overlap
      const int32_t lim = __builtin_amdgcn_readlane(kv_lim, src), sink_end = __builtin_amdgcn_readlane(m.sink_end, src);
      const int32_t skip = __builtin_amdgcn_readlane(m.skip, src);
      const int32_t row = 64 * (item - before - __builtin_amdgcn_readlane(incl, src) + __builtin_amdgcn_readlane(tiles, src)) +
                          16 * wave;
      if (row >= p.st.cap) return;  // (a chunk longer than announced)
      const int32_t pos = row < sink_end ? row : row + skip, chunk = pos >> 4, cpp = PAGES ? 1 : p.bs >> 4;
      const bool inside = pos < lim;
      const int32_t phys = inside ? tables[(int64_t)(b0 + src) * p.M + (cpp == 1 ? chunk : chunk / cpp)] : 0;
      const bool ok = phys >= 0 && phys < p.nb;
      if (kvh == 0 && lane == 0) p.st.links[((int64_t)slot * p.st.cap + row) / 16] = ok ? 1 : 0;
      if (!inside) continue;
      const int64_t out = (((int64_t)slot * p.st.cap + row) * p.Hk + kvh) * D, ts = (int64_t)p.Hk * D;
      if constexpr (PAGES) {
        constexpr int DL = D / 8, W = D / 64;  // dims and words of a token per lane
        const int t = lane >> 3, d0 = DL * (lane & 7);
        uint32_t kw[2][W], vw[2 * W];  // K words of tokens t and t + 8; V words hold four dims of both
        uint32_t ks = 0, vs = 0;
#pragma unroll
        for (int j = 0; j < 2 * W; ++j) kw[j / W][j % W] = vw[j] = 0x88888888u;
        if (ok) {
          const uint8_t *blk = p.k + (int64_t)phys * p.kv_ps + kvh * p.kv_hs;
          const uint32_t *kc = reinterpret_cast<const uint32_t *>(blk + f.kcodes) + 2 * W * lane;
          const uint32_t *vc = reinterpret_cast<const uint32_t *>(blk + f.vcodes) + 2 * W * lane;
#pragma unroll
          for (int j = 0; j < 2 * W; ++j) {
            kw[j / W][j % W] = kc[j];
            vw[j] = vc[j];
          }
          ks = *reinterpret_cast<const uint32_t *>(blk + f.kscales + 2 * f.scale_idx(t, d0 / 64));
          vs = *reinterpret_cast<const uint32_t *>(blk + f.vscales + 2 * f.scale_idx(t, d0 / 64));
        }
        auto unpack = [&](uint32_t w, uint32_t (&y)[4]) __attribute__((always_inline)) {
          const half2_t b1032 = {(half_t)1032.0f, (half_t)1032.0f}, b72 = {(half_t)72.0f, (half_t)72.0f};
          const uint32_t w8 = w >> 8;
          y[0] = as_u32(as_half2((w & 0x000F000Fu) | 0x64006400u) - b1032);
          y[1] = as_u32(as_half2((w & 0x00F000F0u) | 0x54005400u) - b72);
          y[2] = as_u32(as_half2((w8 & 0x000F000Fu) | 0x64006400u) - b1032);
          y[3] = as_u32(as_half2((w8 & 0x00F000F0u) | 0x54005400u) - b72);
        };
        auto scaled = [&](uint32_t w, uint32_t (&y)[4]) __attribute__((always_inline)) {
          unpack(w, y);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = as_u32(as_half2(y[i]) * as_half2(vs));
        };
        if (lane < 16) {  // token `lane`
          float first = 0.0f, last = 0.0f;
          if (ok) {
            const half_t *sc = reinterpret_cast<const half_t *>(p.k + (int64_t)phys * p.kv_ps + kvh * p.kv_hs + f.kscales);
            first = (float)sc[f.scale_idx(lane, 0)];
            last = (float)sc[f.scale_idx(lane, D / 64 - 1)];
          }
          // (a scale of 0 makes zeros of its codes below; if the last is, the first serves both)
          float *const dst = p.st.factors + ((int64_t)slot * p.Hk + kvh) * 2 * p.st.cap + row + lane;
          dst[0] = last == 0.0f ? 1.0f : first / last;
          dst[p.st.cap] = (last == 0.0f ? first : last) * p.qk_scale_log2;
        }
        constexpr uint32_t LO = 0x05040100u, HI = 0x07060302u;
        half_t *const ko = p.st.k + out + t * ts + d0, *const vo = p.st.v + out + t * ts + d0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool gone = ((h ? ks >> 16 : ks) & 0x7FFFu) == 0;
#pragma unroll
          for (int j = 0; j < W; ++j) {
            uint32_t y[4];
            unpack(gone ? 0x88888888u : kw[h][j], y);
            *reinterpret_cast<u32x4_t *>(ko + 8 * h * ts + 8 * j) =
                u32x4_t{__builtin_amdgcn_perm(y[1], y[0], LO), __builtin_amdgcn_perm(y[3], y[2], LO),
                        __builtin_amdgcn_perm(y[1], y[0], HI), __builtin_amdgcn_perm(y[3], y[2], HI)};
          }
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
          uint32_t y[4], z[4];
          scaled(vw[2 * j], y);
          scaled(vw[2 * j + 1], z);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t sel = h ? HI : LO;
            *reinterpret_cast<u32x4_t *>(vo + 8 * h * ts + 8 * j) =
                u32x4_t{__builtin_amdgcn_perm(y[1], y[0], sel), __builtin_amdgcn_perm(y[3], y[2], sel),
                        __builtin_amdgcn_perm(z[1], z[0], sel), __builtin_amdgcn_perm(z[3], z[2], sel)};
          }
        }
      } else {
        constexpr int PPR = D / 8, NP = 16 * PPR / 64;  // 16-byte pieces of a row, and per lane
        const int64_t at = (int64_t)phys * p.kv_ps + (int64_t)(16 * (chunk - chunk / cpp * cpp)) * p.kv_ts + kvh * p.kv_hs;
        u32x4_t kx[NP], vx[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const int t = (64 * j + lane) / PPR, d = 8 * (lane % PPR);
          kx[j] = vx[j] = (u32x4_t){};
          if (ok) {
            kx[j] = *reinterpret_cast<const u32x4_t *>(p.k + at + t * p.kv_ts + 2 * d);
            vx[j] = *reinterpret_cast<const u32x4_t *>(p.v + at + t * p.kv_ts + 2 * d);
          }
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const int t = (64 * j + lane) / PPR, d = 8 * (lane % PPR);
          *reinterpret_cast<u32x4_t *>(p.st.k + out + t * ts + d) = kx[j];
          *reinterpret_cast<u32x4_t *>(p.st.v + out + t * ts + d) = vx[j];
        }
      }
    }
    before += total;
    slots += (int32_t)__popcll(staged);
  }
}

// Steps (32 tokens) that a block can need.
static int64_t packed_steps(const memopt_packed_desc &d) {
  return ((int64_t)d.max_blocks_per_seq * d.block_size + 31) / 32;
}

// Query rows per block: 8 or 16 where no sequence has more.
struct PackedPlan {
  int32_t qn, waves, wgs;
  bool rest;       // no sequence has more than kRestRows
  int64_t blocks;  // at most this many
  int32_t min_rows, slots;  // staged sequences
  int64_t cap;
};

// Rows from which a sequence's chunk attends from a staged copy, by the rows of
// the whole batch and all key heads as tiles of 128, which are not split along
// the keys (some 17 us for 1024 of them) as the blocks here are: 512 where there
// are two tiles for each CU, 1024 where there is one, none below. 32 query over 8
// key heads of 128, us staged and not: 32 chunks of 512 rows over contexts of 4096
// 472 and 509, 16 of 512 over 1024 66 and 86; 8 of 1024 over 4096 182 and 263, 2 of
// 2048 (256 tiles) 111 and 130; but 8 of 512 (256 tiles) over 16384 558 and 475, 32 of
// 256 over 4096 320 and 258, one of 1024 (64 tiles) 95 and 45.
static int32_t staged_rows(int64_t rows) {
  const int64_t per_cu = rows / (128LL * compute_units());
  return per_cu >= 2 ? 512 : per_cu >= 1 ? 1024 : INT32_MAX;
}
// Of staged copies at most this much (a prefill budget counts on it: autochunk.py).
static constexpr int64_t kStagedBytes = 2LL << 30;

static PackedPlan packed_plan(const memopt_packed_desc &d) {
  PackedPlan pl = {};
  const int64_t G = d.num_heads / d.num_kv_heads, most = (int64_t)std::min(d.max_query_len, d.tokens) * G;
  pl.qn = most > 16 ? 32 : most > 8 || d.kv_format == MEMOPT_KV_FP16 ? 16 : 8;
  pl.rest = most <= kRestRows;
  // sum over the sequences of ceil(rows / qn)
  pl.blocks = (d.tokens * G + (int64_t)(pl.qn - 1) * std::min(d.batch, d.tokens)) / pl.qn;
  // Workgroups of 4 waves, three to a CU: they hide each other's starts and
  // ends. Where a sequence falls to more than 8 of them and there is enough to
  // read, 12 waves in one workgroup per CU, a third as many partial sums, are
  // faster (us with 4 and 12 waves, 32 query over 8 key heads of 128: one sequence
  // of 131072 tokens 40.0 and 35.1, one of 8000 17.6 and 15.3, 4 of 8000 20.8 and
  // 15.1, 8 of 16000 35.3 and 32.5; but one of 4000 12.6 and 14.1, 4 of 1000 9.5
  // and 12.4, 32 of 2700 to 8192 43.3 and 46.0). fp16 rows take their registers
  // from the ring's share: 8 waves, one workgroup.
  auto wgs = [&](int waves) {
    const int64_t n = (int64_t)resident(waves, pl.qn) * compute_units() / d.num_kv_heads;
    return (int32_t)std::max<int64_t>(1, std::min<int64_t>(n, kMaxParts));
  };
  pl.waves = pl.qn == 32 ? 4 : d.kv_format == MEMOPT_KV_FP16 ? 8 : 4;
  if (pl.waves == 4 && pl.qn <= 16 && wgs(4) > 8LL * d.batch && packed_steps(d) * d.batch * d.head_dim >= 32000)
    pl.waves = 12;
  pl.wgs = wgs(pl.waves);
  pl.min_rows = staged_rows((int64_t)d.tokens * d.num_heads);
  if (most >= pl.min_rows) {
    const int64_t W = std::min(effective_window(d.window_size, d.max_seq_len), 1 << 30);
    const int64_t sinks = std::max(0, d.num_sink_tokens);
    auto up64 = [](int64_t x) { return (x + 63) / 64 * 64; };
    pl.cap = std::min(up64((int64_t)d.max_blocks_per_seq * d.block_size),
                      up64(W + std::min(d.max_query_len, d.tokens)) + 128 + up64(sinks));
    const int64_t fit = kStagedBytes / (pl.cap * d.num_kv_heads * d.head_dim * 4);
    const int64_t most_seqs = std::min<int64_t>(d.batch, d.tokens * G / pl.min_rows);
    pl.slots = (int32_t)std::min(most_seqs, fit);
    // Room for fewer than could come: chunks of which no more than that fit into the batch.
    if (fit < most_seqs) pl.min_rows = (int32_t)(d.tokens * G / (fit + 1) + 1);
  }
  return pl;
}

struct PackedWorkspace {
  // Bytes of the counters; offsets of the (m, l) pairs and of the staged copies' parts.
  int64_t counters, ml, links, factors, k, v, total;
};
static PackedWorkspace packed_workspace(const memopt_packed_desc &d, const PackedPlan &pl) {
  PackedWorkspace w;
  w.counters = (pl.blocks * d.num_kv_heads * 4 + 255) / 256 * 256;
  const int64_t rows = 2LL * pl.wgs * d.num_kv_heads * pl.qn;
  w.ml = w.counters + rows * d.head_dim * 4;
  auto up256 = [](int64_t x) { return (x + 255) / 256 * 256; };
  w.links = up256(w.ml + rows * 8);
  w.factors = up256(w.links + pl.slots * pl.cap / 16);
  w.k = w.factors;
  if (d.kv_format == MEMOPT_KV_INT4) w.k = up256(w.factors + pl.slots * pl.cap * d.num_kv_heads * 8);
  const int64_t staged = pl.slots * pl.cap * d.num_kv_heads * d.head_dim * 2;
  w.v = w.k + staged;
  w.total = w.v + staged;
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

template <int D, int FMT, int QN, int NW, Rest REST>
static void launch_packed(const PackedParams &p, const memopt_packed_desc &d, hipStream_t stream) {
  hipLaunchKernelGGL((packed_kernel<D, FMT, QN, NW, REST>), dim3((unsigned)((int64_t)p.wgs * p.Hk)), dim3(64 * NW), 0, stream,
                     p, d.query_starts, d.context_lens, d.block_tables);
}
template <int D>
static void launch_packed(const PackedParams &p, const memopt_packed_desc &d, const PackedPlan &pl, hipStream_t s) {
  if (d.kv_format == MEMOPT_KV_INT4) {
    if (pl.qn == 32 && pl.rest) launch_packed<D, MEMOPT_KV_INT4, 32, 4, kAllRest>(p, d, s);
    else if (pl.qn == 32) launch_packed<D, MEMOPT_KV_INT4, 32, 4, kShortRest>(p, d, s);
    else if (pl.qn == 16 && pl.waves == 12) launch_packed<D, MEMOPT_KV_INT4, 16, 12, kAllRest>(p, d, s);
    else if (pl.qn == 16) launch_packed<D, MEMOPT_KV_INT4, 16, 4, kAllRest>(p, d, s);
    else if (pl.waves == 12) launch_packed<D, MEMOPT_KV_INT4, 8, 12, kNoRest>(p, d, s);
    else launch_packed<D, MEMOPT_KV_INT4, 8, 4, kNoRest>(p, d, s);
  } else {
    if (pl.qn == 32) launch_packed<D, MEMOPT_KV_FP16, 32, 4, kNoRest>(p, d, s);
    else launch_packed<D, MEMOPT_KV_FP16, 16, 8, kNoRest>(p, d, s);
  }
}

template <int D>
static void launch_stage(const PackedParams &p, const memopt_packed_desc &d, dim3 grid, hipStream_t s) {
  if (d.kv_format == MEMOPT_KV_INT4)
    hipLaunchKernelGGL((stage_kernel<D, MEMOPT_KV_INT4>), grid, dim3(256), 0, s, p, d.query_starts, d.context_lens,
                       d.block_tables);
  else
    hipLaunchKernelGGL((stage_kernel<D, MEMOPT_KV_FP16>), grid, dim3(256), 0, s, p, d.query_starts, d.context_lens,
                       d.block_tables);
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
  MEMOPT_REQUIRE((int64_t)d.max_blocks_per_seq * d.block_size <= 1 << 30, MEMOPT_ERR_UNSUPPORTED,
                 "packed_attention: positions less a window must fit 32 bits: block tables of up to 2^30 tokens");
  const PackedPlan pl = packed_plan(d);
  const PackedWorkspace w = packed_workspace(d, pl);
  MEMOPT_REQUIRE(d.workspace && d.workspace_bytes >= w.total, MEMOPT_ERR_INVALID,
                 "packed_attention: workspace needs " + std::to_string(w.total) + " bytes");
  MEMOPT_REQUIRE((int64_t)d.tokens * d.num_heads <= INT32_MAX - 255 && pl.blocks * packed_steps(d) < (1LL << 31),
                 MEMOPT_ERR_UNSUPPORTED, "packed_attention: too many (row, page) pairs for one call");
  PackedParams p = {};
  p.q = (const half_t *)d.query;
  p.out = (half_t *)d.out;
  p.q_ts = d.q_token_stride;
  p.q_hs = d.q_head_stride;
  p.o_ts = d.o_token_stride;
  p.o_hs = d.o_head_stride;
  p.T = d.tokens;
  p.B = d.batch;
  p.Hq = d.num_heads;
  p.Hk = d.num_kv_heads;
  p.G = d.num_heads / d.num_kv_heads;
  p.by_g = Divisor::of((uint32_t)p.G);
  p.span = pl.qn / p.G + 1;
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
  if (pl.slots > 0) {
    uint8_t *const ws = (uint8_t *)d.workspace;
    p.st = {pl.min_rows, std::min(d.max_query_len, d.tokens), pl.slots, (int32_t)pl.cap, (half_t *)(ws + w.k),
            (half_t *)(ws + w.v), ws + w.links,
            d.kv_format == MEMOPT_KV_INT4 ? (float *)(ws + w.factors) : nullptr};
    const int64_t wgs = std::min<int64_t>(8LL * compute_units() / p.Hk, pl.slots * pl.cap / 64);
    const dim3 grid((unsigned)(std::max<int64_t>(1, wgs) * p.Hk));
    if (d.head_dim == 128) launch_stage<128>(p, d, grid, s);
    else launch_stage<64>(p, d, grid, s);
    if ((rc = check_launch("packed_attention(stage)")) != MEMOPT_OK) return rc;
    const PagedTiles t = {p.q, p.out, p.q_ts, p.q_hs, p.o_ts, p.o_hs, d.query_starts, d.context_lens, p.T, p.B, p.Hk, p.G,
                          d.head_dim, (int32_t)std::min<int64_t>((int64_t)p.M * p.bs, INT32_MAX), p.W, p.sinks,
                          p.qk_scale_log2, p.st};
    if ((rc = launch_paged_tiles(t, s)) != MEMOPT_OK) return rc;
  }
  if (d.head_dim == 128) launch_packed<128>(p, d, pl, s);
  else launch_packed<64>(p, d, pl, s);
  return check_launch("packed_attention");
}
