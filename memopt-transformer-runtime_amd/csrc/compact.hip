// compact.hip — tokens of least weight leave the cache (gfx950).
//
// Of a request's tokens, each key head keeps n = min(keep, live ones): the
// first `sinks`, the last `recent`, and of the others those with the largest
// scores (ties: the first). They stay in their order and become the request's
// whole context: they move to the fresh pages that the ring of free pages
// gives, and the old pages go back to its end. Copying into other pages rather
// than moving up in place makes every row's copy independent of the others
// (in place, a row's new place is another row's old one, so one workgroup
// would have to walk a whole sequence), and leaves the old pages whole.
//
// Three launches. The first counts each request's tokens (a workgroup each).
// The second finds the tokens that stay (a workgroup per request and key head:
// radix selection); the workgroup that ends last also says what each request
// gets, by prefix sums over the requests as in batch.hip. The third copies (a
// wave per 16 new tokens and head) and writes tables and ring.
//
// Measured (medians): one request of 1024 tokens, two heads: 2.5 + 10 + 4 us,
// a chain of launches, reads and barriers (14.8 a call in a captured graph). 16
// requests of up to 8192 tokens, 8 heads, 2048 kept, INT4: 4 + 17.4 + 20.4 us:
// the copies' 71 MB at 3.5 TB/s; the selection's fixed 9 us (four passes of
// four barriers, the plan) and 1 us per 1024 tokens, one workgroup a row. One
// request of 16384 tokens, 8192 kept, fp16: 2.5 + 24 + 13.5 us: eight rows
// leave 248 compute units idle in the selection (sharing a row among several
// workgroups, with a histogram in memory and a launch of 2.5 us per digit or a
// last one to arrive, has not been built).
#include <algorithm>
#include <iterator>

#include "page_format.hpp"
#include "tiles.hpp"

namespace memopt {

struct CompactParams {
  const float *scores;
  float *scores_out;
  int32_t *kept;
  uint8_t *k, *v;
  int64_t nb;
  int32_t N, Hk, D, M, bs, C, L, K, sinks, recent;
  const int32_t *bt, *ctx, *keep, *span;
  int32_t *bt_out, *ctx_out, *status, *ring, *span_out;
  // workspace
  int32_t *stay;    // [N]: tokens that stay per head, -1 where the request is left as it is
  int32_t *holes;   // [N]: 1 where a page of the context is not linked
  int32_t *back;    // [N]: linked pages; then the first place that they get at the ring's end
  int32_t *fresh;   // [N]: the first fresh page's place in the ring, from its front
  int32_t *state;   // [N]: MEMOPT_COMPACT_*, as far as it is known
  int32_t *counts;  // [4]: workgroups of the second launch that ended; the ring's front and pages
  int32_t *marks;   // [nb]
  int32_t in_lds;   // tokens whose orders the selection keeps in LDS
};

static constexpr int32_t kMaxCompacted = 4096;

__device__ __forceinline__ bool page_ok(const CompactParams &p, int32_t page) { return page >= 0 && page < p.nb; }

// Pages of request b's context: 0 where no table can hold that many tokens.
__device__ __forceinline__ int32_t pages_held(const CompactParams &p, int32_t c) {
  return c < 0 || (int64_t)c > (int64_t)p.M * p.bs ? 0 : (c + p.bs - 1) / p.bs;
}

// What a request holds and asks for. A page that two entries list would go
// back to the ring twice, or while the other request still has it: each entry
// leaves its number at the page, and who finds another's there (the second
// launch) tells both requests. Refused requests take part: they keep their pages.
__global__ __launch_bounds__(256) void compact_count_kernel(const CompactParams p) {
  __shared__ int32_t s_part[2][4];
  const int32_t b = blockIdx.x, c = p.ctx[b], keep = p.keep[b];
  const bool bad = c < 0 || (int64_t)c > (int64_t)p.M * p.bs || c > p.L || keep > p.K;
  const int32_t have = pages_held(p, c);
  int32_t live = 0, back = 0;
  for (int32_t i = threadIdx.x; i < have; i += 256) {
    const int32_t page = p.bt[(int64_t)b * p.M + i];
    if (!page_ok(p, page)) continue;
    ++back;
    live += min(p.bs, c - i * p.bs);
    p.marks[page] = b * p.M + i;
  }
  live = wave_sum(live);
  back = wave_sum(back);
  if ((threadIdx.x & 63) == 0) {
    s_part[0][threadIdx.x >> 6] = live;
    s_part[1][threadIdx.x >> 6] = back;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  live = s_part[0][0] + s_part[0][1] + s_part[0][2] + s_part[0][3];
  back = s_part[1][0] + s_part[1][1] + s_part[1][2] + s_part[1][3];
  const bool asks = !bad && keep >= 0 && live > keep;
  p.stay[b] = asks ? keep : -1;
  p.holes[b] = live < c;
  p.back[b] = back;
  p.state[b] = bad ? MEMOPT_COMPACT_INVALID : asks ? MEMOPT_COMPACT_DONE : MEMOPT_COMPACT_LEFT;
  if (b == 0) p.counts[0] = 0;
}

// What each request gets: sums of what is asked decide, sums of what is served
// place; 1024 requests at a time. One workgroup of 1024 threads.
__device__ __forceinline__ void plan_requests(const CompactParams &p, uint32_t (*s_part)[16]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int32_t head = p.span[0] % p.C;
  if (head < 0) head += p.C;
  const int32_t count = min(max(p.span[1], 0), p.C);
  uint32_t asked_need = 0, asked_back = 0, got_need = 0, got_back = 0;
  auto scan = [&](uint32_t a, uint32_t z, uint32_t &ta, uint32_t &tz, uint32_t &ea, uint32_t &ez) {
    ea = wave_scan(a);
    ez = wave_scan(z);
    __syncthreads();
    if (lane == 63) {
      s_part[0][wave] = ea;
      s_part[1][wave] = ez;
    }
    __syncthreads();
    ta = tz = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      if (w == wave) {
        ea = __builtin_elementwise_add_sat(ea, ta);
        ez = __builtin_elementwise_add_sat(ez, tz);
      }
      ta = __builtin_elementwise_add_sat(ta, s_part[0][w]);
      tz = __builtin_elementwise_add_sat(tz, s_part[1][w]);
    }
  };
  for (int32_t b0 = 0; b0 < p.N; b0 += 1024) {
    const int32_t b = b0 + (int32_t)threadIdx.x;
    int32_t st = b < p.N ? __hip_atomic_load(&p.state[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : MEMOPT_COMPACT_INVALID;
    uint32_t need = 0, back = 0, ta, tz, ea, ez;
    const int32_t stay = b < p.N ? p.stay[b] : 0;
    if (st == MEMOPT_COMPACT_DONE) {
      need = (uint32_t)((stay + p.bs - 1) / p.bs);
      back = (uint32_t)p.back[b];
    }
    scan(need, back, ta, tz, ea, ez);
    if (st == MEMOPT_COMPACT_DONE && (__builtin_elementwise_add_sat(asked_need, ea) > (uint32_t)count ||
                                      __builtin_elementwise_add_sat(asked_back, ez) > (uint32_t)(p.C - count)))
      st = MEMOPT_COMPACT_NO_PAGES;
    asked_need = __builtin_elementwise_add_sat(asked_need, ta);
    asked_back = __builtin_elementwise_add_sat(asked_back, tz);
    if (st != MEMOPT_COMPACT_DONE) need = back = 0;
    scan(need, back, ta, tz, ea, ez);
    if (b < p.N) {
      p.status[b] = st;
      p.ctx_out[b] = st == MEMOPT_COMPACT_DONE ? stay : p.ctx[b];
      p.fresh[b] = (int32_t)(got_need + ea - need);
      p.back[b] = (int32_t)(got_back + ez - back);
    }
    got_need += ta;
    got_back += tz;
  }
  if (threadIdx.x == 0) {
    p.counts[1] = head;
    p.counts[2] = count;
    p.span_out[0] = (int32_t)(((int64_t)head + got_need) % p.C);
    p.span_out[1] = count - (int32_t)got_need + (int32_t)got_back;
  }
}

// Scores as integers in their order, above 0 and below ~0; NaN lowest, both zeros alike.
__device__ __forceinline__ uint32_t order_of(float x) {
  uint32_t u = __float_as_uint(x);
  if ((u << 1) == 0) u = 0;
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 1;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
static constexpr uint32_t kGone = 0, kStays = 0xFFFFFFFFu;  // orders of tokens that no score decides about

// The tokens that stay, per request and key head: the order of the last one
// to stay is found digit by digit (8 bits each) from histograms, then
// each wave lists its part of the row. Orders of rows of up to kInLds tokens
// are worked out once and kept in LDS (in registers, the unrolled passes are
// 80 KB of code, whose fetch took longer than they did: 1024 tokens 15 us);
// longer rows are read in every pass. Lanes that meet in one bin or bank wait
// for each other, and scores have few exponents: a bin has sixteen counters
// side by side, for every sixteenth lane.
static constexpr int kInLds = 28672;
struct SelectShared {
  uint4 hist[256][4];
  uint32_t part[16], eq[16], gt[16], bin, above, safe;
};
template <bool LDS>
__device__ __forceinline__ void select_row(const CompactParams &p, SelectShared &sh, uint32_t *s_key, int32_t b,
                                           const float *src, float *dst, int32_t *kept, int32_t n) {
  constexpr int NW = 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t c = p.ctx[b], sinks = min(p.sinks, n), recent0 = c - min(p.recent, n - sinks);
  const bool holes = p.holes[b] != 0;
  auto live = [&](int32_t j) { return !holes || page_ok(p, p.bt[(int64_t)b * p.M + j / p.bs]); };
  auto safe = [&](int32_t j) { return j < sinks || j >= recent0; };
  auto order_at = [&](int32_t j, float x) { return !live(j) ? kGone : safe(j) ? kStays : order_of(x); };
  // Wave w takes tokens [j0, j1), 64 at a time.
  const int32_t part = ((c + NW - 1) / NW + 63) / 64 * 64;
  const int32_t j0 = min(wave * part, c), j1 = min(j0 + part, c);
  // Eight reads before the first is looked at, past the end the last token's: under a condition, or behind a store,
  // each would be waited for by itself.
  constexpr int U = 8;
  auto each = [&](auto f) __attribute__((always_inline)) {  // f(token, score), all lanes together
    for (int32_t base = j0; base < j1; base += 64 * U) {
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = src[min(base + 64 * u + lane, c - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (base + 64 * u < j1) f(base + 64 * u + lane, x[u]);
    }
  };
  if constexpr (LDS)  // (each wave reads its own later)
    each([&](int32_t j, float x) __attribute__((always_inline)) {
      if (j < j1) s_key[j] = order_at(j, x);
    });
  auto each_key = [&](auto f) __attribute__((always_inline)) {  // f(order, of a token or kGone), all lanes together
    if constexpr (LDS) {
#pragma unroll 4
      for (int32_t j = j0 + lane; j - lane < j1; j += 64) f(j < j1 ? s_key[j] : kGone);
    } else {
      each([&](int32_t j, float x) __attribute__((always_inline)) { f(j < j1 ? order_at(j, x) : kGone); });
    }
  };

  // Protected tokens.
  if (threadIdx.x == 0) sh.safe = 0;
  __syncthreads();
  if (holes) {
    uint32_t k = 0;
    for (int32_t j = threadIdx.x; j < c; j += 1024) k += safe(j) && live(j);
    k = (uint32_t)wave_sum((int32_t)k);
    if (lane == 0) atomicAdd(&sh.safe, k);
  } else if (threadIdx.x == 0) {
    sh.safe = (uint32_t)(sinks + c - recent0);  // (n <= c: they do not overlap)
  }
  __syncthreads();
  uint32_t want = (uint32_t)n - sh.safe;  // to be taken by score
  uint32_t prefix = kStays - 1;           // (above every score's order)
  if (want > 0) {
    prefix = 0;
    uint32_t mask = 0;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      (&sh.hist[0][0])[threadIdx.x] = uint4{0, 0, 0, 0};
      __syncthreads();
      each_key([&](uint32_t u) __attribute__((always_inline)) {
        if (u != kGone && u != kStays && (u & mask) == prefix)
          atomicAdd(reinterpret_cast<uint32_t *>(sh.hist[(u >> shift) & 255]) + (lane & 15), 1u);
      });
      __syncthreads();
      // Bins from the top: thread t < 256 holds bin 255 - t.
      const int bin = 255 - (int)threadIdx.x;
      uint32_t held = 0, incl = 0;
      if (wave < 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 x = sh.hist[bin][i];
          held += (x.x + x.y) + (x.z + x.w);
        }
        incl = wave_scan(held);
        if (lane == 63) sh.part[wave] = incl;
      }
      __syncthreads();
      if (wave < 4) {
        uint32_t before = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) before += w < wave ? sh.part[w] : 0;
        const uint32_t end = before + incl, begin = end - held;
        if (begin < want && want <= end) {  // (one thread: the last token to stay is in its bin)
          sh.bin = (uint32_t)bin;
          sh.above = begin;
        }
      }
      __syncthreads();
      prefix |= sh.bin << shift;
      mask |= 255u << shift;
      want -= sh.above;
    }
  }
  // `want` tokens of the order `prefix` stay, the first ones; all above it do.
  uint32_t gt = 0, eq = 0;
  each_key([&](uint32_t u) __attribute__((always_inline)) {
    gt += (uint32_t)__popcll(__ballot(u > prefix));
    eq += (uint32_t)__popcll(__ballot(u == prefix));
  });
  if (lane == 0) {
    sh.gt[wave] = gt;
    sh.eq[wave] = eq;
  }
  __syncthreads();
  uint32_t at = 0, ties = 0;
  for (int w = 0; w < wave; ++w) {
    at += sh.gt[w] + min(sh.eq[w], want - min(want, ties));
    ties += sh.eq[w];
  }
  const uint64_t below = (1ull << lane) - 1;
  each([&](int32_t j, float x) __attribute__((always_inline)) {
    const uint32_t u = j >= j1 ? kGone : LDS ? s_key[j] : order_at(j, x);
    const uint64_t tie = __ballot(u == prefix);
    const bool take = u > prefix || (u == prefix && ties + (uint32_t)__popcll(tie & below) < want);
    const uint64_t all = __ballot(take);
    const uint32_t i = at + (uint32_t)__popcll(all & below);
    if (take && i < (uint32_t)n) {  // (never past n, unless the scores change under the call)
      kept[i] = j;
      dst[i] = x;
    }
    at += (uint32_t)__popcll(all);
    ties += (uint32_t)__popcll(tie);
  });
  for (int32_t j = n + (int32_t)threadIdx.x; j < p.L; j += 1024) dst[j] = 0.0f;
  for (int32_t j = n + (int32_t)threadIdx.x; j < p.K; j += 1024) kept[j] = -1;
}

// A row that stays as it is.
__device__ __forceinline__ void leave_row(const CompactParams &p, int64_t unit, int32_t threads) {
  for (int32_t j = threadIdx.x; j < p.L; j += threads) p.scores_out[unit * p.L + j] = p.scores[unit * p.L + j];
  for (int32_t j = threadIdx.x; j < p.K; j += threads) p.kept[unit * p.K + j] = -1;
}

__global__ __launch_bounds__(1024) void compact_select_kernel(const CompactParams p) {
  __shared__ SelectShared sh;
  extern __shared__ uint32_t s_key[];  // [in_lds]
  __shared__ uint32_t s_part[2][16];
  __shared__ int32_t s_last;
  const int32_t h = blockIdx.x, b = blockIdx.y;
  const int64_t unit = (int64_t)b * p.Hk + h;
  const int32_t n = p.stay[b], c = p.ctx[b];
  if (h == 0) {
    const int32_t have = pages_held(p, c);
    // (a refused request stays one: whether it is does not change in this launch)
    auto shares = [&](int32_t who) {
      if (__hip_atomic_load(&p.state[who], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != MEMOPT_COMPACT_INVALID)
        __hip_atomic_store(&p.state[who], MEMOPT_COMPACT_SHARED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    for (int32_t i = threadIdx.x; i < have; i += 1024) {
      const int32_t page = p.bt[(int64_t)b * p.M + i];
      if (!page_ok(p, page)) continue;
      const int32_t id = p.marks[page];
      if (id == b * p.M + i) continue;
      shares(b);
      shares(id / p.M);
    }
  }
  const float *src = p.scores + unit * p.L;
  float *dst = p.scores_out + unit * p.L;
  int32_t *kept = p.kept + unit * p.K;
  if (n < 0) leave_row(p, unit, 1024);
  else if (c <= p.in_lds) select_row<true>(p, sh, s_key, b, src, dst, kept, n);
  else select_row<false>(p, sh, s_key, b, src, dst, kept, n);
  // The last workgroup to get here has all states before it: they alone pass between workgroups, by agent-scope
  // stores that have arrived once they are waited for (a fence would write the whole L2 back).
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    s_last = __hip_atomic_fetch_add(&p.counts[0], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.Hk * p.N - 1;
  __syncthreads();
  if (s_last) plan_requests(p, s_part);
}

// A request's tables and its old pages' places at the ring's end; what the
// second launch wrote for one that is not served after all. One workgroup.
__device__ __forceinline__ void write_tables(const CompactParams &p, int32_t b) {
  __shared__ int32_t s_count[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)b * p.M;
  if (p.status[b] != MEMOPT_COMPACT_DONE) {
    for (int32_t i = threadIdx.x; i < p.M; i += 256) p.bt_out[row + i] = p.bt[row + i];
    if (p.stay[b] >= 0)
      for (int32_t h = 0; h < p.Hk; ++h) leave_row(p, (int64_t)b * p.Hk + h, 256);
    return;
  }
  const int32_t need = (p.stay[b] + p.bs - 1) / p.bs, have = (p.ctx[b] + p.bs - 1) / p.bs;
  for (int32_t i = threadIdx.x; i < p.M; i += 256)
    p.bt_out[row + i] = i < need ? p.ring[(int32_t)(((int64_t)p.counts[1] + p.fresh[b] + i) % p.C)] : -1;
  int32_t at = p.back[b];
  for (int32_t i0 = 0; i0 < have; i0 += 256) {
    const int32_t i = i0 + (int32_t)threadIdx.x, page = i < have ? p.bt[row + i] : -1;
    const uint64_t m = __ballot(page_ok(p, page));
    if (lane == 0) s_count[wave] = (int32_t)__popcll(m);
    __syncthreads();
    int32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      before += w < wave ? s_count[w] : 0;
      all += s_count[w];
    }
    if (page_ok(p, page))
      p.ring[(int32_t)(((int64_t)p.counts[1] + p.counts[2] + at + before + __popcll(m & ((1ull << lane) - 1))) % p.C)] = page;
    at += all;
    __syncthreads();
  }
}

// The copies: a wave per 16 new tokens and head.
template <int FMT, int D>
__global__ __launch_bounds__(256) void compact_move_kernel(const CompactParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x == 0) return write_tables(p, blockIdx.y);
  const int32_t h = (int32_t)((blockIdx.x - 1) % p.Hk), chunk = (int32_t)((blockIdx.x - 1) / p.Hk) * 4 + wave, b = blockIdx.y;
  const int32_t n = p.stay[b], i0 = 16 * chunk;
  if (i0 >= n || p.status[b] != MEMOPT_COMPACT_DONE) return;
  const int64_t unit = (int64_t)b * p.Hk + h;
  const int32_t page = __builtin_amdgcn_readfirstlane(
      p.ring[(int32_t)(((int64_t)p.counts[1] + p.fresh[b] + i0 / p.bs) % p.C)]);
  if (!page_ok(p, page)) return;  // (the ring held something that is no page)
  // Old page and place of new token i0 + t, in lane t.
  const int32_t mine = i0 + (lane & 15) < n ? p.kept[unit * p.K + i0 + (lane & 15)] : -1;
  // (Only tokens of linked pages are kept; where scores change under the call a place of the list may be left as it was,
  // and hold any number.)
  const int32_t entry = mine < 0 || mine >= p.ctx[b] ? -1 : p.bt[(int64_t)b * p.M + mine / p.bs];
  const int32_t old = page_ok(p, entry) ? entry : -1, at = mine < 0 ? 0 : mine % p.bs;
  if constexpr (FMT == MEMOPT_KV_INT4) {
    // Lane 8 q + c owns tokens q and q + 8 of the new block, as in page_format.hpp.
    constexpr int BPL = D / 8, G = D / 64, W = BPL / 4;  // bytes and words of a lane's K (and of its V)
    const int q = lane >> 3, c = lane & 7;
    const int64_t block = Int4Page(D).block;
    const int32_t pg[2] = {__shfl(old, q, 64), __shfl(old, q + 8, 64)}, t[2] = {__shfl(at, q, 64), __shfl(at, q + 8, 64)};
    uint8_t *to = p.k + ((int64_t)page * p.Hk + h) * block;
    uint32_t kw[2][W / 2 ? W / 2 : 1], vw[2][W];
    uint16_t sk[2] = {0, 0};
    // scales: lane 8 q + c, c < 2 G: K (c < G) or V, group c % G
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint8_t *from = pg[x] >= 0 ? p.k + ((int64_t)pg[x] * p.Hk + h) * block : to;
      const int src = pg[x] >= 0 ? 8 * (t[x] & 7) + c : lane, half = pg[x] >= 0 ? t[x] >> 3 : x;
      const uint32_t *kp = reinterpret_cast<const uint32_t *>(from + src * BPL + half * (BPL / 2));
      const uint32_t *vp = reinterpret_cast<const uint32_t *>(from + 8 * D + src * BPL);
#pragma unroll
      for (int i = 0; i < W / 2; ++i) kw[x][i] = kp[i];
#pragma unroll
      for (int i = 0; i < W; ++i) vw[x][i] = (vp[i] >> (16 * half)) & 0xFFFFu;
      if (c < 2 * G) {
        const int tok = pg[x] >= 0 ? t[x] : q + 8 * x;
        sk[x] = reinterpret_cast<const uint16_t *>(from + 16 * D)[c * 16 + 2 * (tok & 7) + (tok >> 3)];
      }
    }
    uint32_t *kd = reinterpret_cast<uint32_t *>(to + lane * BPL), *vd = reinterpret_cast<uint32_t *>(to + 8 * D + lane * BPL);
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      kd[i] = kw[0][i];
      kd[W / 2 + i] = kw[1][i];
    }
#pragma unroll
    for (int i = 0; i < W; ++i) vd[i] = vw[0][i] | vw[1][i] << 16;
    if (c < 2 * G) reinterpret_cast<uint32_t *>(to + 16 * D)[c * 8 + q] = sk[0] | (uint32_t)sk[1] << 16;
  } else {
    constexpr int LPR = D / 8, RPW = 64 / LPR;  // lanes of a row, rows of a copy
    const int64_t row = (int64_t)p.Hk * D * 2;
#pragma unroll
    for (int t = 0; t < 16 / RPW; ++t) {
      const int tok = t * RPW + lane / LPR;
      const int32_t pg = __shfl(old, tok, 64), off = __shfl(at, tok, 64);
      if (pg < 0) continue;
      const int64_t from = ((int64_t)pg * p.bs + off) * row + h * (D * 2) + 16 * (lane % LPR);
      const int64_t to = ((int64_t)page * p.bs + i0 % p.bs + tok) * row + h * (D * 2) + 16 * (lane % LPR);
      *reinterpret_cast<uint4 *>(p.k + to) = *reinterpret_cast<const uint4 *>(p.k + from);
      *reinterpret_cast<uint4 *>(p.v + to) = *reinterpret_cast<const uint4 *>(p.v + from);
    }
  }
}

// A call without requests: the ring stays, its span within its bounds.
__global__ void compact_no_requests_kernel(const CompactParams p) {
  const int32_t head = p.span[0] % p.C, count = min(max(p.span[1], 0), p.C);
  p.span_out[0] = head < 0 ? head + p.C : head;
  p.span_out[1] = count;
}

static int64_t compact_workspace(const memopt_compact_desc &d) {
  return ((5 * (int64_t)d.num_requests + 4 + d.num_kv_blocks) * 4 + 255) / 256 * 256;
}

// Whether a result shares memory with an input or another result (free_span_out may be free_span itself).
static bool compact_overlaps(const memopt_compact_desc &d) {
  const int64_t N = d.num_requests, rows = N * d.num_kv_heads;
  const int64_t cache = d.kv_format == MEMOPT_KV_INT4 ? d.num_kv_blocks * d.num_kv_heads * Int4Page(d.head_dim).block
                                                      : d.num_kv_blocks * d.num_kv_heads * d.block_size * d.head_dim * 2;
  const Memory out[] = {{d.scores_out, 4 * rows * d.scores_len}, {d.kept, 4 * rows * d.max_keep},
                        {d.block_tables_out, 4 * N * d.max_blocks_per_seq}, {d.context_lens_out, 4 * N}, {d.status, 4 * N},
                        {d.free_span_out, 8}};
  const Memory in[] = {{d.scores, 4 * rows * d.scores_len}, {d.key_cache, cache},
                       {d.value_cache, d.kv_format == MEMOPT_KV_INT4 ? 0 : cache}, {d.block_tables, 4 * N * d.max_blocks_per_seq},
                       {d.context_lens, 4 * N}, {d.keep, 4 * N}, {d.free_pages, 4LL * d.num_free_pages},
                       {d.free_span_out == d.free_span ? nullptr : d.free_span, d.free_span_out == d.free_span ? 0 : 8}};
  for (size_t i = 0; i < std::size(out); ++i) {
    for (const Memory &x : in)
      if (overlap(out[i], x)) return true;
    for (size_t k = 0; k < i; ++k)
      if (overlap(out[i], out[k])) return true;
  }
  return false;
}

static int validate_compact(const memopt_compact_desc &d) {
  MEMOPT_REQUIRE(d.num_requests >= 0 && d.scores_len >= 0 && d.max_keep >= 0, MEMOPT_ERR_INVALID,
                 "compact_cache: negative size");
  MEMOPT_REQUIRE(d.num_kv_heads > 0 && d.num_kv_blocks > 0 && d.max_blocks_per_seq > 0 && d.block_size > 0 &&
                     d.num_free_pages > 0,
                 MEMOPT_ERR_INVALID, "compact_cache: empty cache, block table or ring");
  MEMOPT_REQUIRE(d.num_requests <= kMaxCompacted, MEMOPT_ERR_UNSUPPORTED,
                 "compact_cache: more than " + std::to_string(kMaxCompacted) + " requests");
  MEMOPT_REQUIRE(d.kv_format == MEMOPT_KV_FP16 || d.kv_format == MEMOPT_KV_INT4, MEMOPT_ERR_UNSUPPORTED,
                 "compact_cache: the cache must be an fp16 pool or INT4 pages");
  MEMOPT_REQUIRE(d.head_dim == 64 || d.head_dim == 128, MEMOPT_ERR_UNSUPPORTED,
                 "compact_cache: head_dim must be 64 or 128");
  MEMOPT_REQUIRE(d.kv_format == MEMOPT_KV_FP16 ? d.block_size % 16 == 0 : d.block_size == 16, MEMOPT_ERR_UNSUPPORTED,
                 "compact_cache: pages must hold 16 tokens (fp16 pools: a multiple of 16)");
  MEMOPT_REQUIRE((int64_t)d.max_blocks_per_seq * d.block_size <= 1 << 30 && d.scores_len <= 1 << 30 &&
                     d.max_keep <= d.scores_len && d.num_kv_blocks <= INT32_MAX &&
                     (int64_t)d.num_requests * d.max_blocks_per_seq <= INT32_MAX,
                 MEMOPT_ERR_UNSUPPORTED,
                 "compact_cache: block tables and scores of up to 2^30 tokens, no more of them kept than there are scores");
  MEMOPT_REQUIRE(d.num_kv_heads <= 65535 && (((int64_t)d.max_keep / 64 + 1) * d.num_kv_heads + 1) * std::max(1, d.num_requests) < (1LL << 24) &&
                     (int64_t)d.num_kv_heads * d.num_requests < (1LL << 22),
                 MEMOPT_ERR_UNSUPPORTED, "compact_cache: too many pages for one call");
  return MEMOPT_OK;
}

}  // namespace memopt

using namespace memopt;

extern "C" int memopt_compact_workspace_size(const memopt_compact_desc *desc, int64_t *bytes) {
  MEMOPT_REQUIRE(desc && bytes, MEMOPT_ERR_INVALID, "compact_workspace_size: null pointer");
  *bytes = 0;
  int rc = validate_compact(*desc);
  if (rc != MEMOPT_OK || desc->num_requests == 0) return rc;
  *bytes = compact_workspace(*desc);
  return MEMOPT_OK;
}

extern "C" int memopt_compact_cache(const memopt_compact_desc *desc, void *stream) {
  MEMOPT_REQUIRE(desc, MEMOPT_ERR_INVALID, "compact_cache: null descriptor");
  const memopt_compact_desc &d = *desc;
  int rc = validate_compact(d);
  if (rc != MEMOPT_OK) return rc;
  MEMOPT_REQUIRE(d.free_span && d.free_span_out && d.free_pages, MEMOPT_ERR_INVALID, "compact_cache: null pointer");
  MEMOPT_REQUIRE(d.num_requests == 0 ||
                     (d.key_cache && (d.value_cache || d.kv_format == MEMOPT_KV_INT4) && d.block_tables && d.context_lens &&
                      d.keep && d.block_tables_out && d.context_lens_out && d.status &&
                      (d.scores_len == 0 || (d.scores && d.scores_out)) && (d.max_keep == 0 || d.kept)),
                 MEMOPT_ERR_INVALID, "compact_cache: null pointer");
  MEMOPT_REQUIRE(d.num_requests == 0 ||
                     ((d.scores_len == 0 || d.scores_out != d.scores) && d.block_tables_out != d.block_tables &&
                      d.context_lens_out != d.context_lens),
                 MEMOPT_ERR_INVALID, "compact_cache: results must not overlap the inputs");
  MEMOPT_REQUIRE(((uintptr_t)d.key_cache & 15) == 0 && ((uintptr_t)d.value_cache & 15) == 0 &&
                     ((uintptr_t)d.workspace & 15) == 0,
                 MEMOPT_ERR_INVALID, "compact_cache: caches and workspace must be 16-byte aligned");
  const int64_t need = d.num_requests == 0 ? 0 : compact_workspace(d);
  MEMOPT_REQUIRE(need == 0 || (d.workspace && d.workspace_bytes >= need), MEMOPT_ERR_INVALID,
                 "compact_cache: workspace needs " + std::to_string(need) + " bytes");
  MEMOPT_REQUIRE(d.num_requests == 0 || !compact_overlaps(d), MEMOPT_ERR_INVALID,
                 "compact_cache: results must not overlap the inputs, nor each other");
  CompactParams p = {};
  p.scores = d.scores;
  p.scores_out = d.scores_out;
  p.kept = d.kept;
  p.k = (uint8_t *)d.key_cache;
  p.v = (uint8_t *)d.value_cache;
  p.nb = d.num_kv_blocks;
  p.N = d.num_requests;
  p.Hk = d.num_kv_heads;
  p.D = d.head_dim;
  p.M = d.max_blocks_per_seq;
  p.bs = d.block_size;
  p.C = d.num_free_pages;
  p.L = d.scores_len;
  p.K = d.max_keep;
  p.sinks = std::max(0, d.num_sink_tokens);
  p.recent = std::max(0, d.num_recent_tokens);
  p.bt = d.block_tables;
  p.ctx = d.context_lens;
  p.keep = d.keep;
  p.span = d.free_span;
  p.bt_out = d.block_tables_out;
  p.ctx_out = d.context_lens_out;
  p.status = d.status;
  p.ring = d.free_pages;
  p.span_out = d.free_span_out;
  p.stay = (int32_t *)d.workspace;
  p.holes = p.stay + p.N;
  p.back = p.holes + p.N;
  p.fresh = p.back + p.N;
  p.state = p.fresh + p.N;
  p.counts = p.state + p.N;
  p.marks = p.counts + 4;
  hipStream_t s = (hipStream_t)stream;
  if (p.N == 0) {
    hipLaunchKernelGGL(compact_no_requests_kernel, dim3(1), dim3(1), 0, s, p);
    return check_launch("compact_cache");
  }
  hipLaunchKernelGGL(compact_count_kernel, dim3(p.N), dim3(256), 0, s, p);
  if ((rc = check_launch("compact_cache(count)")) != MEMOPT_OK) return rc;
  // (no request is longer than its table or its scores)
  p.in_lds = (int32_t)std::min<int64_t>(kInLds, std::min<int64_t>((int64_t)p.M * p.bs, p.L));
  const hipError_t set = allow_lds<&compact_select_kernel>(4 * kInLds);
  MEMOPT_REQUIRE(set == hipSuccess, MEMOPT_ERR_HIP, std::string("compact_cache: ") + hipGetErrorString(set));
  hipLaunchKernelGGL(compact_select_kernel, dim3(p.Hk, p.N), dim3(1024), 4 * p.in_lds, s, p);
  if ((rc = check_launch("compact_cache(select)")) != MEMOPT_OK) return rc;
  const dim3 grid((unsigned)(((int64_t)p.K + 63) / 64 * p.Hk + 1), p.N);
  if (d.kv_format == MEMOPT_KV_INT4) {
    if (p.D == 128) hipLaunchKernelGGL((compact_move_kernel<MEMOPT_KV_INT4, 128>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((compact_move_kernel<MEMOPT_KV_INT4, 64>), grid, dim3(256), 0, s, p);
  } else {
    if (p.D == 128) hipLaunchKernelGGL((compact_move_kernel<MEMOPT_KV_FP16, 128>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((compact_move_kernel<MEMOPT_KV_FP16, 64>), grid, dim3(256), 0, s, p);
  }
  return check_launch("compact_cache(move)");
}
