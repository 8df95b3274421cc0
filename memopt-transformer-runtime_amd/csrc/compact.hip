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
// Three launches: what each request gets (one workgroup: prefix sums over the
// requests, as in batch.hip), which tokens stay (one workgroup per request and
// key head: radix selection), and the copies (one wave per page and head).
#include <algorithm>

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
  int32_t *stay;   // [N]: tokens that stay per head, -1 where the request is left as it is
  int32_t *holes;  // [N]: 1 where a page of the context is not linked
  int32_t *marks;  // [nb]
};

static constexpr int32_t kMaxCompacted = 4096;

__device__ __forceinline__ bool page_ok(const CompactParams &p, int32_t page) { return page >= 0 && page < p.nb; }

// Live tokens of a row's first `have` pages, and whether a page is missing. One wave.
__device__ __forceinline__ int32_t live_tokens(const CompactParams &p, int32_t b, int32_t c, int32_t have) {
  const int lane = threadIdx.x & 63;
  int32_t live = 0;
  for (int32_t i = lane; i < have; i += 64)
    if (page_ok(p, p.bt[(int64_t)b * p.M + i])) live += min(p.bs, c - i * p.bs);
  return wave_sum(live);
}

// What each request gets: fresh pages in request order while they last.
__global__ __launch_bounds__(1024) void compact_plan_kernel(const CompactParams p) {
  __shared__ int32_t s_need[kMaxCompacted], s_back[kMaxCompacted], s_status[kMaxCompacted];
  __shared__ uint32_t s_part[2][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int32_t head = p.span[0] % p.C;
  if (head < 0) head += p.C;
  const int32_t count = min(max(p.span[1], 0), p.C);
  // A page that two entries list would go back twice: each entry leaves its
  // number at the page, and who finds another's tells both requests.
  for (int32_t b = wave; b < p.N; b += 16) {
    const int32_t c = p.ctx[b], keep = p.keep[b];
    const bool bad = c < 0 || (int64_t)c > (int64_t)p.M * p.bs || c > p.L || keep > p.K;
    const int32_t have = bad ? 0 : (c + p.bs - 1) / p.bs;
    const int32_t live = live_tokens(p, b, c, have), n = min(keep, live);
    const bool asks = !bad && keep >= 0 && live > keep;
    int32_t back = 0;
    for (int32_t i = lane; i < have; i += 64) {
      const int32_t page = p.bt[(int64_t)b * p.M + i];
      if (!page_ok(p, page)) continue;
      ++back;
      __hip_atomic_store(&p.marks[page], b * p.M + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    back = wave_sum(back);
    if (lane == 0) {
      s_status[b] = bad ? MEMOPT_COMPACT_INVALID : asks ? MEMOPT_COMPACT_DONE : MEMOPT_COMPACT_LEFT;
      s_need[b] = asks ? (n + p.bs - 1) / p.bs : 0;
      s_back[b] = asks ? back : 0;
      p.stay[b] = asks ? n : -1;
      p.holes[b] = live < c;
    }
  }
  __threadfence();
  __syncthreads();
  for (int32_t b = wave; b < p.N; b += 16) {
    if (s_status[b] == MEMOPT_COMPACT_INVALID) continue;
    const int32_t have = (p.ctx[b] + p.bs - 1) / p.bs;
    for (int32_t i = lane; i < have; i += 64) {
      const int32_t page = p.bt[(int64_t)b * p.M + i];
      if (!page_ok(p, page)) continue;
      const int32_t id = __hip_atomic_load(&p.marks[page], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (id != b * p.M + i) {
        atomicExch(&s_status[b], MEMOPT_COMPACT_SHARED);
        atomicExch(&s_status[id / p.M], MEMOPT_COMPACT_SHARED);
      }
    }
  }
  __syncthreads();
  // Requests in order, 1024 at a time: sums of what is asked decide, sums of what is served place.
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
    int32_t st = b < p.N ? s_status[b] : MEMOPT_COMPACT_INVALID;
    uint32_t need = 0, back = 0, ta, tz, ea, ez;
    if (st == MEMOPT_COMPACT_DONE) {
      need = (uint32_t)s_need[b];
      back = (uint32_t)s_back[b];
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
      const int32_t c = p.ctx[b];
      if (st != MEMOPT_COMPACT_DONE) p.stay[b] = -1;
      p.status[b] = s_status[b] = st;
      p.ctx_out[b] = st == MEMOPT_COMPACT_DONE ? p.stay[b] : c;
      s_need[b] = (int32_t)(got_need + ea - need);  // first fresh page, first place at the ring's end
      s_back[b] = (int32_t)(got_back + ez - back);
    }
    got_need += ta;
    got_back += tz;
  }
  __syncthreads();
  for (int32_t b = wave; b < p.N; b += 16) {
    const int64_t row = (int64_t)b * p.M;
    if (s_status[b] != MEMOPT_COMPACT_DONE) {
      for (int32_t i = lane; i < p.M; i += 64) p.bt_out[row + i] = p.bt[row + i];
      continue;
    }
    const int32_t need = (__hip_atomic_load(&p.stay[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + p.bs - 1) / p.bs;
    const int32_t have = (p.ctx[b] + p.bs - 1) / p.bs;
    for (int32_t i = lane; i < p.M; i += 64)
      p.bt_out[row + i] = i < need ? p.ring[(int32_t)(((int64_t)head + s_need[b] + i) % p.C)] : -1;
    int32_t at = s_back[b];
    for (int32_t i0 = 0; i0 < have; i0 += 64) {
      const int32_t page = i0 + lane < have ? p.bt[row + i0 + lane] : -1;
      const uint64_t m = __ballot(page_ok(p, page));
      if (page_ok(p, page))
        p.ring[(int32_t)(((int64_t)head + count + at + __popcll(m & ((1ull << lane) - 1))) % p.C)] = page;
      at += (int32_t)__popcll(m);
    }
  }
  if (threadIdx.x == 0) {
    p.span_out[0] = (int32_t)(((int64_t)head + got_need) % p.C);
    p.span_out[1] = count - (int32_t)got_need + (int32_t)got_back;
  }
}

// Scores as integers in their order; NaN lowest, both zeros alike.
__device__ __forceinline__ uint32_t order_of(float x) {
  uint32_t u = __float_as_uint(x);
  if ((u << 1) == 0) u = 0;
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The tokens that stay, per request and key head: the value of the last one
// to stay is found digit by digit (11, 11 and 10 bits) from histograms, then
// each wave lists its part of the row in order.
__global__ __launch_bounds__(1024) void compact_select_kernel(const CompactParams p) {
  constexpr int NW = 16;
  __shared__ uint32_t s_hist[2048];
  __shared__ uint32_t s_part[NW], s_eq[NW], s_gt[NW], s_bin, s_above, s_safe;
  const int32_t h = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)b * p.Hk + h;
  const float *src = p.scores + unit * p.L;
  float *dst = p.scores_out + unit * p.L;
  int32_t *kept = p.kept + unit * p.K;
  const int32_t n = p.stay[b];
  if (n < 0) {
    for (int32_t j = threadIdx.x; j < p.L; j += 1024) dst[j] = src[j];
    for (int32_t j = threadIdx.x; j < p.K; j += 1024) kept[j] = -1;
    return;
  }
  const int32_t c = p.ctx[b], sinks = min(p.sinks, n), recent0 = c - min(p.recent, n - sinks);
  const bool holes = p.holes[b] != 0;
  auto live = [&](int32_t j) { return !holes || page_ok(p, p.bt[(int64_t)b * p.M + j / p.bs]); };
  auto safe = [&](int32_t j) { return j < sinks || j >= recent0; };

  // Protected tokens.
  if (threadIdx.x == 0) s_safe = 0;
  __syncthreads();
  if (holes) {
    uint32_t x = 0;
    for (int32_t j = threadIdx.x; j < c; j += 1024) x += safe(j) && live(j);
    x = (uint32_t)wave_sum((int32_t)x);
    if (lane == 0) atomicAdd(&s_safe, x);
  } else if (threadIdx.x == 0) {
    s_safe = (uint32_t)(sinks + c - recent0);  // (n <= c: they do not overlap)
  }
  __syncthreads();
  uint32_t want = (uint32_t)n - s_safe;  // to be taken by score
  uint32_t prefix = 0, mask = 0;
  if (want > 0) {
    constexpr int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = shifts[pass];
      const uint32_t digits = (1u << widths[pass]) - 1;
      for (int i = threadIdx.x; i < 2048; i += 1024) s_hist[i] = 0;
      __syncthreads();
      for (int32_t j = threadIdx.x; j < c; j += 1024) {
        if (safe(j) || !live(j)) continue;
        const uint32_t u = order_of(src[j]);
        if ((u & mask) == prefix) atomicAdd(&s_hist[(u >> shift) & digits], 1u);
      }
      __syncthreads();
      // Bins from the top: thread t holds bins 2047 - 2 t and 2046 - 2 t.
      const int top = 2047 - 2 * (int)threadIdx.x;
      const uint32_t x0 = s_hist[top], x1 = s_hist[top - 1], incl = wave_scan(x0 + x1);
      if (lane == 63) s_part[wave] = incl;
      __syncthreads();
      uint32_t before = 0;
      for (int w = 0; w < wave; ++w) before += s_part[w];
      const uint32_t end = before + incl, begin = end - x0 - x1;
      if (begin < want && want <= end) {  // (one thread: the last token to stay is in one of its bins)
        const bool first = want <= begin + x0;
        s_bin = (uint32_t)(first ? top : top - 1);
        s_above = first ? begin : begin + x0;
      }
      __syncthreads();
      prefix |= s_bin << shift;
      mask |= digits << shift;
      want -= s_above;
      __syncthreads();
    }
  } else {
    prefix = 0xFFFFFFFFu;  // (no score reaches it)
  }
  // `want` tokens of the value `prefix` stay, the first ones; all above it do.
  const int32_t part = ((c + NW - 1) / NW + 63) / 64 * 64;
  const int32_t j0 = min(wave * part, c), j1 = min(j0 + part, c);
  uint32_t gt = 0, eq = 0;
  auto kind = [&](int32_t j, float &x) {  // 2: stays, 1: stays while there are ties to take
    if (j >= j1) return 0;
    x = src[j];
    if (!live(j)) return 0;
    if (safe(j)) return 2;
    const uint32_t u = order_of(x);
    return u > prefix ? 2 : u == prefix ? 1 : 0;
  };
  for (int32_t j = j0 + lane; j - lane < j1; j += 64) {
    float x;
    const int k = kind(j, x);
    gt += (uint32_t)__popcll(__ballot(k == 2));
    eq += (uint32_t)__popcll(__ballot(k == 1));
  }
  if (lane == 0) {
    s_gt[wave] = gt;
    s_eq[wave] = eq;
  }
  __syncthreads();
  uint32_t at = 0, ties = 0;
  for (int w = 0; w < wave; ++w) {
    at += s_gt[w] + min(s_eq[w], want - min(want, ties));
    ties += s_eq[w];
  }
  const uint64_t below = (1ull << lane) - 1;
  for (int32_t j = j0 + lane; j - lane < j1; j += 64) {
    float x;
    const int k = kind(j, x);
    const uint64_t tie = __ballot(k == 1);
    const bool take = k == 2 || (k == 1 && ties + (uint32_t)__popcll(tie & below) < want);
    const uint64_t all = __ballot(take);
    if (take) {
      const uint32_t i = at + (uint32_t)__popcll(all & below);
      kept[i] = j;
      dst[i] = x;
    }
    at += (uint32_t)__popcll(all);
    ties += (uint32_t)__popcll(tie);
  }
  for (int32_t j = n + (int32_t)threadIdx.x; j < p.L; j += 1024) dst[j] = 0.0f;
  for (int32_t j = n + (int32_t)threadIdx.x; j < p.K; j += 1024) kept[j] = -1;
}

// The copies: a wave per 16 new tokens and head.
template <int FMT, int D>
__global__ __launch_bounds__(256) void compact_move_kernel(const CompactParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t h = (int32_t)(blockIdx.x % p.Hk), chunk = (int32_t)(blockIdx.x / p.Hk) * 4 + wave, b = blockIdx.y;
  const int32_t n = p.stay[b], i0 = 16 * chunk;
  if (i0 >= n) return;
  const int64_t unit = (int64_t)b * p.Hk + h;
  const int32_t page = __builtin_amdgcn_readfirstlane(p.bt_out[(int64_t)b * p.M + i0 / p.bs]);
  if (!page_ok(p, page)) return;  // (the ring held something that is no page)
  // Old page and place of new token i0 + t, in lane t.
  const int32_t mine = i0 + (lane & 15) < n ? p.kept[unit * p.K + i0 + (lane & 15)] : -1;
  const int32_t old = mine < 0 ? -1 : p.bt[(int64_t)b * p.M + mine / p.bs], at = mine < 0 ? 0 : mine % p.bs;
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

static int64_t compact_workspace(const memopt_compact_desc &d) {
  return ((2 * (int64_t)d.num_requests + d.num_kv_blocks) * 4 + 255) / 256 * 256;
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
  MEMOPT_REQUIRE(d.num_kv_heads <= 65535 && ((int64_t)d.max_keep / 64 + 1) * d.num_kv_heads * std::max(1, d.num_requests) < (1LL << 24),
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
  p.marks = p.holes + p.N;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(1024), 0, s, p);
  rc = check_launch("compact_cache(plan)");
  if (rc != MEMOPT_OK || p.N == 0) return rc;
  hipLaunchKernelGGL(compact_select_kernel, dim3(p.Hk, p.N), dim3(1024), 0, s, p);
  if ((rc = check_launch("compact_cache(select)")) != MEMOPT_OK || p.K == 0) return rc;
  const dim3 grid((unsigned)(((int64_t)p.K + 63) / 64 * p.Hk), p.N);
  if (d.kv_format == MEMOPT_KV_INT4) {
    if (p.D == 128) hipLaunchKernelGGL((compact_move_kernel<MEMOPT_KV_INT4, 128>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((compact_move_kernel<MEMOPT_KV_INT4, 64>), grid, dim3(256), 0, s, p);
  } else {
    if (p.D == 128) hipLaunchKernelGGL((compact_move_kernel<MEMOPT_KV_FP16, 128>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((compact_move_kernel<MEMOPT_KV_FP16, 64>), grid, dim3(256), 0, s, p);
  }
  return check_launch("compact_cache(move)");
}
