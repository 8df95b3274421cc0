// batch.hip — the index tensors of a batch's next step, built on the GPU:
// block tables, slot map, positions, query starts and context lengths from
// the requests' token counts and a ring of free pages.
//
// The host-side counterpart is PagedKVCache (memopt_runtime/kv_cache.py); the
// slot convention is the reference's (TheRadDani/memopt-transformer-runtime
// src/csrc/kv_cache.cu:244-259: slot = page * block_size + offset), and the
// ring keeps its free list's FIFO order (:163-185).
//
// Request b holds ctx tokens and asks for n more. With have = ceil(ctx / bs)
// and need = ceil((ctx + n) / bs) - have, requests are served in order while
// the running sums of need and n, over all valid requests so far, stay within
// the free pages and the rows; a request that needs no page is never refused
// for pages. Served requests take pages from the ring's head in request order
// and rows one behind the other. So the whole step is two pairs of prefix
// sums: of what is asked (which decides who is served; saturating, so that no
// sum wraps) and of what is served (which places rows and pages).
//
// Bound: latency. A step moves a few kilobytes, so what counts is one launch
// and a short chain of dependent round trips: the lengths, the tail entries,
// two block-wide scans, the ring's pages, then the slots from LDS. 8 requests:
// 3.1 us (256 threads); 512: 6.4 (1024 threads); 260 with 48000 new rows: 6.4
// and 2.2 for the rows, whose launch of their own spreads them over the GPU.
#include "packed.hpp"

namespace memopt {

struct AdvanceParams {
  const int32_t *new_tokens, *ctx;
  int32_t B;
  int32_t *tables;
  int32_t M;
  const int32_t *ring;
  int32_t C;
  const int32_t *span;
  int32_t bs;
  int32_t rows;
  int32_t *ctx_out, *span_out, *cu, *slots, *positions, *status;
};

static constexpr int32_t kMaxRequests = 4096;   // their row and page offsets are held in LDS
static constexpr int32_t kOneLaunchRows = 8192;  // above: the rows get a launch of their own

struct Sums {
  uint32_t a, b;
};
__device__ __forceinline__ Sums sat_add(Sums x, Sums y) {
  return {__builtin_elementwise_add_sat(x.a, y.a), __builtin_elementwise_add_sat(x.b, y.b)};
}

// Inclusive saturating prefix sums over the workgroup's threads; `total` is
// the sum of all. s_part: one entry per wave.
template <int NT>
__device__ __forceinline__ Sums block_scan(Sums v, Sums *s_part, Sums &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = {wave_scan(v.a), wave_scan(v.b)};
  __syncthreads();  // s_part is free
  if (lane == 63) s_part[wave] = v;
  __syncthreads();
  Sums before = {0, 0};
  total = {0, 0};
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w == wave) before = total;
    total = sat_add(total, s_part[w]);
  }
  return sat_add(before, v);
}

// The last index i in [0, n) with start[i] <= t (start ascends from 0, n >= 1).
__device__ __forceinline__ int32_t owner_of(const int32_t *start, int32_t n, int32_t t) {
  int32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (start[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Slot and position of row t (-1 behind the last row). A page whose slots pass
// 32 bits gives -1 too: the writers skip it, where a wrapped slot would be
// somebody else's.
template <class Ctx>
__device__ __forceinline__ void place_row(const AdvanceParams &p, const int32_t *s_cu, Ctx ctx, int32_t rows, int32_t t) {
  int32_t slot = -1, pos = -1;
  if (t < rows) {
    const int32_t b = owner_of(s_cu, p.B, t);
    pos = ctx(b) - (s_cu[b + 1] - t);
    const int64_t x = (int64_t)p.tables[(int64_t)b * p.M + pos / p.bs] * p.bs + pos % p.bs;
    slot = x >= 0 && x <= INT32_MAX ? (int32_t)x : -1;
  }
  p.slots[t] = slot;
  p.positions[t] = pos;
}

template <int NT>
__global__ __launch_bounds__(NT) void advance_kernel(const AdvanceParams p, const int fill) {
  // First row, first page and new context of each request.
  __shared__ int32_t s_cu[kMaxRequests + 1], s_first[kMaxRequests + 1], s_ctx[kMaxRequests];
  __shared__ Sums s_part[NT / 64];
  const int tid = threadIdx.x;
  int32_t head = p.span[0] % p.C;
  if (head < 0) head += p.C;
  const int32_t count = min(max(p.span[1], 0), p.C);
  const int64_t most = (int64_t)p.M * p.bs;

  Sums asked = {0, 0}, served = {0, 0};  // pages, rows of the requests already looked at
  for (int32_t b0 = 0; b0 < p.B; b0 += NT) {
    const int32_t b = b0 + tid;
    int32_t c = 0, n = 0, st = 0, have = 0, need = 0;
    if (b < p.B) {
      c = p.ctx[b];
      n = p.new_tokens[b];
      if (n < 0 || c < 0 || (int64_t)c + n > most) {
        st = 1;
        n = 0;
      } else {
        have = (int32_t)(((int64_t)c + p.bs - 1) / p.bs);
        if (n > 0 && c % p.bs != 0 && p.tables[(int64_t)b * p.M + have - 1] < 0) {
          st = 2;
          n = 0;
        }
      }
      if (n > 0) need = (int32_t)(((int64_t)c + n + p.bs - 1) / p.bs) - have;
    }
    Sums total;
    const Sums ask = sat_add(asked, block_scan<NT>({(uint32_t)need, (uint32_t)n}, s_part, total));
    asked = sat_add(asked, total);
    if (need > 0 && ask.a > (uint32_t)count) st = 3;
    else if (n > 0 && ask.b > (uint32_t)p.rows) st = 4;
    if (st != 0) n = need = 0;
    Sums got = block_scan<NT>({(uint32_t)need, (uint32_t)n}, s_part, total);
    got.a += served.a;
    got.b += served.b;
    served = {served.a + total.a, served.b + total.b};
    if (b < p.B) {
      s_cu[b] = (int32_t)got.b - n;
      s_first[b] = (int32_t)got.a - need;
      p.cu[b + 1] = (int32_t)got.b;
      s_ctx[b] = p.ctx_out[b] = c + n;
      p.status[b] = st;
    }
  }
  const int32_t rows = (int32_t)served.b, pages = (int32_t)served.a;
  if (tid == 0) {
    s_cu[p.B] = rows;
    s_first[p.B] = pages;
    p.cu[0] = 0;
    p.span_out[0] = (int32_t)(((int64_t)head + pages) % p.C);
    p.span_out[1] = count - pages;
  }
  __syncthreads();
  // Pages: the j-th of the step belongs to the request whose range holds j,
  // behind the pages its old context has.
  for (int32_t j = tid; j < pages; j += NT) {
    const int32_t b = owner_of(s_first, p.B, j);
    const int32_t c = s_ctx[b] - (s_cu[b + 1] - s_cu[b]);
    const int32_t have = (int32_t)(((int64_t)c + p.bs - 1) / p.bs);
    p.tables[(int64_t)b * p.M + have + j - s_first[b]] = p.ring[(int32_t)(((int64_t)head + j) % p.C)];
  }
  if (!fill) return;
  __syncthreads();
  for (int32_t t = tid; t < p.rows; t += NT) place_row(p, s_cu, [&](int32_t b) { return s_ctx[b]; }, rows, t);
}

// Slots and positions from the step's query starts, context lengths and tables.
__global__ __launch_bounds__(256) void advance_rows_kernel(const AdvanceParams p) {
  __shared__ int32_t s_cu[kMaxRequests + 1];
  for (int32_t i = threadIdx.x; i <= p.B; i += 256) s_cu[i] = p.cu[i];
  __syncthreads();
  const int32_t rows = s_cu[p.B];
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < p.rows; t += (int64_t)gridDim.x * 256)
    place_row(p, s_cu, [&](int32_t b) { return p.ctx_out[b]; }, rows, (int32_t)t);
}

}  // namespace memopt

using namespace memopt;

extern "C" int memopt_advance_batch(const memopt_advance_desc *desc, void *stream) {
  MEMOPT_REQUIRE(desc, MEMOPT_ERR_INVALID, "advance_batch: null descriptor");
  const memopt_advance_desc &d = *desc;
  MEMOPT_REQUIRE(d.num_requests > 0 && d.max_blocks_per_seq > 0 && d.num_free_pages > 0 && d.block_size > 0 &&
                     d.num_rows >= 0,
                 MEMOPT_ERR_INVALID, "advance_batch: sizes must be positive");
  MEMOPT_REQUIRE(d.num_requests <= kMaxRequests, MEMOPT_ERR_UNSUPPORTED,
                 "advance_batch: more than " + std::to_string(kMaxRequests) + " requests");
  MEMOPT_REQUIRE((int64_t)d.max_blocks_per_seq * d.block_size < (1LL << 31), MEMOPT_ERR_UNSUPPORTED,
                 "advance_batch: a block table of 2^31 tokens and more");
  MEMOPT_REQUIRE(d.new_tokens && d.context_lens && d.block_tables && d.free_pages && d.free_span &&
                     d.context_lens_out && d.free_span_out && d.query_starts && d.status &&
                     (d.num_rows == 0 || (d.slots && d.positions)),
                 MEMOPT_ERR_INVALID, "advance_batch: null pointer");
  const int32_t num_requests = d.num_requests, num_rows = d.num_rows;
  const AdvanceParams p = {d.new_tokens, d.context_lens, num_requests, d.block_tables, d.max_blocks_per_seq,
                           d.free_pages, d.num_free_pages, d.free_span, d.block_size, num_rows, d.context_lens_out,
                           d.free_span_out, d.query_starts, d.slots, d.positions, d.status};
  hipStream_t s = (hipStream_t)stream;
  const int fill = num_rows <= kOneLaunchRows;
  if (num_requests <= 256 && num_rows <= 1024)
    hipLaunchKernelGGL(advance_kernel<256>, dim3(1), dim3(256), 0, s, p, fill);
  else
    hipLaunchKernelGGL(advance_kernel<1024>, dim3(1), dim3(1024), 0, s, p, fill);
  int rc = check_launch("advance_batch");
  if (rc != MEMOPT_OK || fill) return rc;
  const int64_t wgs = ((int64_t)num_rows + 255) / 256;
  hipLaunchKernelGGL(advance_rows_kernel, dim3((unsigned)(wgs < 1024 ? wgs : 1024)), dim3(256), 0, s, p);
  return check_launch("advance_batch(rows)");
}
