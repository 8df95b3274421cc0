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
#include <algorithm>
#include <cmath>

#include "attention.hpp"
#include "lds_dma.hpp"

namespace memopt {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4p_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2p_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

struct PromptParams {
  const uint16_t *q, *k, *v;  // 16-bit elements; strides in elements
  uint16_t *out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
  const int32_t *cu;
  int32_t T, B, Hq, Hk, W, sinks;
  float qk_scale_log2;
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
  static __device__ __forceinline__ float add2(uint32_t w, float s) {
    return __builtin_amdgcn_fdot2(as_half2(w), half2_t{(half_t)1.0f, (half_t)1.0f}, s, false);
  }
  static __device__ __forceinline__ float value(uint16_t x) { return (float)__builtin_bit_cast(half_t, x); }
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
  static __device__ __forceinline__ float add2(uint32_t w, float s) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(x2, w), __builtin_bit_cast(x2, 0x3F803F80u), s, false);
  }
  static __device__ __forceinline__ float value(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
  static constexpr uint32_t kExponent = 0x7F80u;
};

__device__ __forceinline__ float both_halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Sum of a wave's lanes, in every lane.
__device__ __forceinline__ int32_t wave_sum(int32_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return __builtin_amdgcn_readfirstlane(v);
}

// The query tile (R rows of one sequence) that comes rank-th when the tiles of
// all sequences are ordered by their place in their sequence, last places
// first: under the causal mask those see the most keys, and a grid that ends
// with its longest workgroups leaves the GPU idle behind them. Each lane holds
// the tile counts of up to four sequences; the tiles at place >= x are
// counted with one sum over the wave, x found by bisection. More than 256
// sequences are taken in order instead. Returns false past the last tile.
struct Tile {
  int32_t b, t;
};
template <int R>
__device__ __forceinline__ bool find_tile(const int32_t *cu, int32_t B, int32_t T, int32_t rank, Tile &out) {
  const int lane = threadIdx.x & 63;
  auto tiles_of = [&](int32_t b) {
    if (b >= B) return 0;
    const int32_t lo = min(max(cu[b], 0), T), hi = min(max(cu[b + 1], lo), T);
    return (hi - lo + R - 1) / R;
  };
  if (B <= 256) {
    int32_t n[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) n[k] = 64 * k < B ? tiles_of(64 * k + lane) : 0;
    auto at_or_past = [&](int32_t x) {
      int32_t s = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) s += max(0, n[k] - x);
      return wave_sum(s);
    };
    if (rank >= at_or_past(0)) return false;
    int32_t lo = 0, hi = (T + R - 1) / R;  // at_or_past(lo) > rank >= at_or_past(hi)
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (at_or_past(mid) > rank) lo = mid;
      else hi = mid;
    }
    int32_t r = rank - at_or_past(hi);  // among the sequences with more than lo tiles
    out.t = lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t m = __ballot(n[k] > lo);
      const int32_t c = __popcll(m);
      if (r >= 0 && r < c) {
        const bool mine = n[k] > lo && (int32_t)__popcll(m & ((1ull << lane) - 1)) == r;
        out.b = 64 * k + (int32_t)__builtin_ctzll(__ballot(mine));
      }
      r = r < c ? -1 : r - c;
      if (r < 0) break;
    }
    return true;
  }
  int32_t before = 0;
  for (int32_t b0 = 0; b0 < B; b0 += 64) {
    const int32_t n = tiles_of(b0 + lane);
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
      return true;
    }
    before += total;
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

// Zeroes the elements of four operands that are inf or NaN; whether any lane had one.
template <class E>
__device__ __forceinline__ bool drop_odd(u32x4p_t (&v)[4]) {
  constexpr uint32_t m = E::kExponent * 0x10001u, step = 0x80008000u - m;  // a full exponent carries into bit 15
  uint32_t any = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= (v[c][i] & m) + step;
  if (!__any((any & 0x80008000u) != 0)) return false;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t f = (v[c][i] & m) + step;
      v[c][i] &= ((f & 0x8000u) ? 0u : 0xFFFFu) | ((f & 0x80000000u) ? 0u : 0xFFFF0000u);
    }
  return true;
}

template <class E, int D, int NW>
__global__ __launch_bounds__(NW * 64, 2) void prompt_kernel(const PromptParams p) {
  constexpr int TK = 64, R = 32 * NW;             // keys per tile, query rows per workgroup
  constexpr int RB = 2 * D, CPR = RB / 16;         // bytes and 16-byte pieces of an LDS row
  constexpr int NCH = D / 16, NDB = D / 32;
  constexpr int RPC = 1024 / RB, NC = TK / RPC / NW;  // rows per copy; copies per wave of K (and of V)
  __shared__ __attribute__((aligned(16))) uint8_t lds_k[2][TK * RB], lds_v[2][TK * RB];

  const int lane = threadIdx.x & 63, n = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t slot = (int32_t)(blockIdx.x % p.Hq);
  Tile tile;
  if (!find_tile<R>(p.cu, p.B, p.T, (int32_t)(blockIdx.x / p.Hq), tile)) return;
  const int32_t b = __builtin_amdgcn_readfirstlane(tile.b);
  const int32_t G = p.Hq / p.Hk;
  // Workgroup i runs on XCD i % 8: the query heads of one key head share an
  // XCD and its L2 where the heads deal out evenly.
  int32_t kvh = slot / G, h = slot;
  if (p.Hk % 8 == 0) {
    kvh = (slot & 7) + 8 * ((slot >> 3) / G);
    h = kvh * G + (slot >> 3) % G;
  }
  const int32_t s0 = min(max(p.cu[b], 0), p.T), len = min(max(p.cu[b + 1], s0), p.T) - s0;
  const int32_t q0 = R * __builtin_amdgcn_readfirstlane(tile.t), qw0 = q0 + 32 * wave, qi = qw0 + n;
  const bool q_ok = qi < len;

  u32x4p_t qf[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) qf[c] = (u32x4p_t){};
  if (q_ok) {
    const uint16_t *src = p.q + (int64_t)(s0 + qi) * p.q_ts + h * p.q_hs + 8 * hl;
#pragma unroll
    for (int c = 0; c < NCH; ++c) qf[c] = *reinterpret_cast<const u32x4p_t *>(src + 16 * c);
  }

  // Tiles of the workgroup: sinks, then the window of its rows.
  const int32_t q_last = min(q0 + R, len) - 1, hi = q_last + 1;
  const int32_t sink_tiles = (min(p.sinks, hi) + TK - 1) / TK;
  const int32_t t_first = max(max(0, q0 - p.W + 1) / TK, sink_tiles), t_last = (hi + TK - 1) / TK;
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
  const uint8_t *k_base = reinterpret_cast<const uint8_t *>(p.k + (int64_t)s0 * p.k_ts + kvh * p.k_hs);
  const uint8_t *v_base = reinterpret_cast<const uint8_t *>(p.v + (int64_t)s0 * p.v_ts + kvh * p.v_hs);
  const uint32_t wave_lds = (uint32_t)wave * NC * 1024;
  const uint32_t mk[2] = {lds_u32(lds_k[0]) + wave_lds, lds_u32(lds_k[1]) + wave_lds};
  const uint32_t mv[2] = {lds_u32(lds_v[0]) + wave_lds, lds_u32(lds_v[1]) + wave_lds};
  // A tile's rows through a descriptor of their own: 64-bit bases, and rows
  // past the sequence lie outside its range and read as zeros.
  auto rows_at = [&](const uint8_t *base, uint32_t rb, int32_t key0) __attribute__((always_inline)) {
    const int32_t rows = min(TK, len - key0);
    return __builtin_amdgcn_make_buffer_rsrc((void *)(base + (int64_t)key0 * rb), (short)0,
                                             (int)((rows - 1) * rb + RB), 0x00020000);
  };
  auto load_tile = [&](int32_t it, int buf) __attribute__((always_inline)) {
    const int32_t key0 = tile_base(it);
    lds_dma_range<0, NC>(rows_at(k_base, k_rb, key0), mk[buf], k_off, 0);
    lds_dma_range<0, NC>(rows_at(v_base, v_rb, key0), mv[buf], v_off, 0);
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
  float ncm = 0.0f, thr = -INFINITY, lsum = 0.0f;
  const int32_t w_last = min(qw0 + 31, len - 1);  // the wave's last row

  if (n_tiles > 0) load_tile(0, 0);
  for (int32_t it = 0; it < n_tiles; ++it) {
    const int P = it & 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // tile it is in LDS; every wave has read tile it - 1
    if (it + 1 < n_tiles) load_tile(it + 1, P ^ 1);
    const int32_t tb = tile_base(it);
    if (qw0 >= len || tb > w_last || (tb + TK <= qw0 - p.W + 1 && tb >= p.sinks)) continue;  // nothing to see
    const bool full = tb + TK - 1 <= qw0 && (tb >= qw0 + 31 - p.W + 1 || tb + TK <= p.sinks);

    f32x16_t s[2];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const u32x4p_t a = *reinterpret_cast<const u32x4p_t *>(&lds_k[P][32 * blk * RB + ka[c]]);
        s[blk] = E::mfma(a, qf[c], c == 0 ? (f32x16_t){} : s[blk]);
      }
    // Register r of block blk holds key tb + 32 blk + 8 (r / 4) + 4 hl + r % 4.
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[blk][r] = fmaf(s[blk][r], p.qk_scale_log2, ncm);
    const int32_t key0 = tb + 4 * hl;
    if (!full) {
      const int32_t last = q_ok ? qi - key0 : -1, first = qi - p.W + 1 - key0, sink = p.sinks - key0;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int32_t c = 32 * blk + 8 * (r >> 2) + (r & 3);
          s[blk][r] = (c <= last) & ((c >= first) | (c < sink)) ? s[blk][r] : -INFINITY;
        }
    }
    float t = s[0][0];
#pragma unroll
    for (int r = 1; r < 16; ++r) t = fmaxf(t, s[0][r]);
#pragma unroll
    for (int r = 0; r < 16; ++r) t = fmaxf(t, s[1][r]);
    t = both_halves_max(t);
    if (__any(t > thr)) {
      const bool start = thr == -INFINITY, found = t > -INFINITY;
      const float shift = start ? (found ? t - kTop : 0.0f) : fmaxf(t - kTop, 0.0f);
      const float alpha = start ? (found ? 0.0f : 1.0f) : (shift > 0.0f ? fast_exp2(-shift) : 1.0f);
      lsum *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[db] *= alpha;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) s[blk] -= shift;
      ncm -= shift;
      thr = (start && !found) ? thr : kTop + 8.0f;
    }
    u32x4p_t pf[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * (c & 1) + 2 * i;
        s[c >> 1][r] = fast_exp2(s[c >> 1][r]);
        s[c >> 1][r + 1] = fast_exp2(s[c >> 1][r + 1]);
        pf[c][i] = E::pack(s[c >> 1][r], s[c >> 1][r + 1]);
        lsum = E::add2(pf[c][i], lsum);
      }
    // Probabilities of 16 keys (two register quads) are the second product's
    // operand as they are; V^T comes transposed from LDS in the same order.
    bool odd = false;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      u32x4p_t vf[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const u32x2p_t lo = v_read(lds_v[P], va[db] + 16 * c * RB), hi8 = v_read(lds_v[P], va[db] + (16 * c + 8) * RB);
        vf[c] = u32x4p_t{lo[0], lo[1], hi8[0], hi8[1]};
      }
      if (!full) odd |= drop_odd<E>(vf);
#pragma unroll
      for (int c = 0; c < 4; ++c) o[db] = E::mfma(vf[c], pf[c], o[db]);
    }
    if (!full && odd) {  // wave-uniform
      // Elements of V that are inf or NaN were left out above, as they must not
      // meet the weight 0 of a row that does not see them; each is added here
      // to the rows that do.
      const int32_t last = q_ok ? qi - tb : -1, first = qi - p.W + 1 - tb, sink = p.sinks - tb;
#pragma unroll 1
      for (int key = 0; key < TK; ++key) {
        const int reg = 16 * (key >> 5) + 4 * ((key >> 3) & 3) + (key & 3);
        float pk = 0.0f;
#pragma unroll
        for (int x = 0; x < 32; ++x) pk = x == reg ? s[x >> 4][x & 15] : pk;
        pk = __shfl(pk, n + 32 * ((key >> 2) & 1), 64);
        const bool see = (key <= last) & ((key >= first) | (key < sink));
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint8_t *src = &lds_v[P][key * RB + 16 * ((4 * db + g) ^ v_swz(key)) + 8 * hl];
            const u32x2p_t w = *reinterpret_cast<const u32x2p_t *>(src);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint16_t bits = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
              if (see && (bits & E::kExponent) == E::kExponent)
                o[db][4 * g + e] = fmaf(pk, E::value(bits), o[db][4 * g + e]);
            }
          }
      }
    }
  }

  const float l = xor32_sum(lsum);
  if (!q_ok) return;
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  uint16_t *dst = p.out + (int64_t)(s0 + qi) * p.o_ts + h * p.o_hs + 4 * hl;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<u32x2p_t *>(dst + 32 * db + 8 * g) =
          u32x2p_t{E::pack(o[db][4 * g] * inv, o[db][4 * g + 1] * inv),
                   E::pack(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv)};
}

template <class E, int D>
static void launch_prompt(const PromptParams &p, hipStream_t stream) {
  const int64_t tiles = ((int64_t)p.T + 127LL * std::min(p.B, p.T)) / 128;
  hipLaunchKernelGGL((prompt_kernel<E, D, 4>), dim3((unsigned)(tiles * p.Hq)), dim3(256), 0, stream, p);
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
  PromptParams p;
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
  p.cu = d.query_starts;
  p.T = d.tokens;
  p.B = d.batch;
  p.Hq = d.num_heads;
  p.Hk = d.num_kv_heads;
  p.W = d.window_size <= 0 ? 1 << 30 : std::min(d.window_size, 1 << 30);  // (position - W stays in 32 bits)
  p.sinks = std::max(0, d.num_sink_tokens);
  p.qk_scale_log2 = 1.4426950408889634f / sqrtf((float)d.head_dim);
  MEMOPT_REQUIRE(((int64_t)d.tokens / 32 + d.batch) * d.num_heads < (1LL << 31), MEMOPT_ERR_UNSUPPORTED,
                 "prompt_attention: too many query tiles");
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
