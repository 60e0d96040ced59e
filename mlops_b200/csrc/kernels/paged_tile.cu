// Attention over the paged cache for many queries per request (mlops_paged_attend): chunks of prompts and whole prompts, on tcgen05 tensor cores with
// TMEM accumulators.
//
// A row of work is (request, KV head, 256 rows); row c of a request and KV head is query c / group with query head c % group. Its units are the tiles of
// 128 tokens that its last row sees. All units form one list, of which every CTA has an equal contiguous run; a row of work that is cut is joined from
// partial rows (o, m', l) by the CTA that comes last, in the order of the tokens.
//
// Per tile of tokens and half X of the rows (128 each), with FP32 accumulators in tensor memory:
//   S_X[128 x 128] = Q_X K^T,   O_X[128 x 128] += P_X V
// K and V are code * scale, exact in FP16; Q is FP16 after a power of two per row (paged_attend.cuh); P = 2^(s - m') in FP16 takes S_X's place in tensor
// memory. m' moves only where a score would pass 2^15, then O and l are rescaled; l sums the unrounded P. Rows of at most 128 use both halves too: the
// even tiles of tokens go to X = 0, the odd ones to X = 1, with the same queries, and the halves are joined at the end.
//
// Warps 0-3 and 4-7 (a thread per row): softmax of X = 0 and 1. Warps 8-11: operands, from packed pages to two stages each of K and V in shared
// memory, token rows of 128 bytes (64 channels) with 16-byte chunk c of row r at c ^ (r % 8): for S that is K-major, for O V's MN-major. Warps 12, 13: one thread
// each issues the products of its X. Every wait is bounded: where one gives up, the rows become NaN.
#include "fbla_launch.h"
#include "fbla_tc.cuh"
#include "paged_attend.cuh"

namespace paged {
namespace {

namespace tc = fbla::tc;

constexpr int ROWS = 128, TOKENS = 128;     // of a product
constexpr int SLAB = 128 * 128, TILE = 2 * SLAB;  // bytes of a slab (128 rows of 64 channels) and of an operand
constexpr int STAGES = 2, PRODUCER0 = 8, ISSUER0 = 12, THREADS = 16 * 32;  // (four warps share a register count: 12, 13 issue, 14, 15 idle)
constexpr float TOP = 15.f, REST = 9.f;
constexpr uint32_t WAIT_LIMIT = 1u << 18;
constexpr uint32_t IDESC_S = tc::IDESC_F16, IDESC_O = tc::IDESC_F16 | (1u << 16);  // V: MN-major

struct __align__(1024) Smem {
  uint8_t q[2][TILE];  // at a row of work's end: half 1's sums, to be joined with half 0's
  uint8_t k[STAGES][TILE], v[STAGES][TILE];
  uint64_t q_ready[2], k_full[STAGES], v_full[STAGES], k_empty[STAGES], v_empty[STAGES], s_ready[2], p_ready[2], o_done[2];
  uint8_t there[4][8];  // [tile of tokens % 4][block]: 1 where the table names a page
  float2 ml[ROWS];      // half 1's (m', l)
  long long warp_sum[THREADS / 32];
  uint32_t tmem;
  int abort, last;
  long long before[];   // [batch + 1]: the requests' first units
};

__device__ __forceinline__ bool wait(Smem &sm, uint64_t *bar, uint32_t parity) {
  if (tc::try_wait_hint(bar, parity)) return true;
  for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
    if (*reinterpret_cast<volatile int *>(&sm.abort)) return false;
    if (tc::try_wait_hint(bar, parity)) return true;
  }
  *reinterpret_cast<volatile int *>(&sm.abort) = 1;
  return false;
}

// V as the B operand of a product: 64 channels are contiguous, slabs of them SLAB apart, groups of eight tokens 1024 bytes apart
__device__ __forceinline__ uint64_t v_desc(const void *tile, uint32_t byte_offset) {
  return tc::smem_desc_at(tile, byte_offset) | ((uint64_t)(SLAB >> 4) << 16);
}

__device__ __forceinline__ int rows_of(const Call &k, const Request &r) { return r.n * k.group; }
// tiles of tokens that rows up to 256 (pair + 1) of a request see
__device__ __forceinline__ int tiles_of(const Call &k, const Request &r, int pair) {
  const int last = min(2 * ROWS * (pair + 1), rows_of(k, r)) - 1, seen = min(r.length - r.n + last / k.group + 1, r.tokens);
  return max((seen + TOKENS - 1) / TOKENS, 1);  // (rows that see nothing have a tile all the same: their zeros are written like the others' sums)
}
__device__ __forceinline__ bool taken(const Call &k, const Request &r) { return r.tokens > 0 && r.n * k.group > k.wide; }

// a row of work and its part in this CTA's run: tiles of tokens n0 .. n1 - 1 of `tiles`
struct Row {
  Request r;
  int b, head, pair, tiles, n0, n1;
  long long unit0;
  __device__ __forceinline__ int rows(const Call &k) const { return min(rows_of(k, r) - 2 * ROWS * pair, 2 * ROWS); }
  __device__ __forceinline__ bool halves(const Call &k) const { return rows(k) <= ROWS; }  // both X have the same rows
};
// the first row of work of the run [lo, hi)
__device__ __forceinline__ Row first_row(const Call &k, const long long *before, long long lo, long long hi) {
  Row w;
  int a = 0;
  for (int e = k.a.batch; e - a > 1;) {
    const int mid = (a + e) >> 1;
    if (before[mid] <= lo) a = mid; else e = mid;
  }
  w.b = a;
  w.r = request(k, a);
  const long long per_head = (before[a + 1] - before[a]) / k.c.kv_heads, x = lo - before[a];
  w.head = (int)(x / per_head);
  long long rest = x - w.head * per_head;
  w.pair = 0;
  while (rest >= (w.tiles = tiles_of(k, w.r, w.pair))) rest -= w.tiles, ++w.pair;
  w.n0 = (int)rest;
  w.unit0 = lo - rest;
  w.n1 = (int)min((long long)w.tiles, hi - w.unit0);
  return w;
}
// the row of work behind w in the run; false where there is none
__device__ __forceinline__ bool next_row(const Call &k, const long long *before, long long hi, Row &w) {
  w.unit0 += w.tiles;
  if (w.unit0 >= hi) return false;
  if (2 * ROWS * ++w.pair >= rows_of(k, w.r)) {
    w.pair = 0;
    if (++w.head == k.c.kv_heads) {
      w.head = 0;
      do ++w.b; while (before[w.b + 1] <= w.unit0);
      w.r = request(k, w.b);
    }
  }
  w.tiles = tiles_of(k, w.r, w.pair);
  w.n0 = 0;
  w.n1 = (int)min((long long)w.tiles, hi - w.unit0);
  return true;
}
// whether half X has a part in tile n of w: w's second half in row order, or every second tile where the halves share the rows; a first half
// whose rows see less than the second one's leaves the last tile out
__device__ __forceinline__ int tiles_of_half(const Call &k, const Row &w, int x) {
  const int last = min(2 * ROWS * w.pair + ROWS * (x + 1), rows_of(k, w.r)) - 1, seen = min(w.r.length - w.r.n + last / k.group + 1, w.r.tokens);
  return max((seen + TOKENS - 1) / TOKENS, 1);
}
struct Part {
  bool shared;
  int limit;  // tiles
  __device__ __forceinline__ bool has(int n, int x) const { return shared ? (n & 1) == x : n < limit; }
};

// ---- operands -------------------------------------------------------------------------------------------------------------------
struct Raw {  // a lane's part of a tensor's two blocks of a tile: [block][half of its tokens]
  uint4 codes[4];
  uint32_t scales[4];
};
__device__ __forceinline__ void load_raw(Raw &x, const uint8_t *const (&block)[2], int codes, int scales, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int token = 8 * (i & 1) + (lane & 7), quarter = lane >> 3;
    x.codes[i] = make_uint4(0, 0, 0, 0);
    x.scales[i] = 0;
    if (block[i >> 1]) {
      x.codes[i] = __ldg(reinterpret_cast<const uint4 *>(block[i >> 1] + codes + token * CODE_BYTES + 16 * quarter));
      x.scales[i] = __ldg(reinterpret_cast<const uint16_t *>(block[i >> 1] + scales + token * SCALE_BYTES + 2 * quarter));
    }
  }
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ void store_operand(uint8_t *tile, const Raw &x, int row0, int lane) {
  const int quarter = lane >> 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 8 * i + (lane & 7);
    uint8_t *const line = tile + (quarter >> 1) * SLAB + row * 128;
    const uint32_t s = scales_to_half2(x.scales[i]), w[4] = {x.codes[i].x, x.codes[i].y, x.codes[i].z, x.codes[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t h[4];
      codes_to_half2(w[j], h);
      const uint32_t f = __byte_perm(s, 0, j < 2 ? 0x1010 : 0x3232);
      *reinterpret_cast<uint4 *>(line + (((4 * (quarter & 1) + j) ^ (row & 7)) << 4)) = make_uint4(times(h[0], f), times(h[1], f), times(h[2], f), times(h[3], f));
    }
  }
}

__device__ __forceinline__ void produce(const Call &k, Smem &sm, long long lo, long long hi, int warp, int lane) {
  const int per_page = k.c.page_size / BT;
  uint32_t at = 0;  // tiles of tokens so far
  Row w = first_row(k, sm.before, lo, hi);
  bool more = true, ok = true;
  int n = w.n0;
  // this warp's two blocks of tile n of w, null where the table names no page
  auto find = [&](const Row &w, int n, const uint8_t *(&block)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int number = 8 * n + 2 * warp + j, column = number / per_page;
      block[j] = nullptr;
      if (number * BT < w.r.tokens) {
        const int page = __ldg(k.a.table + (size_t)w.b * k.a.table_stride + column);
        if ((unsigned)page < (unsigned)k.c.pages)
          block[j] = k.c.units + (size_t)page * k.c.page_stride + (size_t)w.head * k.c.head_stride + (size_t)(number - column * per_page) * BLOCK_BYTES;
      }
    }
  };
  const uint8_t *block[2];
  Raw rk, rv;
  find(w, n, block);
  load_raw(rk, block, 0, K_SCALES, lane);
  load_raw(rv, block, V_CODES, V_SCALES, lane);
  while (more && ok) {
    const int stage = at % STAGES, tokens = w.r.tokens, number = n;
    const uint32_t parity = (at / STAGES & 1) ^ 1;
    const bool here[2] = {block[0] != nullptr, block[1] != nullptr};
    // the tile behind this one
    if (++n == w.n1) {
      more = next_row(k, sm.before, hi, w);
      n = w.n0;
    }
    if (more) find(w, n, block);
    if (at >= STAGES) ok = wait(sm, &sm.k_empty[stage], parity);
    if (lane < 2) sm.there[at & 3][2 * warp + lane] = here[lane];
    store_operand(sm.k[stage], rk, 32 * warp, lane);
    fbla::fence_async_smem();
    tc::mbar_arrive(&sm.k_full[stage]);
    if (more) load_raw(rk, block, 0, K_SCALES, lane);
    if (TOKENS * (number + 1) > tokens) {  // (what is stored behind the last token may be anything, NaN too)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (TOKENS * number + 32 * warp + 8 * i + (lane & 7) >= tokens) rv.scales[i] = 0;
    }
    if (at >= STAGES && ok) ok = wait(sm, &sm.v_empty[stage], parity);
    store_operand(sm.v[stage], rv, 32 * warp, lane);
    fbla::fence_async_smem();
    tc::mbar_arrive(&sm.v_full[stage]);
    if (more) load_raw(rv, block, V_CODES, V_SCALES, lane);
    ++at;
  }
}

// ---- products -------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void issue(const Call &k, Smem &sm, long long lo, long long hi, int x) {  // by one thread
  const uint32_t s_at = sm.tmem + 128 * x, o_at = sm.tmem + 256 + 128 * x;
  uint32_t at = 0, mine = 0, items = 0;
  bool ok = true;
  Row w = first_row(k, sm.before, lo, hi);
  do {
    const Part part{w.halves(k), tiles_of_half(k, w, x)};
    ok = ok && wait(sm, &sm.q_ready[x], items++ & 1);
    bool first = true;
    for (int n = w.n0; n < w.n1 && ok; ++n, ++at) {
      const int stage = at % STAGES;
      const uint32_t parity = at / STAGES & 1;
      ok = wait(sm, &sm.k_full[stage], parity);
      if (!part.has(n, x)) {
        if (mine) ok = ok && wait(sm, &sm.o_done[x], (mine - 1) & 1);  // (not ahead of its own softmax, which reads `there`)
        tc::mbar_arrive(&sm.k_empty[stage]);
        ok = ok && wait(sm, &sm.v_full[stage], parity);
        tc::mbar_arrive(&sm.v_empty[stage]);
        continue;
      }
      if (mine) ok = ok && wait(sm, &sm.o_done[x], (mine - 1) & 1);  // (P is in S's place)
      if (!ok) break;
      tc::tc_fence_after();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t offset = (i >> 2) * SLAB + (i & 3) * 32;
        tc::mma_f16(s_at, tc::smem_desc_at(sm.q[x], offset), tc::smem_desc_at(sm.k[stage], offset), IDESC_S, i > 0);
      }
      tc::mma_commit(&sm.s_ready[x]);
      tc::mma_commit(&sm.k_empty[stage]);
      ok = wait(sm, &sm.p_ready[x], mine & 1) && wait(sm, &sm.v_full[stage], parity);
      if (!ok) break;
      tc::tc_fence_after();
#pragma unroll
      for (int i = 0; i < 8; ++i) tc::mma_f16_ts(o_at, s_at + 8 * i, v_desc(sm.v[stage], i * 2048), IDESC_O, !first || i > 0);
      tc::mma_commit(&sm.o_done[x]);
      tc::mma_commit(&sm.v_empty[stage]);
      first = false;
      ++mine;
    }
  } while (next_row(k, sm.before, hi, w));
}

// ---- softmax --------------------------------------------------------------------------------------------------------------------
// Q's row c of the row of work, times a power of two that puts its largest element into [2^8, 2^9); returns the factor that undoes it
template <int TYPE> __device__ __forceinline__ float load_q(const Call &k, const Row &w, int c, bool live, uint8_t *tile, int line) {
  uint4 raw[16] = {};
  if (live) {
    const uint16_t *const src = static_cast<const uint16_t *>(k.a.q) + (int64_t)(w.r.start + c / k.group) * k.a.q_token_stride +
                                (int64_t)(w.head * k.group + c % k.group) * k.a.q_head_stride;
#pragma unroll
    for (int e = 0; e < 16; ++e) raw[e] = __ldg(reinterpret_cast<const uint4 *>(src) + e);
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint32_t word[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = to_floats<TYPE>(word[i]);
      top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
    }
  }
  float down;
  const float up = q_factor(top, down);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint32_t word[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = to_floats<TYPE>(word[i]);
      h[i] = from_floats<MLOPS_PAGED_FP16>(f.x * up, f.y * up);
    }
    *reinterpret_cast<uint4 *>(tile + (e >> 3) * SLAB + line * 128 + (((e & 7) ^ (line & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
  }
  return down;
}

// P of 128 scores in the thread's lane at `s`: 64 words of FP16 pairs; returns the largest exponent, adds the sum to l. MASK: scores of tokens above
// `limit` (in the tile) and of blocks that are not `there` count as -infinity
template <bool MASK> __device__ __forceinline__ float exponentials(uint32_t s, float mult, float m, int limit, const uint8_t *there, uint32_t (&p)[64], float &l) {
  float high = NOTHING;
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t r[32];
    tc::tmem_ld32(s + 32 * c, r);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 e = __ffma2_rn(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), make_float2(mult, mult), make_float2(-m, -m));
      if (MASK) {
        const int token = 32 * c + 2 * i;
        const bool page = there[token >> 4];
        if (token > limit || !page) e.x = -FBLA_INF;
        if (token + 1 > limit || !page) e.y = -FBLA_INF;
      }
      high = fbla::max3(high, e.x, e.y);
      const float2 f = make_float2(ex2(e.x), ex2(e.y));
      sum = __fadd2_rn(sum, f);
      p[16 * c + i] = from_floats<MLOPS_PAGED_FP16>(f.x, f.y);
    }
  }
  l += sum.x + sum.y;
  return high;
}
// the largest of the thread's 128 scores times mult
template <bool MASK> __device__ __forceinline__ float largest(uint32_t s, float mult, int limit, const uint8_t *there) {
  float high = NOTHING;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t r[32];
    tc::tmem_ld32(s + 32 * c, r);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (!MASK || (32 * c + i <= limit && there[(32 * c + i) >> 4])) high = fmaxf(high, __uint_as_float(r[i]) * mult);
  }
  return high;
}

template <int TYPE> __device__ __forceinline__ void soften(const Call &k, Smem &sm, long long lo, long long hi, int x, int warp, int lane) {
  const int line = 32 * (warp & 3) + lane;
  const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, s_at = sm.tmem + 128 * x + lanes, o_at = sm.tmem + 256 + 128 * x + lanes;
  uint32_t mine = 0, at = 0;
  bool ok = true;
  Row w = first_row(k, sm.before, lo, hi);
  do {
    const int rows = w.rows(k);
    const bool shared = rows <= ROWS;
    const Part part{shared, tiles_of_half(k, w, x)};
    const int c = line + (shared ? 0 : ROWS * x);           // of the row of work
    const bool live = c < rows, warp_live = c - lane < rows;
    const int col = 2 * ROWS * w.pair + c, limit = live ? w.r.length - w.r.n + col / k.group : -1;
    const int low = w.r.length - w.r.n + (col - lane) / k.group;  // of the warp's rows, the smallest
    const float mult = k.sl * __ldg(k.c.k_scale + w.head) * load_q<TYPE>(k, w, col, live, sm.q[x], line);
    fbla::fence_async_smem();
    tc::mbar_arrive(&sm.q_ready[x]);
    float m = NOTHING, l = 0.f;
    bool first = true;
    for (int n = w.n0; n < w.n1; ++n, ++at) {
      if (!part.has(n, x)) continue;
      ok = __all_sync(FULL, ok && wait(sm, &sm.s_ready[x], mine & 1));
      tc::tc_fence_after();
      if (warp_live && ok) {
        const uint8_t *const there = sm.there[at & 3];
        const uint2 all = *reinterpret_cast<const uint2 *>(there);
        const bool mask = TOKENS * n + TOKENS - 1 > low || (all.x & all.y) != 0x01010101u;
        const int in_tile = min(limit - TOKENS * n, TOKENS);
        uint32_t p[64];
        const float l_before = l;
        float high = mask ? exponentials<true>(s_at, mult, m, in_tile, there, p, l) : exponentials<false>(s_at, mult, m, 0, there, p, l);
        if (__any_sync(FULL, high > TOP)) {
          // m' moves for the rows that need it
          const float top = mask ? largest<true>(s_at, mult, in_tile, there) : largest<false>(s_at, mult, 0, there);
          float keep = 1.f;
          if (top - m > TOP) {
            keep = ex2(m - (top - REST));
            m = top - REST;
          }
          l = l_before * keep;
          if (!first) {
            ok = __all_sync(FULL, wait(sm, &sm.o_done[x], (mine - 1) & 1));
            tc::tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
              uint32_t r[32];
              tc::tmem_ld32(o_at + 32 * i, r);
#pragma unroll
              for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * keep);
              tc::tmem_st32(o_at + 32 * i, r);
            }
          }
          mask ? exponentials<true>(s_at, mult, m, in_tile, there, p, l) : exponentials<false>(s_at, mult, m, 0, there, p, l);
        }
        tc::tmem_st32(s_at, reinterpret_cast<const uint32_t(&)[32]>(p[0]));
        tc::tmem_st32(s_at + 32, reinterpret_cast<const uint32_t(&)[32]>(p[32]));
      }
      tc::tc_fence_before();
      tc::mbar_arrive(&sm.p_ready[x]);
      first = false;
      ++mine;
    }
    if (!first) ok = __all_sync(FULL, ok && wait(sm, &sm.o_done[x], (mine - 1) & 1));
    tc::tc_fence_after();
    if (!ok) l = __int_as_float(0x7fc00000);  // (a wait that gave up: the rows are NaN)
    // the halves of shared rows: X = 1 leaves its sums in Q's place, X = 0 takes them
    float other = 0.f;
    if (shared) {
      asm volatile("bar.sync 1, 256;" ::: "memory");  // (both halves' products have read Q)
      if (x == 1 && warp_live) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          uint32_t r[32];
          tc::tmem_ld32(o_at + 32 * i, r);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4 *>(sm.q[0] + line * 512 + (((8 * i + e) ^ (line & 7)) << 4)) = first ? make_uint4(0, 0, 0, 0) : make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
        }
        sm.ml[line] = make_float2(m, l);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    if (warp_live && (x == 0 || !shared)) {
      float keep = first ? 0.f : 1.f;  // (a half without tiles has nothing in its accumulator)
      if (shared) {
        const float2 y = sm.ml[line];
        const float top = fmaxf(m, y.x);
        keep = first ? 0.f : ex2(m - top);
        other = ex2(y.x - top);
        l = l * ex2(m - top) + y.y * other;
        m = top;
      }
      const bool whole = w.n0 == 0 && w.n1 == w.tiles;
      const int row = w.r.start + col / k.group, head = w.head * k.group + col % k.group;
      const float f = l == 0.f ? 0.f : __ldg(k.c.v_scale + w.head) / l;
      float *const slot = k.tile_part + (((size_t)blockIdx.x * 2 + (w.n0 ? 0 : 1)) * 2 * ROWS + c) * PSTRIDE;
      uint16_t *const dst = out_row(k, row, head);
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        uint32_t r[32];
        tc::tmem_ld32(o_at + 32 * i, r);
        float4 o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          o[e] = first ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(__uint_as_float(r[4 * e]) * keep, __uint_as_float(r[4 * e + 1]) * keep, __uint_as_float(r[4 * e + 2]) * keep, __uint_as_float(r[4 * e + 3]) * keep);
          if (shared) {
            const float4 y = *reinterpret_cast<const float4 *>(sm.q[0] + line * 512 + (((8 * i + e) ^ (line & 7)) << 4));
            o[e] = make_float4(fmaf(y.x, other, o[e].x), fmaf(y.y, other, o[e].y), fmaf(y.z, other, o[e].z), fmaf(y.w, other, o[e].w));
          }
        }
        if (!live) continue;
        if (whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            reinterpret_cast<uint4 *>(dst)[4 * i + e] = pack8<TYPE>(make_float4(o[2 * e].x * f, o[2 * e].y * f, o[2 * e].z * f, o[2 * e].w * f),
                                                                    make_float4(o[2 * e + 1].x * f, o[2 * e + 1].y * f, o[2 * e + 1].z * f, o[2 * e + 1].w * f));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) __stcg(reinterpret_cast<float4 *>(slot) + 8 * i + e, o[e]);
        }
      }
      if (whole) {
        if (live && k.a.lse) k.a.lse[(size_t)row * k.a.q_heads + head] = lse_of(m, l);
      } else if (live) {
        __stcg(reinterpret_cast<float2 *>(slot + D), make_float2(m, l));
      }
    }
    tc::tc_fence_before();
    if (shared) asm volatile("bar.sync 1, 256;" ::: "memory");  // (Q's place is free again)
  } while (next_row(k, sm.before, hi, w));
}

// CTA of unit u when `ctas` CTAs share `total` units: CTA c has [total c / ctas, total (c + 1) / ctas)
__device__ __forceinline__ int cta_of(long long u, long long total, int ctas) { return (int)(((u + 1) * ctas - 1) / total); }

// the partial rows of row of work w, joined by the CTA that comes last
template <int TYPE> __device__ __forceinline__ void join_row(const Call &k, Smem &sm, const Row &w, long long total, int tid) {
  const int ctas = (int)min(total, (long long)gridDim.x), c0 = cta_of(w.unit0, total, ctas), c1 = cta_of(w.unit0 + w.tiles - 1, total, ctas);
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    sm.last = atomicAdd(k.tile_counters + c0, 1) == c1 - c0;
    if (sm.last) k.tile_counters[c0] = 0;
  }
  __syncthreads();
  if (!sm.last) return;
  __threadfence();
  const int rows = w.rows(k);
  for (int e = tid; e < rows * 32; e += THREADS) {
    const int c = e >> 5, x = e & 31, col = 2 * ROWS * w.pair + c;
    float m, l;
    const float4 o = join(c1 - c0 + 1, [&](int i) { return k.tile_part + (((size_t)(c0 + i) * 2 + (i ? 0 : 1)) * 2 * ROWS + c) * PSTRIDE; }, x, m, l);
    store_joined<TYPE>(k, w.r.start + col / k.group, w.head, w.head * k.group + col % k.group, x, o, m, l);
  }
  __syncthreads();
}

template <int TYPE> __global__ void __launch_bounds__(THREADS, 1) tile_kernel(const Call k) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem &sm = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      fbla::mbar_init(&sm.q_ready[i], ROWS);
      fbla::mbar_init(&sm.s_ready[i], 1);
      fbla::mbar_init(&sm.p_ready[i], ROWS);
      fbla::mbar_init(&sm.o_done[i], 1);
      fbla::mbar_init(&sm.k_full[i], 128);
      fbla::mbar_init(&sm.v_full[i], 128);
      fbla::mbar_init(&sm.k_empty[i], 2);
      fbla::mbar_init(&sm.v_empty[i], 2);
    }
    sm.abort = 0;
    fbla::mbar_init_fence();
  }
  fbla::wait_previous_pass();
  fbla::allow_next_pass();

  long long total = 0;
  for (int b0 = 0; b0 < k.a.batch; b0 += THREADS) {
    const int b = b0 + tid;
    long long n = 0;
    if (b < k.a.batch) {
      const Request r = request(k, b);
      if (taken(k, r)) {
        for (int p = 0; 2 * ROWS * p < rows_of(k, r); ++p) n += tiles_of(k, r, p);
        n *= k.c.kv_heads;
      }
    }
    long long sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(FULL, sum, o);
      if (lane >= o) sum += y;
    }
    if (lane == 31) sm.warp_sum[warp] = sum;
    __syncthreads();
    long long base = total;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) base += sm.warp_sum[i];
      total += sm.warp_sum[i];
    }
    if (b < k.a.batch) sm.before[b] = base + sum - n;
    __syncthreads();
  }
  if (tid == 0) sm.before[k.a.batch] = total;
  const int ctas = (int)min(total, (long long)gridDim.x);  // (each has a unit at least: a row's CTAs are consecutive)
  if ((int)blockIdx.x >= ctas) return;
  const long long lo = total * blockIdx.x / ctas, hi = total * (blockIdx.x + 1) / ctas;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(fbla::smem_u32(&sm.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();

  // 512 threads of 128 registers: 256 of 168 and 256 of 88
  if (warp < PRODUCER0) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    soften<TYPE>(k, sm, lo, hi, warp >> 2, warp, lane);
    asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < ISSUER0) produce(k, sm, lo, hi, warp - PRODUCER0, lane);
    else if (warp < ISSUER0 + 2 && lane == 0) issue(k, sm, lo, hi, warp - ISSUER0);
    __syncwarp();
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
  }

  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sm.tmem) : "memory");

  // the run's first and last rows of work, where they are cut
  Row w = first_row(k, sm.before, lo, hi);
  if (w.n0 > 0 || w.n1 < w.tiles) join_row<TYPE>(k, sm, w, total, tid);
  while (next_row(k, sm.before, hi, w))
    if (w.n1 < w.tiles) join_row<TYPE>(k, sm, w, total, tid);
}

}  // namespace

template <int TYPE> cudaError_t launch_tile(const Call &k, int sms, cudaStream_t stream) {
  static thread_local bool ready[64] = {false};
  const cudaError_t e = allow_shared(tile_kernel<TYPE>, ready);
  if (e != cudaSuccess) return e;
  return fbla::launch(true, 1, tile_kernel<TYPE>, dim3(sms), THREADS, 1024 + offsetof(Smem, before) + ((size_t)k.a.batch + 1) * sizeof(long long), stream, k);
}
template cudaError_t launch_tile<MLOPS_PAGED_BF16>(const Call &, int, cudaStream_t);
template cudaError_t launch_tile<MLOPS_PAGED_FP16>(const Call &, int, cudaStream_t);
static_assert(1024 + offsetof(Smem, before) + (PAGED_K_MAX_ATTENDED + 1) * sizeof(long long) <= 232448, "the operands and the largest batch fit");

}  // namespace paged
