// Attention over the paged cache for many queries per request (mlops_paged_attend, mlops_paged_cross_attend, mlops_paged_attend_shared: paged_tile*.cu): chunks of prompts, whole prompts,
// target texts, the common tokens of many requests, on tcgen05 tensor cores with TMEM accumulators.
//
// A row of work is (item, KV head, 256 rows); row c of an item and KV head is query c / group with query head c % group. Its units are HEAD and then the
// tiles of 128 tokens that its last row sees. All units form one list, of which every CTA has an equal contiguous run; a row of work that is cut is joined from
// partial rows (o, m', l), in the order of the tokens, by the CTA that comes last or (mlops_paged_attend_shared) by merge_kernel.
//
// Per tile of tokens and half X of the rows (128 each), with FP32 accumulators in tensor memory:
//   S_X[128 x 128] = Q_X K^T,   O_X[128 x 128] += P_X V
// K and V are code * scale, exact in FP16; Q is FP16 after a power of two per row (paged_attend.cuh); P = 2^(s - m') in FP16 takes S_X's place in tensor
// memory, rounded as in paged_stream.cuh. m' moves only where a score would pass 2^15, then O and l are rescaled; l sums the unrounded P. Rows of at most
// 128 use both halves too: the even tiles of tokens go to X = 0, the odd ones to X = 1, with the same queries, and the halves are joined at the end.
//
// Everything goes 64 tokens of a tile at a time: while the softmax has the second half of a tile, the first half's P is multiplied and the next tile's first scores take its place, so that
// the softmax finds scores whenever it is through. Each X has four warps, a thread per row, and a thread of its own that issues its products; the two X only share the operands.
// A tile takes 3 800 cycles. Its exponentials are 2 048 (16 per cycle and SM), its products 2 048 at their rate, but the scores' with 64 tokens read Q again for each half and are
// bound by shared memory: 2 560 in all, beside 512 of the operands' stores. Measured (clocks in the kernel): a thread's half takes 1 300 to 1 500 cycles, of which the exponentials, both X's
// at once, are 1 100; some 250 are the way through barriers; the issuing threads wait for the tensor cores two thirds of the time. Instructions are fetched at that rate too: the same code with
// the two halves' softmax unrolled took 1.27 times the time, with the rare path's exponentials apart 1.02, with a mask that the compiler predicates 1.04. Two prompts of 8192 tokens, 32 / 8 heads:
// 1.22 ms = 900 TFLOP/s, 0.54 of the measured burst rate. Tried: scores 128 tokens at a time (4 600 cycles: softmax and products of an X in turn), with both X's softmax in turn (5 000), with 32
// scores on their way while 32 are used (5 150); eight warps for X = 0 and then for X = 1, two threads per row (4 300); all 64 scores in registers for both passes (1.03 times the time); a third of
// the exponentials as polynomials on the FMA units, then 1.07 times the time; operand warps that look up their blocks themselves (the registers spill, and every load is waited for at once). The kernel
// stores 28 to 60 bytes of registers per thread to local memory and loads 108 to 204.
//
// Around the tiles a CTA spends some 45 000 cycles: its code comes from the L2 (10 cycles per instruction that is run for the first time), lengths, table, queries and pages are read one after the
// other (16 000 until the first product), the first tile takes 9 000 more than the others, the sums' way out 7 000.
//
// Warps 0-7: softmax. Warps 8-15: operands, from packed pages to two stages each of K and V in shared
// memory, token rows of 128 bytes (64 channels) with 16-byte chunk c of row r at c ^ (r % 8): for S that is K-major, for O V's MN-major. Warps 16, 17: one thread
// each issues the products of its X. Warp 18 looks up where the tiles' blocks lie. Every wait is bounded: where one gives up, the rows become NaN.
#pragma once
#include "fbla_launch.h"
#include "fbla_tc.cuh"
#include "paged_attend.cuh"
#include <climits>

namespace paged {
namespace {

namespace tc = fbla::tc;

constexpr int ROWS = 128;  // of a product, with 128 tokens
constexpr int SLAB = 128 * 128, TILE = 2 * SLAB;  // bytes of a slab (128 rows of 64 channels) and of an operand
constexpr int STAGES = 2, PRODUCER0 = 8, PRODUCERS = 8, ISSUER0 = 16, FINDER = 18, THREADS = 20 * 32;  // (four warps share a register count: 19 idles)
constexpr int WINDOW = 16;  // tiles whose blocks are looked up at a time
constexpr int NO_TILE = -0x7fffffff;
constexpr float TOP = 15.f, REST = 9.f;
constexpr long long WAIT_CYCLES = 2000000000;
constexpr uint32_t IDESC_S = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24),  // N 64: the scores of half of a tile
                    IDESC_O = tc::IDESC_F16 | (1u << 16);  // V: MN-major

// a row of work and its part in this CTA's run: tiles of tokens n0 .. n1 - 1 of `tiles`
template <int MODE> struct Row {
  Request<MODE> r;
  int b, head, pair, tiles, n0, n1;
  long long unit0;
  __device__ __forceinline__ int rows(const Call &k) const { return min(rows_of(k, r) - 2 * ROWS * pair, 2 * ROWS); }
  __device__ __forceinline__ bool halves(const Call &k) const { return rows(k) <= ROWS; }  // both X have the same rows
};
template <int MODE> struct __align__(1024) Smem {
  uint8_t q[2][TILE];
  uint8_t k[STAGES][TILE], v[STAGES][TILE];
  const uint8_t *block[2 * WINDOW][8];  // [tile of the run % (2 WINDOW)][block]: where it lies; null: the table names no page, or the request has no such block
  int left[2 * WINDOW];         // tokens of the request from the tile's first on
  uint64_t places_full[2], places_empty[2];  // of WINDOW tiles each
  uint64_t drained[2];  // the issuing threads' products, after a wait that gave up
  uint64_t q_ready[2], k_full[STAGES], v_full[STAGES], k_empty[STAGES], v_empty[STAGES], s_ready[2][2], p_ready[2][2], o_done[2][2];  // [X], [X][half of the tokens]
  uint8_t there[4][8];  // [tile of tokens % 4][block]: 1 where the table names a page
  float down[2][ROWS];      // the rows' factors
  float2 exchange[2][ROWS];  // (m, l) between the two threads of a row that both X have, l -1 where one has seen no tile
  int v_nan, nan_from[8];   // some V of the run has a NaN scale; [16 channels] of a row of work: the first token with one
  Row<MODE> begin, row[8];  // the run's first row of work; the softmax warps' rows
  long long warp_sum[THREADS / 32];
  uint32_t tmem;
  int abort, last;
  int others, share;  // SHARED: the stream's units, the CTAs that have tiles
  long long before[];   // [items + 1]: the items' first units
};

// waits for the phase with the given parity, about a second at most; gives up at once where another thread has
template <int MODE> __device__ __forceinline__ bool wait(Smem<MODE> &sm, uint64_t *bar, uint32_t parity) {
  if (tc::try_wait_hint(bar, parity)) return true;
  for (const long long begin = clock64(); clock64() - begin < WAIT_CYCLES;) {
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

// a / b for a >= 0, b > 0: in 32 bits where both have no more
__device__ __forceinline__ long long divide(long long a, long long b) { return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b); }

// the first row of work of the run [lo, hi), found by a warp
template <int MODE> __device__ __forceinline__ Row<MODE> first_row(const Call &k, const long long *before, long long lo, long long hi, int lane) {
  Row<MODE> w;
  int a = 0;
  for (int e = items_of<MODE>(k); e - a > 1;) {
    const int mid = (a + e) >> 1;
    if (before[mid] <= lo) a = mid; else e = mid;
  }
  w.b = a;
  w.r = request<MODE>(k, a);
  const long long per_head = divide(before[a + 1] - before[a], k.c.kv_heads), x = lo - before[a];
  w.head = (int)divide(x, per_head);
  long long rest = x - w.head * per_head;
  for (int pair0 = 0;; pair0 += 32) {  // 32 pairs at a time
    const int pair = pair0 + lane, units = 2 * ROWS * pair < rows_of(k, w.r) ? HEAD + tiles_of<MODE>(k, w.r, pair) : 0;
    int sum = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(FULL, sum, o);
      if (lane >= o) sum += y;
    }
    const uint32_t behind = __ballot_sync(FULL, sum > rest);
    const int here = behind ? __ffs(behind) - 1 : 31;
    const int through = __shfl_sync(FULL, sum, here), own = __shfl_sync(FULL, units, here);
    if (behind) {
      w.pair = pair0 + here;
      w.tiles = own - HEAD;
      rest -= through - own;
      break;
    }
    rest -= through;
  }
  w.n0 = max((int)rest - HEAD, 0);
  w.unit0 = lo - rest;
  w.n1 = (int)min((long long)w.tiles, hi - w.unit0 - HEAD);  // (not above n0 where the run ends before the row's first tile)
  return w;
}
// the row of work behind w in the run; false where none has a tile in it, and w as it was
template <int MODE> __device__ __forceinline__ bool next_row(const Call &k, const long long *before, long long hi, Row<MODE> &w) {
  const long long unit0 = w.unit0 + HEAD + w.tiles;
  if (unit0 + HEAD >= hi) return false;
  w.unit0 = unit0;
  if (2 * ROWS * ++w.pair >= rows_of(k, w.r)) {
    w.pair = 0;
    if (++w.head == k.c.kv_heads) {
      w.head = 0;
      do ++w.b; while (before[w.b + 1] <= unit0);
      w.r = request<MODE>(k, w.b);
    }
  }
  w.tiles = tiles_of<MODE>(k, w.r, w.pair);
  w.n0 = 0;
  w.n1 = (int)min((long long)w.tiles, hi - unit0 - HEAD);
  return true;
}
// whether half X has a part in tile n of w: w's second half in row order, or every second tile where the halves share the rows; a first half
// whose rows see less than the second one's leaves the last tile out
template <int MODE> __device__ __forceinline__ int tiles_of_half(const Call &k, const Row<MODE> &w, int x) {
  const int last = min(2 * ROWS * w.pair + ROWS * (x + 1), rows_of(k, w.r)) - 1, seen = min(limit_of<MODE>(w.r, query_of(k, last)) + 1, w.r.tokens);
  return max((seen + TOKENS - 1) / TOKENS, 1);
}
struct Part {
  bool shared;
  int limit;  // tiles
  __device__ __forceinline__ bool has(int n, int x) const { return shared ? (n & 1) == x : n < limit; }
};

// ---- operands -------------------------------------------------------------------------------------------------------------------
struct Raw {  // a lane's part of a tensor's block: two of its tokens, 32 channels of each
  uint4 codes[2];
  uint32_t scales[2];
};
__device__ __forceinline__ void load_raw(Raw &x, const uint8_t *block, int codes, int scales, int lane) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int token = 8 * i + (lane & 7), quarter = lane >> 3;
    x.codes[i] = make_uint4(0, 0, 0, 0);
    x.scales[i] = 0;
    if (block) {
      x.codes[i] = __ldg(reinterpret_cast<const uint4 *>(block + codes + token * CODE_BYTES + 16 * quarter));
      x.scales[i] = __ldg(reinterpret_cast<const uint16_t *>(block + scales + token * SCALE_BYTES + 2 * quarter));
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
  for (int i = 0; i < 2; ++i) {
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

// bit 7 of every byte of four scales that is NaN (0x7f, 0xff)
__device__ __forceinline__ uint32_t nan_scales(uint32_t scales) { return ((scales & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Where the run's blocks lie, two lanes per tile, up to 32 tiles ahead of the producers, NO_TILE behind the last one: by one warp.
template <int MODE> __device__ __forceinline__ void look_up(const Call &k, Smem<MODE> &sm, long long hi, int lane) {
  const int per_page = k.c.page_size / BT, half = lane & 1;
  Row<MODE> w = sm.begin;
  int reached = 0, n = w.n0;  // the tile that this lane looked up last, in the run and in its row of work
  bool ok = true, more = true;
  for (int i = 0; ok && __all_sync(FULL, more); ++i) {
    if (i >= 2) ok = wait(sm, &sm.places_empty[i & 1], (i / 2 & 1) ^ 1);
    const int tile = WINDOW * i + (lane >> 1);
    n += tile - reached;
    reached = tile;
    while (more && n >= w.n1) {
      n -= w.n1;
      more = next_row(k, sm.before, hi, w);
    }
    if (half == 0) sm.left[tile % (2 * WINDOW)] = more ? w.r.tokens - TOKENS * n : NO_TILE;
    if (more) {
      const int *const entries = table_row<MODE>(k, w.r, w.b);
      const uint8_t *const head = k.c.units + (size_t)w.head * k.c.head_stride;
      const int number = 8 * n + 4 * half;
      const int in_row = number + first_token<MODE>(w.r) / BT;
      int column = in_row / per_page, at = in_row - column * per_page;
      int page[4], in_page[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // (all on their way before the first is used)
        page[j] = (number + j) * BT < w.r.tokens ? __ldg(entries + column) : -1;
        in_page[j] = at;
        if (++at == per_page) at = 0, ++column;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sm.block[tile % (2 * WINDOW)][4 * half + j] = (unsigned)page[j] < (unsigned)k.c.pages ? head + (size_t)page[j] * k.c.page_stride + (size_t)in_page[j] * BLOCK_BYTES : nullptr;
    }
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.places_full[i & 1]);
  }
}

// Producer warp `warp` turns block `warp` of every tile into rows 16 warp .. of the operands, K of a tile before V of the tile before it, which is wanted
// later; a tensor's codes are loaded while its last tile's are waited for and used.
template <int MODE> __device__ __forceinline__ void produce(Smem<MODE> &sm, int warp, int lane) {
  struct Place {
    const uint8_t *block;
    int left;  // the request's tokens from the block's first on; NO_TILE: behind the run
  };
  bool ok = true;
  auto place = [&](int tile) {
    if (tile % WINDOW == 0) {
      const int i = tile / WINDOW;
      if (i && lane == 0) tc::mbar_arrive(&sm.places_empty[(i & 1) ^ 1]);
      ok = ok && wait(sm, &sm.places_full[i & 1], i >> 1 & 1);
    }
    Place p{nullptr, ok ? sm.left[tile % (2 * WINDOW)] : NO_TILE};
    if (p.left != NO_TILE) {
      p.block = sm.block[tile % (2 * WINDOW)][warp];
      p.left -= BT * warp;
    }
    return p;
  };
  auto store = [&](uint8_t *tile, const Raw &x, uint64_t *full) {
    store_operand(tile, x, 16 * warp, lane);
    fbla::fence_async_smem();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(full);
  };
  auto store_k = [&](int tile, const Raw &x, bool there) {
    const int stage = tile % STAGES;
    if (tile >= STAGES) ok = ok && wait(sm, &sm.k_empty[stage], (tile / STAGES & 1) ^ 1);
    ok = __all_sync(FULL, ok);
    if (lane == 0) sm.there[tile & 3][warp] = there;
    store(sm.k[stage], x, &sm.k_full[stage]);
  };
  Raw rk, rv;
  Place now = place(0), next;
  load_raw(rk, now.block, 0, K_SCALES, lane);
  load_raw(rv, now.block, V_CODES, V_SCALES, lane);
  store_k(0, rk, now.block != nullptr);
  next = place(1);
  load_raw(rk, next.block, 0, K_SCALES, lane);
#pragma unroll 1
  for (int at = 0; now.left != NO_TILE && ok; ++at) {
    Place behind = next;
    if (next.left != NO_TILE) {
      behind = place(at + 2);
      store_k(at + 1, rk, next.block != nullptr);
      load_raw(rk, behind.block, 0, K_SCALES, lane);
    }
    if (now.left < BT) {  // (what is stored behind the last token may be anything, NaN too)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (8 * i + (lane & 7) >= now.left) rv.scales[i] = 0;
    }
    // (0 times NaN is NaN, for rows too that do not see the token: such scales are taken as 0, and spoil_rows puts NaN into the rows that see them)
    if (const uint32_t nan = nan_scales(rv.scales[0] | rv.scales[1] << 16)) {
      const uint32_t keep = ~((nan >> 7) * 255u);
      rv.scales[0] &= keep;
      rv.scales[1] &= keep >> 16;
      sm.v_nan = 1;
    }
    if (at >= STAGES) ok = ok && wait(sm, &sm.v_empty[at % STAGES], (at / STAGES & 1) ^ 1);
    ok = __all_sync(FULL, ok);
    store(sm.v[at % STAGES], rv, &sm.v_full[at % STAGES]);
    load_raw(rv, next.block, V_CODES, V_SCALES, lane);
    now = next;
    next = behind;
  }
}

// ---- products -------------------------------------------------------------------------------------------------------------------
// The way from P to the next scores of the same half of a tile has to be shorter than the softmax of the other half: nothing else is waited for or released on it. A stage is free when both X
// have read it; where a tile is one X's alone, that one arrives for the other.
template <int MODE> __device__ __forceinline__ void issue(const Call &k, Smem<MODE> &sm, long long hi, int x) {  // by one thread
  const uint32_t s_at = sm.tmem + 128 * x, o_at = sm.tmem + 256 + 128 * x;
  uint32_t row_at = 0, mine = 0, items = 0;  // tiles of the run before the row, of this X; rows of work
  bool ok = true;
  Row<MODE> w = sm.begin;
  do {
    const bool shared = w.halves(k);
    const int step = shared ? 2 : 1, end = shared ? w.n1 : min(w.n1, tiles_of_half(k, w, x)), both = shared ? 0 : tiles_of_half(k, w, 0);  // tiles below `both` are both X's
    const uint8_t *const q = sm.q[shared ? 0 : x];
    int n = w.n0 + (shared && (w.n0 & 1) != x);
    auto at = [&](int n) { return row_at + (n - w.n0); };
    auto scores = [&](int h) {
      const int stage = at(n) % STAGES;
      tc::tc_fence_after();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t offset = (i >> 2) * SLAB + (i & 3) * 32;
        tc::mma_f16(s_at + 64 * h, tc::smem_desc_at(q, offset), tc::smem_desc_at(sm.k[stage], offset + 64 * 128 * h), IDESC_S, i > 0);
      }
      tc::mma_commit(&sm.s_ready[x][h]);
      if (h == 0) return;
      tc::mma_commit(&sm.k_empty[stage]);
      if (n >= both) tc::mbar_arrive(&sm.k_empty[stage]);
    };
    ok = ok && wait(sm, &sm.q_ready[x], items++ & 1);
    if (n < end) {
      ok = ok && wait(sm, &sm.k_full[at(n) % STAGES], at(n) / STAGES & 1);
      if (ok) scores(0), scores(1);
    }
    for (bool first = true; n < end && ok; first = false) {
      const int stage = at(n) % STAGES, alone = n >= both, here = n;
      ok = wait(sm, &sm.v_full[stage], at(n) / STAGES & 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ok = ok && wait(sm, &sm.p_ready[x][h], mine & 1);
        if (!ok) break;
        tc::tc_fence_after();
#pragma unroll
        for (int i = 0; i < 4; ++i) tc::mma_f16_ts(o_at, s_at + 64 * h + 8 * i, v_desc(sm.v[stage], (4 * h + i) * 2048), IDESC_O, !first || h > 0 || i > 0);
        tc::mma_commit(&sm.o_done[x][h]);
        n = here + step;
        if (n < end) {  // the next tile's scores of this half (P is in their place: its products have to be through)
          ok = (h || wait(sm, &sm.k_full[at(n) % STAGES], at(n) / STAGES & 1)) && wait(sm, &sm.o_done[x][h], mine & 1);
          if (ok) scores(h);
        }
      }
      if (!ok) break;
      if (n < end) tc::mbar_arrive(&sm.v_empty[stage]);
      else tc::mma_commit(&sm.v_empty[stage]);
      if (alone) tc::mbar_arrive(&sm.v_empty[stage]);
      ++mine;
    }
    row_at += w.n1 - w.n0;
  } while (next_row(k, sm.before, hi, w));
}

// ---- softmax --------------------------------------------------------------------------------------------------------------------
// Warps 0-3 have the rows of X = 0, a thread each, warps 4-7 those of X = 1. Where both X have the same rows, warps w and w + 4 join their sums, each for half of the channels.
__device__ __forceinline__ void pair_meet(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); }

// the larger magnitudes of two pairs of 16-bit numbers (NaN where both are)
template <int TYPE> __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
  uint32_t y;
  if (TYPE == MLOPS_PAGED_BF16) asm("{.reg .b32 x;\n\tabs.bf16x2 x, %2;\n\tmax.bf16x2 %0, %1, x;}" : "=r"(y) : "r"(a), "r"(b));
  else asm("{.reg .b32 x;\n\tabs.f16x2 x, %2;\n\tmax.f16x2 %0, %1, x;}" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

// Q's rows first + 32 quarter .. of the row of work as FP16 in `tile`, each times a power of two (q_factor) whose inverse goes to `down`; by a warp, four lanes of 32 channels each
// per row, all loads ahead of the arithmetic
template <int TYPE, int MODE> __device__ __forceinline__ void load_q(const Call &k, const Row<MODE> &w, int first, uint8_t *tile, float *down, int quarter, int lane) {
  const int part = lane & 3, rows = w.rows(k) - first - 32 * quarter, line0 = 32 * quarter + (lane >> 2);
  int query, head;
  split_column(k, 2 * ROWS * w.pair + first + 32 * quarter + min(lane, max(rows - 1, 0)), query, head);
  const long long mine = (int64_t)(w.r.start + query) * k.a.q_token_stride + (int64_t)(w.head * k.group + head) * k.a.q_head_stride;  // of the lane's row
  uint4 raw[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * i + (lane >> 2);
    const uint4 *const from = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(k.a.q) + __shfl_sync(FULL, mine, row)) + 4 * part;
#pragma unroll
    for (int e = 0; e < 4; ++e) raw[i][e] = row < rows ? __ldg(from + e) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int line = line0 + 8 * i;
    uint32_t tops = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) tops = larger<TYPE>(larger<TYPE>(larger<TYPE>(larger<TYPE>(tops, raw[i][e].x), raw[i][e].y), raw[i][e].z), raw[i][e].w);
    const float2 t = to_floats<TYPE>(tops);
    float top = fmaxf(t.x, t.y);
    top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
    top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
    float inverse;
    const float up = q_factor(__float_as_uint(top) & 0x7fffffffu, inverse);
    if (part == 0) down[line] = inverse;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t word[4] = {raw[i][e].x, raw[i][e].y, raw[i][e].z, raw[i][e].w};
      uint32_t h[4];
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const float2 x = __fmul2_rn(to_floats<TYPE>(word[f]), make_float2(up, up));
        h[f] = from_floats<MLOPS_PAGED_FP16>(x.x, x.y);
      }
      *reinterpret_cast<uint4 *>(tile + (part >> 1) * SLAB + line * 128 + (((4 * (part & 1) + e) ^ (line & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
}

// 32 columns of the thread's lane from `at` on, to be waited for (tcgen05.wait::ld); PAGED_HOLD32 behind the wait keeps every use of them behind it
#define PAGED_LD32(at, r) \
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];" \
               : "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]), "=r"((r)[6]), "=r"((r)[7]), "=r"((r)[8]), "=r"((r)[9]), "=r"((r)[10]), "=r"((r)[11]), \
                 "=r"((r)[12]), "=r"((r)[13]), "=r"((r)[14]), "=r"((r)[15]), "=r"((r)[16]), "=r"((r)[17]), "=r"((r)[18]), "=r"((r)[19]), "=r"((r)[20]), "=r"((r)[21]), "=r"((r)[22]), \
                 "=r"((r)[23]), "=r"((r)[24]), "=r"((r)[25]), "=r"((r)[26]), "=r"((r)[27]), "=r"((r)[28]), "=r"((r)[29]), "=r"((r)[30]), "=r"((r)[31]) : "r"(at) : "memory")
#define PAGED_HOLD32(r) \
  asm volatile("" : "+r"((r)[0]), "+r"((r)[1]), "+r"((r)[2]), "+r"((r)[3]), "+r"((r)[4]), "+r"((r)[5]), "+r"((r)[6]), "+r"((r)[7]), "+r"((r)[8]), "+r"((r)[9]), "+r"((r)[10]), "+r"((r)[11]), \
                    "+r"((r)[12]), "+r"((r)[13]), "+r"((r)[14]), "+r"((r)[15]), "+r"((r)[16]), "+r"((r)[17]), "+r"((r)[18]), "+r"((r)[19]), "+r"((r)[20]), "+r"((r)[21]), "+r"((r)[22]), \
                    "+r"((r)[23]), "+r"((r)[24]), "+r"((r)[25]), "+r"((r)[26]), "+r"((r)[27]), "+r"((r)[28]), "+r"((r)[29]), "+r"((r)[30]), "+r"((r)[31]))
struct Scores {  // 32 of a row's
  uint32_t r[32];
  __device__ __forceinline__ void load(uint32_t at) {
    PAGED_LD32(at, r);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    PAGED_HOLD32(r);
  }
  __device__ __forceinline__ float score(int i) const { return __uint_as_float(r[i]); }
  // scores of tokens above `last` and of blocks whose byte in `there` is 0 become -infinity
  __device__ __forceinline__ void mask(int last, uint32_t there) {
    __syncwarp();  // (a branch: the warps that need no mask do not run it)
    const int n = min(max(last + 1, 0), 32);  // tokens that are seen
    const uint32_t seen = (((there & 1) * 0xffffu) | ((there >> 8 & 1) * 0xffff0000u)) & (n ? ~0u >> (32 - n) : 0u);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (!(seen >> i & 1)) r[i] = __float_as_uint(-FBLA_INF);
  }
  __device__ __forceinline__ float largest() const {
    float top[4] = {NOTHING, NOTHING, NOTHING, NOTHING};
#pragma unroll
    for (int i = 0; i < 16; ++i) top[i & 3] = fbla::max3(top[i & 3], score(2 * i), score(2 * i + 1));
    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  }
  // 2^(score mult - m) as 16 words of FP16 pairs in r; their sum
  __device__ __forceinline__ float exponentials(float mult, float m) {
    float2 sum[2] = {};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 e = __ffma2_rn(make_float2(score(2 * i), score(2 * i + 1)), make_float2(mult, mult), make_float2(-m, -m));
      const float2 f = make_float2(ex2(e.x), ex2(e.y));
      sum[i & 1] = __fadd2_rn(sum[i & 1], f);
      r[i] = from_floats<MLOPS_PAGED_FP16>(f.x, f.y);
    }
    return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
  }
  __device__ __forceinline__ void store(uint32_t at) const {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
                 "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
  }
};

// a thread's row
struct Line {
  float m, l, mult;
  int limit;     // the last token that the row sees
  bool started;  // O holds sums, or will
};

// 64 tokens of a tile, from first_token on: scores in tensor memory at s become P there. o_done: of the products with the 64 tokens before. The scores are read twice, for their maximum and
// for their exponentials, 32 at a time.
template <int MODE>
__device__ __forceinline__ bool take_half(Smem<MODE> &sm, Line &q, uint32_t s, uint32_t o, int first_token, int low, uint32_t blocks, uint64_t *o_done, uint32_t o_parity) {
  const bool mask = first_token + 63 > low || blocks != 0x01010101u;  // some row does not see all of them
  bool ok = true;
  float high = NOTHING, sum = 0.f;
  Scores x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x.load(s + 32 * i);
    if (mask) x.mask(q.limit - first_token - 32 * i, blocks >> (16 * i));
    high = fmaxf(high, x.largest());
  }
  high *= q.mult;  // (mult is positive)
  if (__any_sync(FULL, high - q.m > TOP)) {
    float keep = 1.f;
    if (high - q.m > TOP) {
      keep = ex2(q.m - (high - REST));
      q.m = high - REST;
    }
    q.l *= keep;
    if (q.started) {
      ok = __all_sync(FULL, wait(sm, o_done, o_parity));
      tc::tc_fence_after();
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        uint32_t y[16];
        tc::tmem_ld16(o + 16 * i, y);
        tc::tmem_ld_wait(y);
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * keep);
        tc::tmem_st8(o + 16 * i, reinterpret_cast<const uint32_t(&)[8]>(y[0]));
        tc::tmem_st8(o + 16 * i + 8, reinterpret_cast<const uint32_t(&)[8]>(y[8]));
      }
      tc::tmem_st_wait();
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x.load(s + 32 * i);
    if (mask) x.mask(q.limit - first_token - 32 * i, blocks >> (16 * i));
    sum += x.exponentials(q.mult, q.m);
    x.store(s + 16 * i);  // (where the thread's own scores have been read)
  }
  tc::tmem_st_wait();
  q.l += sum;
  q.started = true;
  return ok;
}

// CTA of unit u when `ctas` CTAs share `total` units: CTA c has [total c / ctas, total (c + 1) / ctas)
__device__ __forceinline__ int cta_of(long long u, long long total, int ctas) { return (int)(((u + 1) * ctas - 1) / total); }

template <int TYPE, int MODE> __device__ __forceinline__ void soften(const Call &k, Smem<MODE> &sm, long long hi, int warp, int lane) {
  const int x = warp >> 2, quarter = warp & 3, line = 32 * quarter + lane;
  const uint32_t lanes = (uint32_t)(32 * quarter) << 16, s_at = sm.tmem + 128 * x + lanes, o_at = sm.tmem + 256 + lanes;
  uint32_t mine = 0, at = 0;
  bool ok = true;
  Row<MODE> &w = sm.row[warp];  // (not in registers: they are all needed)
  if (lane == 0) w = sm.begin;
  __syncwarp();
  bool more;
  do {
    const bool shared = w.halves(k);
    const int row0 = shared ? 0 : ROWS * x, rows = w.rows(k) - row0;  // the X's rows: row0 .. of the row of work
    if (!shared || x == 0) {  // (the warp's part of Q's place: nobody else writes or, its products being through, reads there)
      load_q<TYPE, MODE>(k, w, row0, sm.q[x], sm.down[x], quarter, lane);
      fbla::fence_async_smem();
    }
    __syncwarp();
    if (shared) pair_meet(quarter);
    if (lane == 0 && (!shared || x == 0)) {
      tc::mbar_arrive(&sm.q_ready[x]);
      if (shared) tc::mbar_arrive(&sm.q_ready[1]);
    }
    const bool warp_live = 32 * quarter < rows;
    const int col = 2 * ROWS * w.pair + row0 + line;  // of the item
    Line q{NOTHING, 0.f, fmaxf(k.sl * __ldg(k.c.k_scale + w.head) * sm.down[shared ? 0 : x][line], 1e-37f),  // (mult is not 0: masked scores are -infinity)
           line < rows ? limit_of<MODE>(w.r, query_of(k, col)) : -1, false};
    const int low = limit_of<MODE>(w.r, query_of(k, col - lane));  // the smallest limit of the warp's rows
    const Part part{shared, tiles_of_half(k, w, x)};
    const int n0 = w.n0, n1 = w.n1;
    bool any = false;
#pragma unroll 1
    for (int n = n0; n < n1; ++n, ++at) {
      if (!part.has(n, x)) continue;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        ok = __all_sync(FULL, ok && wait(sm, &sm.s_ready[x][h], mine & 1));
        tc::tc_fence_after();
        if (warp_live)
          ok &= take_half(sm, q, s_at + 64 * h, o_at + 128 * x, TOKENS * n + 64 * h, low, *reinterpret_cast<const uint32_t *>(sm.there[at & 3] + 4 * h), &sm.o_done[x][h ^ 1],
                          h ? mine & 1 : (mine - 1) & 1);
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sm.p_ready[x][h]);
      }
      any = true;
      ++mine;
    }
    if (any) ok = __all_sync(FULL, ok && wait(sm, &sm.o_done[x][1], (mine - 1) & 1));
    tc::tc_fence_after();

    // Outputs of whole rows in 16 bits, or sums: through the warp's part of Q's place, from where a half-warp or less stores a row at a time
    const bool whole = w.n0 == 0 && w.n1 == w.tiles, sums = MODE == SHARED || !whole;
    float m = q.m, l = q.l, keep = any ? 1.f : 0.f, other = 0.f;
    if (!ok) l = __int_as_float(0x7fc00000);  // (a wait that gave up: the rows are NaN)
    if (shared) {  // both X's sums are of these rows; this thread has 64 of the channels
      sm.exchange[x][line] = make_float2(m, any ? l : -1.f);
      tc::tc_fence_before();
      pair_meet(quarter);
      tc::tc_fence_after();
      const float2 y = sm.exchange[x ^ 1][line];
      const bool both = y.y != -1.f;
      const float top = both ? fmaxf(m, y.x) : m;
      keep = any ? ex2(m - top) : 0.f;
      other = both ? ex2(y.x - top) : 0.f;
      l = (any ? l * keep : 0.f) + (both ? y.y * other : 0.f);
      m = top;
    }
    const float f = l == 0.f ? 0.f : __ldg(k.c.v_scale + w.head) / l;
    auto slot = [&](int c) {  // where row c's sums go
      if constexpr (MODE == SHARED)
        if (whole) {
          int query, head;
          split_column(k, 2 * ROWS * w.pair + c, query, head);
          return sums_row(k, w.r.common, w.r.start + query, w.head * k.group + head);
        }
      return k.tile_part + (((size_t)blockIdx.x * 2 + (w.n0 ? 0 : 1)) * 2 * ROWS + c) * PSTRIDE;
    };
    uint8_t *const place = sm.q[x] + 32 * quarter * 128;  // 16-byte piece i < 8 of the warp's row r at r * 128 + 16 (i ^ r % 8), pieces from 8 on a slab further
    const int wide = sums ? 4 : 8, pieces = !sums && shared ? 8 : 16, span = wide * pieces;  // channels of a piece, pieces of a row at a time, channels at a time
    if (warp_live) {
#pragma unroll 1
      for (int ch0 = shared ? 64 * x : 0; ch0 < (shared ? 64 * x + 64 : D); ch0 += span) {
#pragma unroll 1
        for (int i = 0; i < span / 16; ++i) {
          uint32_t r[16], y[16];
          float o[16];
          tc::tmem_ld16(o_at + (shared ? 0 : 128 * x) + ch0 + 16 * i, r);
          tc::tmem_ld_wait(r);
          const float a = shared && x ? other : keep, b = shared && x ? keep : other;  // of X = 0's sums, of X = 1's where the rows are both's
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = a == 0.f ? 0.f : __uint_as_float(r[e]) * a;  // (an X without tiles has nothing in its accumulator)
          if (shared) {
            tc::tmem_ld16(o_at + 128 + ch0 + 16 * i, y);
            tc::tmem_ld_wait(y);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = b == 0.f ? o[e] : fmaf(__uint_as_float(y[e]), b, o[e]);
          }
          auto piece = [&](int p) { return reinterpret_cast<uint4 *>(place + (p >> 3) * SLAB + lane * 128 + (((p & 7) ^ (lane & 7)) << 4)); };
          if (sums) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<float4 *>(piece(4 * i + e)) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *piece(2 * i + e) = pack8<TYPE>(make_float4(o[8 * e] * f, o[8 * e + 1] * f, o[8 * e + 2] * f, o[8 * e + 3] * f),
                                              make_float4(o[8 * e + 4] * f, o[8 * e + 5] * f, o[8 * e + 6] * f, o[8 * e + 7] * f));
          }
        }
        __syncwarp();
        const int p = lane & (pieces - 1), live = min(rows - 32 * quarter, 32);
#pragma unroll 4
        for (int r = lane / pieces; r < live; r += 32 / pieces) {
          const uint4 v = *reinterpret_cast<const uint4 *>(place + (p >> 3) * SLAB + r * 128 + (((p & 7) ^ (r & 7)) << 4));
          const int c = row0 + 32 * quarter + r;
          if (sums) {
            __stcg(reinterpret_cast<uint4 *>(slot(c) + ch0) + p, v);
          } else {
            int query, head;
            split_column(k, 2 * ROWS * w.pair + c, query, head);
            reinterpret_cast<uint4 *>(out_row(k, w.r.start + query, w.head * k.group + head) + ch0)[p] = v;
          }
        }
        __syncwarp();
      }
    }
    if (line < rows && (!shared || x == 0)) {
      const int c = row0 + line;
      int query, head;
      split_column(k, 2 * ROWS * w.pair + c, query, head);
      if constexpr (MODE == SHARED) {
        if (whole) __stcg(reinterpret_cast<float4 *>(slot(c) + D), row_end(w.r, m, l));
        else __stcg(reinterpret_cast<float2 *>(slot(c) + D), make_float2(m, l));
        if (!whole && w.n0 == 0) {
          const long long total = sm.before[items_of<MODE>(k)];
          const int pieces = cta_of(w.unit0 + HEAD + w.tiles - 1, total, (int)min(total, (long long)sm.share)) - blockIdx.x + 1;
          __stcg(reinterpret_cast<float4 *>(sums_row(k, w.r.common, w.r.start + query, w.head * k.group + head) + D),
                 pieces_end(w.r, (int)((k.tile_part - k.stream_part) / PSTRIDE) + (blockIdx.x * 2 + 1) * 2 * ROWS + c, 2 * ROWS, pieces));
        }
      } else if (!whole) __stcg(reinterpret_cast<float2 *>(slot(c) + D), make_float2(m, l));
      else if (k.a.lse) k.a.lse[(size_t)(w.r.start + query) * k.a.q_heads + w.head * k.group + head] = lse_of(m, l);
    }
    tc::tc_fence_before();
    if (shared) pair_meet(quarter);  // (both have read both X's sums)
    __syncwarp();
    more = lane == 0 && next_row(k, sm.before, hi, w);
    more = __shfl_sync(FULL, (int)more, 0);
  } while (more);
}

// the partial rows of row of work w, joined by the CTA that comes last
template <int TYPE, int MODE> __device__ __forceinline__ void join_row(const Call &k, Smem<MODE> &sm, const Row<MODE> &w, long long total, int tid) {
  const int ctas = (int)min(total, (long long)gridDim.x), c0 = cta_of(w.unit0 + HEAD, total, ctas), c1 = cta_of(w.unit0 + HEAD + w.tiles - 1, total, ctas);
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    sm.last = atomicAdd(k.tile_counters + c0, 1) == c1 - c0;
    if (sm.last) k.tile_counters[c0] = 0;
  }
  __syncthreads();
  if (!sm.last) return;
  __threadfence();
  // the rows' weights of the pieces first (in Q's place and behind it), then their sums
  const int rows = w.rows(k), pieces = c1 - c0 + 1;
  float *const weights = reinterpret_cast<float *>(sm.q[0]);  // [row][piece]
  auto piece = [&](int i) { return k.tile_part + ((size_t)(c0 + i) * 2 + (i ? 0 : 1)) * 2 * ROWS * PSTRIDE; };
  const float v_scale = __ldg(k.c.v_scale + w.head);
  for (int c = tid; c < rows; c += THREADS) {
    float m = NOTHING, l = 0.f;
#pragma unroll 4
    for (int i = 0; i < pieces; ++i) m = fmaxf(m, __ldcg(piece(i) + c * PSTRIDE + D));
#pragma unroll 4
    for (int i = 0; i < pieces; ++i) {
      const float2 y = __ldcg(reinterpret_cast<const float2 *>(piece(i) + c * PSTRIDE + D));
      weights[c * pieces + i] = ex2(y.x - m);
      l += y.y * ex2(y.x - m);
    }
    const float f = l == 0.f ? 0.f : v_scale / l;
    for (int i = 0; i < pieces; ++i) weights[c * pieces + i] *= f;
    int query, head;
    split_column(k, 2 * ROWS * w.pair + c, query, head);
    if (k.a.lse) k.a.lse[(size_t)(w.r.start + query) * k.a.q_heads + w.head * k.group + head] = lse_of(m, l);
  }
  __syncthreads();
  constexpr int AHEAD = 8;  // float4 of a thread that are on their way at once
  for (int e0 = tid; e0 < rows * 32; e0 += AHEAD * THREADS) {
    float4 o[AHEAD] = {};
    for (int i = 0; i < pieces; ++i) {
      const float *const from = piece(i);
      float4 y[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int e = min(e0 + j * THREADS, rows * 32 - 1);
        y[j] = __ldcg(reinterpret_cast<const float4 *>(from + (e >> 5) * PSTRIDE) + (e & 31));
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const float f = weights[(min(e0 + j * THREADS, rows * 32 - 1) >> 5) * pieces + i];
        o[j] = make_float4(fmaf(y[j].x, f, o[j].x), fmaf(y[j].y, f, o[j].y), fmaf(y[j].z, f, o[j].z), fmaf(y[j].w, f, o[j].w));
      }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int e = e0 + j * THREADS;
      if (e >= rows * 32) break;
      int query, head;
      split_column(k, 2 * ROWS * w.pair + (e >> 5), query, head);
      reinterpret_cast<uint2 *>(out_row(k, w.r.start + query, w.head * k.group + head))[e & 31] = make_uint2(from_floats<TYPE>(o[j].x, o[j].y), from_floats<TYPE>(o[j].z, o[j].w));
    }
  }
  __syncthreads();
}

// NaN into what the CTA has stored of its rows, 16 channels at a time, where a token that the row sees has a NaN scale of V: by all threads, from the pages, only
// where a producer has met such a token. A row sees all tokens up to its limit, so that the first such token of a row of work's tiles decides.
template <int MODE> __device__ __forceinline__ void spoil_rows(const Call &k, Smem<MODE> &sm, long long hi, int tid) {
  Row<MODE> w = sm.begin;
  do {
    if (tid < 8) sm.nan_from[tid] = INT_MAX;
    __syncthreads();
    const int end = min(w.n1 * TOKENS, w.r.tokens);
    for (int t = w.n0 * TOKENS + tid; t < end; t += THREADS) {
      const int in_row = t + first_token<MODE>(w.r), column = in_row / k.c.page_size, at = in_row - column * k.c.page_size, page = __ldg(table_row<MODE>(k, w.r, w.b) + column);
      if ((unsigned)page >= (unsigned)k.c.pages) continue;
      const uint2 scales = __ldg(reinterpret_cast<const uint2 *>(k.c.units + (size_t)page * k.c.page_stride + (size_t)w.head * k.c.head_stride + (size_t)(at / BT) * BLOCK_BYTES +
                                                                 V_SCALES + at % BT * SCALE_BYTES));
      for (int j = 0; j < 8; ++j)
        if (nan_scales(j < 4 ? scales.x : scales.y) >> (8 * (j & 3) + 7) & 1) atomicMin(&sm.nan_from[j], t);
    }
    __syncthreads();
    const bool whole = w.n0 == 0 && w.n1 == w.tiles;
    for (int e = tid; e < w.rows(k) * 8; e += THREADS) {
      const int c = e >> 3, j = e & 7;
      int query, head;
      split_column(k, 2 * ROWS * w.pair + c, query, head);
      if (limit_of<MODE>(w.r, query) < sm.nan_from[j]) continue;
      if (MODE != SHARED && whole) {
        uint4 *const dst = reinterpret_cast<uint4 *>(out_row(k, w.r.start + query, w.head * k.group + head)) + 2 * j;
        dst[0] = dst[1] = make_uint4(0x7fff7fff, 0x7fff7fff, 0x7fff7fff, 0x7fff7fff);
      } else {
        float *slot = k.tile_part + (((size_t)blockIdx.x * 2 + (w.n0 ? 0 : 1)) * 2 * ROWS + c) * PSTRIDE;
        if constexpr (MODE == SHARED)
          if (whole) slot = sums_row(k, w.r.common, w.r.start + query, w.head * k.group + head);
        float4 *const dst = reinterpret_cast<float4 *>(slot) + 4 * j;
        const float x = __int_as_float(0x7fc00000);
        for (int i = 0; i < 4; ++i) __stcg(dst + i, make_float4(x, x, x, x));
      }
    }
    __syncthreads();
  } while (next_row(k, sm.before, hi, w));
}

template <int TYPE, int MODE> __global__ void __launch_bounds__(THREADS, 1) tile_kernel(const Call k) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<MODE> &sm = *reinterpret_cast<Smem<MODE> *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      fbla::mbar_init(&sm.q_ready[i], PRODUCER0 / 2);
      for (int h = 0; h < 2; ++h) {
        fbla::mbar_init(&sm.s_ready[i][h], 1);
        fbla::mbar_init(&sm.p_ready[i][h], PRODUCER0 / 2);
        fbla::mbar_init(&sm.o_done[i][h], 1);
      }
      fbla::mbar_init(&sm.k_full[i], PRODUCERS);
      fbla::mbar_init(&sm.v_full[i], PRODUCERS);
      fbla::mbar_init(&sm.k_empty[i], 2);
      fbla::mbar_init(&sm.v_empty[i], 2);
      fbla::mbar_init(&sm.drained[i], 1);
      fbla::mbar_init(&sm.places_full[i], 1);
      fbla::mbar_init(&sm.places_empty[i], PRODUCERS);
    }
    sm.abort = sm.v_nan = sm.others = 0;
    fbla::mbar_init_fence();
  }
  if (!k.wait_last) fbla::wait_previous_pass();
  fbla::allow_next_pass();

  const int items = items_of<MODE>(k);
  long long total = 0;
  int others = 0;
  for (int b0 = 0; b0 < items; b0 += THREADS) {
    const int b = b0 + tid;
    long long n = 0;
    if (b < items) {
      const Request<MODE> r = request<MODE>(k, b);
      n = tile_units<MODE>(k, r);
      if (MODE == SHARED) others += stream_units(k, r, k.narrow);
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
    if (b < items) sm.before[b] = base + sum - n;
    __syncthreads();
  }
  if (tid == 0) sm.before[items] = total;
  if (MODE == SHARED) {
    others = (int)__reduce_add_sync(FULL, (unsigned)others);
    if (others && lane == 0) atomicAdd(&sm.others, others);
    __syncthreads();
    if (warp == 0) {
      const int share = tile_share(k, total, sm.others, gridDim.x, lane);
      if (lane == 0) sm.share = share;
    }
  }
  __syncthreads();
  const int ctas = (int)min(total, (long long)(MODE == SHARED ? sm.share : gridDim.x));  // (each has a unit at least: a row's CTAs are consecutive)
  if ((int)blockIdx.x >= ctas) {
    if (k.wait_last) fbla::wait_previous_pass();
    return;
  }
  const long long lo = total * blockIdx.x / ctas, hi = total * (blockIdx.x + 1) / ctas;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(fbla::smem_u32(&sm.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 1) {
    const Row<MODE> w = first_row<MODE>(k, sm.before, lo, hi, lane);
    if (lane == 0) sm.begin = w;
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const bool tiles = sm.begin.n0 < sm.begin.n1;  // (a run of less than HEAD may have none)

  // 640 threads of 96 registers: 256 of 128 and 384 of 72. All warps meet before any takes registers back: a warpgroup's warps have to between two
  // such instructions, and registers that were given up are waited for by the softmax warps.
  if (warp < PRODUCER0) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    if (tiles) soften<TYPE, MODE>(k, sm, hi, warp, lane);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (!tiles) {}
    else if (warp < ISSUER0) produce(sm, warp - PRODUCER0, lane);
    else if (warp < FINDER && lane == 0) issue(k, sm, hi, warp - ISSUER0);
    else if (warp == FINDER) look_up(k, sm, hi, lane);
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp < PRODUCER0) asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
  if (sm.abort && warp >= ISSUER0 && warp < FINDER && lane == 0) {  // (nobody has waited for these products: they end, if they do, before what they use is given back)
    tc::mma_commit(&sm.drained[warp - ISSUER0]);
    fbla::mbar_wait_bounded(&sm.drained[warp - ISSUER0], 0, 1u << 20);
  }
  __syncwarp();
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sm.tmem) : "memory");
  if (!tiles) {
    if (k.wait_last) fbla::wait_previous_pass();
    return;
  }
  if (sm.v_nan) spoil_rows(k, sm, hi, tid);

  // the run's first and last rows of work, where they are cut (SHARED: merge_kernel joins them)
  if constexpr (MODE == SHARED) return;
  const Row<MODE> w = sm.begin;
  if (w.n0 > 0 || w.n1 < w.tiles) join_row<TYPE, MODE>(k, sm, w, total, tid);
  const Row<MODE> end = sm.row[0];
  if (end.unit0 > w.unit0 && end.n1 < end.tiles) join_row<TYPE, MODE>(k, sm, end, total, tid);
  if (k.wait_last) fbla::wait_previous_pass();
}

}  // namespace

template <int MODE> constexpr size_t tile_shared_bytes(size_t items) {
  using S = Smem<MODE>;
  return 1024 + offsetof(S, before) + (items + 1) * sizeof(long long);
}
template <int TYPE, int MODE> cudaError_t launch_tile(const Call &k, int sms, cudaStream_t stream) {
  static thread_local bool ready[64] = {false};
  const cudaError_t e = allow_shared(tile_kernel<TYPE, MODE>, ready);
  if (e != cudaSuccess) return e;
  const int pair = MODE == SHARED && sms > 1 ? PAIR : 1;
  return fbla::launch(true, pair, tile_kernel<TYPE, MODE>, dim3(sms / pair * pair), THREADS, tile_shared_bytes<MODE>((size_t)k.a.batch + (MODE == SHARED ? k.common.groups : 0)), stream, k);
}
#define PAGED_TILE(mode)                                                                                             \
  static_assert(tile_shared_bytes<mode>(PAGED_K_MAX_ATTENDED) <= 232448, "the operands and the largest batch fit"); \
  template cudaError_t launch_tile<MLOPS_PAGED_BF16, mode>(const Call &, int, cudaStream_t);                         \
  template cudaError_t launch_tile<MLOPS_PAGED_FP16, mode>(const Call &, int, cudaStream_t)

}  // namespace paged
