// Attention over the paged cache for many queries per request (mlops_paged_attend): chunks of prompts and whole prompts, on tcgen05 tensor cores with
// TMEM accumulators.
//
// A row of work is (request, KV head, 256 rows); row c of a request and KV head is query c / group with query head c % group. Its units are HEAD and then the
// tiles of 128 tokens that its last row sees. All units form one list, of which every CTA has an equal contiguous run; a row of work that is cut is joined from
// partial rows (o, m', l) by the CTA that comes last, in the order of the tokens.
//
// Per tile of tokens and half X of the rows (128 each), with FP32 accumulators in tensor memory:
//   S_X[128 x 128] = Q_X K^T,   O_X[128 x 128] += P_X V
// K and V are code * scale, exact in FP16; Q is FP16 after a power of two per row (paged_attend.cuh); P = 2^(s - m') in FP16 takes S_X's place in tensor
// memory, rounded as in paged_stream.cu. m' moves only where a score would pass 2^15, then O and l are rescaled; l sums the unrounded P. Rows of at most
// 128 use both halves too: the even tiles of tokens go to X = 0, the odd ones to X = 1, with the same queries, and the halves are joined at the end.
//
// The exponentials of a tile take as long as its two products: 16 per cycle and SM, 2048 cycles for both X. Eight warps do those of X = 0 and then those of X = 1, so that
// the tensor cores work for one X while the other one's softmax runs. A tile then takes the softmax of one X (1800 cycles, of which the exponentials are 1024) and the way
// of the other from P to its next scores (2500: two products of 512 among the other X's, three hand-overs through barriers): 4300 cycles where the products alone are
// 2048. Two prompts of 8192 tokens, 32 / 8 heads: 1.40 ms = 785 TFLOP/s, 0.48 of the measured burst rate. Tried: a thread per row and both X's softmax at once
// (7600 cycles: both wait for the tensor cores together); a third of the exponentials as polynomials on the FMA units (1.07 times the time: packed FP32, maxima and
// conversions share their issue slots); operand warps that look up their blocks themselves (the registers spill, and every load is waited for at once). The kernel
// stores 56 bytes of registers per thread to local memory and loads 200.
//
// Warps 0-7 (two threads per row): softmax. Warps 8-15: operands, from packed pages to two stages each of K and V in shared
// memory, token rows of 128 bytes (64 channels) with 16-byte chunk c of row r at c ^ (r % 8): for S that is K-major, for O V's MN-major. Warps 16, 17: one thread
// each issues the products of its X. Warp 18 looks up where the tiles' blocks lie. Every wait is bounded: where one gives up, the rows become NaN.
#include "fbla_launch.h"
#include "fbla_tc.cuh"
#include "paged_attend.cuh"
#include <climits>

namespace paged {
namespace {

namespace tc = fbla::tc;

constexpr int ROWS = 128, TOKENS = 128;     // of a product
constexpr int SLAB = 128 * 128, TILE = 2 * SLAB;  // bytes of a slab (128 rows of 64 channels) and of an operand
constexpr int STAGES = 2, PRODUCER0 = 8, PRODUCERS = 8, ISSUER0 = 16, FINDER = 18, THREADS = 20 * 32;  // (four warps share a register count: 19 idles)
constexpr int HEAD = 4;  // units of a row of work beside its tiles: what loading Q, the first tile and storing O cost (17 000 cycles beside 4 300 per
                         // tile; us for two prompts of 8192 with 0, 2, 4, 6, 8: 2006, 1833, 1732, 1757, 1754 when they were 26 000 and 5 300)
constexpr int WINDOW = 16;  // tiles whose blocks are looked up at a time
constexpr int NO_TILE = -0x7fffffff;
constexpr float TOP = 15.f, REST = 9.f;
constexpr long long WAIT_CYCLES = 2000000000;
constexpr uint32_t IDESC_S = tc::IDESC_F16, IDESC_O = tc::IDESC_F16 | (1u << 16);  // V: MN-major

__device__ __forceinline__ int rows_of(const Call &k, const Request &r) { return r.n * k.group; }

// a row of work and its part in this CTA's run: tiles of tokens n0 .. n1 - 1 of `tiles`
struct Row {
  Request r;
  int b, head, pair, tiles, n0, n1;
  long long unit0;
  __device__ __forceinline__ int rows(const Call &k) const { return min(rows_of(k, r) - 2 * ROWS * pair, 2 * ROWS); }
  __device__ __forceinline__ bool halves(const Call &k) const { return rows(k) <= ROWS; }  // both X have the same rows
};
struct __align__(1024) Smem {
  uint8_t q[2][TILE];
  uint8_t k[STAGES][TILE], v[STAGES][TILE];
  const uint8_t *block[2 * WINDOW][8];  // [tile of the run % (2 WINDOW)][block]: where it lies; null: the table names no page, or the request has no such block
  int left[2 * WINDOW];         // tokens of the request from the tile's first on
  uint64_t places_full[2], places_empty[2];  // of WINDOW tiles each
  uint64_t drained[2];  // the issuing threads' products, after a wait that gave up
  uint64_t q_ready[2], k_full[STAGES], v_full[STAGES], k_empty[STAGES], v_empty[STAGES], s_ready[2], p_ready[2], o_done[2];
  uint8_t there[4][8];  // [tile of tokens % 4][block]: 1 where the table names a page
  float down[2][ROWS];      // the rows' factors
  float exchange[2][ROWS];  // between the two threads of a row
  int v_nan, nan_from[8];   // some V of the run has a NaN scale; [16 channels] of a row of work: the first token with one
  uint8_t over[2][2][4];    // [turn % 2][half of the tokens][quarter of the rows]: a score passes 2^15
  Row begin, row[8];    // the run's first row of work; the softmax warps' rows
  long long warp_sum[THREADS / 32];
  uint32_t tmem;
  int abort, last;
  long long before[];   // [batch + 1]: the requests' first units
};

// waits for the phase with the given parity, about a second at most; gives up at once where another thread has
__device__ __forceinline__ bool wait(Smem &sm, uint64_t *bar, uint32_t parity) {
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

// tiles of tokens that rows up to 256 (pair + 1) of a request see
__device__ __forceinline__ int tiles_of(const Call &k, const Request &r, int pair) {
  const int last = min(2 * ROWS * (pair + 1), rows_of(k, r)) - 1, seen = min(r.at + query_of(k, last) + 1, r.tokens);
  return max((seen + TOKENS - 1) / TOKENS, 1);  // (rows that see nothing have a tile all the same: their zeros are written like the others' sums)
}
__device__ __forceinline__ bool taken(const Call &k, const Request &r) { return r.tokens > 0 && r.n * k.group > k.wide; }

// the first row of work of the run [lo, hi), found by a warp
__device__ __forceinline__ Row first_row(const Call &k, const long long *before, long long lo, long long hi, int lane) {
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
  for (int pair0 = 0;; pair0 += 32) {  // 32 pairs at a time
    const int pair = pair0 + lane, units = 2 * ROWS * pair < rows_of(k, w.r) ? HEAD + tiles_of(k, w.r, pair) : 0;
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
__device__ __forceinline__ bool next_row(const Call &k, const long long *before, long long hi, Row &w) {
  const long long unit0 = w.unit0 + HEAD + w.tiles;
  if (unit0 + HEAD >= hi) return false;
  w.unit0 = unit0;
  if (2 * ROWS * ++w.pair >= rows_of(k, w.r)) {
    w.pair = 0;
    if (++w.head == k.c.kv_heads) {
      w.head = 0;
      do ++w.b; while (before[w.b + 1] <= unit0);
      w.r = request(k, w.b);
    }
  }
  w.tiles = tiles_of(k, w.r, w.pair);
  w.n0 = 0;
  w.n1 = (int)min((long long)w.tiles, hi - unit0 - HEAD);
  return true;
}
// whether half X has a part in tile n of w: w's second half in row order, or every second tile where the halves share the rows; a first half
// whose rows see less than the second one's leaves the last tile out
__device__ __forceinline__ int tiles_of_half(const Call &k, const Row &w, int x) {
  const int last = min(2 * ROWS * w.pair + ROWS * (x + 1), rows_of(k, w.r)) - 1, seen = min(w.r.at + query_of(k, last) + 1, w.r.tokens);
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
__device__ __forceinline__ void look_up(const Call &k, Smem &sm, long long hi, int lane) {
  const int per_page = k.c.page_size / BT, half = lane & 1;
  Row w = sm.begin;
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
      const int *const entries = k.a.table + (size_t)w.b * k.a.table_stride;
      const uint8_t *const head = k.c.units + (size_t)w.head * k.c.head_stride;
      const int number = 8 * n + 4 * half;
      int column = number / per_page, at = number - column * per_page;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t *block = nullptr;
        if ((number + j) * BT < w.r.tokens) {
          const int page = __ldg(entries + column);
          if ((unsigned)page < (unsigned)k.c.pages) block = head + (size_t)page * k.c.page_stride + (size_t)at * BLOCK_BYTES;
        }
        sm.block[tile % (2 * WINDOW)][4 * half + j] = block;
        if (++at == per_page) at = 0, ++column;
      }
    }
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.places_full[i & 1]);
  }
}

// Producer warp `warp` turns block `warp` of every tile into rows 16 warp .. of the operands, K of a tile before V of the tile before it, which is wanted
// later; a tensor's codes are loaded while its last tile's are waited for and used.
__device__ __forceinline__ void produce(Smem &sm, int warp, int lane) {
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
// The way from P to the next scores is what a tile takes: nothing else is waited for or released on it. A stage is free when both X have read it; where a tile
// is one X's alone, that one arrives for the other.
__device__ __forceinline__ void issue(const Call &k, Smem &sm, long long hi, int x) {  // by one thread
  const uint32_t s_at = sm.tmem + 128 * x, o_at = sm.tmem + 256 + 128 * x;
  uint32_t row_at = 0, mine = 0, items = 0;  // tiles of the run before the row, of this X; rows of work
  bool ok = true;
  Row w = sm.begin;
  do {
    const bool shared = w.halves(k);
    const int step = shared ? 2 : 1, end = shared ? w.n1 : min(w.n1, tiles_of_half(k, w, x)), both = shared ? 0 : tiles_of_half(k, w, 0);  // tiles below `both` are both X's
    const uint8_t *const q = sm.q[shared ? 0 : x];
    int n = w.n0 + (shared && (w.n0 & 1) != x);
    auto at = [&](int n) { return row_at + (n - w.n0); };
    auto scores = [&]() {
      const int stage = at(n) % STAGES;
      tc::tc_fence_after();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t offset = (i >> 2) * SLAB + (i & 3) * 32;
        tc::mma_f16(s_at, tc::smem_desc_at(q, offset), tc::smem_desc_at(sm.k[stage], offset), IDESC_S, i > 0);
      }
      tc::mma_commit(&sm.s_ready[x]);
      tc::mma_commit(&sm.k_empty[stage]);
      if (n >= both) tc::mbar_arrive(&sm.k_empty[stage]);
    };
    ok = ok && wait(sm, &sm.q_ready[x], items++ & 1);
    if (n < end) {
      ok = ok && wait(sm, &sm.k_full[at(n) % STAGES], at(n) / STAGES & 1);
      if (ok) scores();
    }
    for (bool first = true; n < end && ok; first = false) {
      const int stage = at(n) % STAGES, alone = n >= both;
      ok = wait(sm, &sm.v_full[stage], at(n) / STAGES & 1) && wait(sm, &sm.p_ready[x], mine & 1);
      if (!ok) break;
      tc::tc_fence_after();
#pragma unroll
      for (int i = 0; i < 8; ++i) tc::mma_f16_ts(o_at, s_at + 64 * (i >> 2) + 8 * (i & 3), v_desc(sm.v[stage], i * 2048), IDESC_O, !first || i > 0);
      tc::mma_commit(&sm.o_done[x]);
      n += step;
      if (n < end) {
        // (P is in S's place: its product has to be through before the next scores)
        ok = wait(sm, &sm.k_full[at(n) % STAGES], at(n) / STAGES & 1) && wait(sm, &sm.o_done[x], mine & 1);
        if (ok) scores();
        tc::mbar_arrive(&sm.v_empty[stage]);
      } else {
        tc::mma_commit(&sm.v_empty[stage]);
      }
      if (alone) tc::mbar_arrive(&sm.v_empty[stage]);
      ++mine;
    }
    row_at += w.n1 - w.n0;
  } while (next_row(k, sm.before, hi, w));
}

// ---- softmax --------------------------------------------------------------------------------------------------------------------
// Two threads have a row: warps w and w + 4 share 32 rows, warp w the first 64 tokens of a tile (and channels of O), w + 4 the others.
__device__ __forceinline__ void pair_meet(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); }

// Q's rows first .. first + 127 of the row of work as FP16 in `tile`, each times a power of two (q_factor) whose inverse goes to `down`; by eight warps, a
// half-warp per row
template <int TYPE> __device__ __forceinline__ void load_q(const Call &k, const Row &w, int first, uint8_t *tile, float *down, int warp, int lane) {
  const int c = lane & 15, rows = w.rows(k);
  uint4 raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int line = 16 * warp + 2 * i + (lane >> 4);
    int query, head;
    split_column(k, 2 * ROWS * w.pair + first + line, query, head);
    raw[i] = make_uint4(0, 0, 0, 0);
    if (first + line < rows)
      raw[i] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(k.a.q) + (int64_t)(w.r.start + query) * k.a.q_token_stride +
                                                     (int64_t)(w.head * k.group + head) * k.a.q_head_stride) + c);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int line = 16 * warp + 2 * i + (lane >> 4);
    const uint32_t word[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    float2 f[4];
    uint32_t top = 0, h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = to_floats<TYPE>(word[e]);
      top = max(top, max(__float_as_uint(f[e].x) & 0x7fffffffu, __float_as_uint(f[e].y) & 0x7fffffffu));
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(FULL, top, o));
    float inverse;
    const float up = q_factor(top, inverse);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = from_floats<MLOPS_PAGED_FP16>(f[e].x * up, f[e].y * up);
    *reinterpret_cast<uint4 *>(tile + (c >> 3) * SLAB + line * 128 + (((c & 7) ^ (line & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
    if (c == 0) down[line] = inverse;
  }
}

// 64 columns of the thread's lane from `at` on, to be waited for by arrived64, which every use of the values follows
#define PAGED_LD32(at, r) \
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];" \
               : "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]), "=r"((r)[6]), "=r"((r)[7]), "=r"((r)[8]), "=r"((r)[9]), "=r"((r)[10]), "=r"((r)[11]), \
                 "=r"((r)[12]), "=r"((r)[13]), "=r"((r)[14]), "=r"((r)[15]), "=r"((r)[16]), "=r"((r)[17]), "=r"((r)[18]), "=r"((r)[19]), "=r"((r)[20]), "=r"((r)[21]), "=r"((r)[22]), \
                 "=r"((r)[23]), "=r"((r)[24]), "=r"((r)[25]), "=r"((r)[26]), "=r"((r)[27]), "=r"((r)[28]), "=r"((r)[29]), "=r"((r)[30]), "=r"((r)[31]) : "r"(at) : "memory")
#define PAGED_HOLD32(r) \
  asm volatile("" : "+r"((r)[0]), "+r"((r)[1]), "+r"((r)[2]), "+r"((r)[3]), "+r"((r)[4]), "+r"((r)[5]), "+r"((r)[6]), "+r"((r)[7]), "+r"((r)[8]), "+r"((r)[9]), "+r"((r)[10]), "+r"((r)[11]), \
                    "+r"((r)[12]), "+r"((r)[13]), "+r"((r)[14]), "+r"((r)[15]), "+r"((r)[16]), "+r"((r)[17]), "+r"((r)[18]), "+r"((r)[19]), "+r"((r)[20]), "+r"((r)[21]), "+r"((r)[22]), \
                    "+r"((r)[23]), "+r"((r)[24]), "+r"((r)[25]), "+r"((r)[26]), "+r"((r)[27]), "+r"((r)[28]), "+r"((r)[29]), "+r"((r)[30]), "+r"((r)[31]))
struct Half {  // of a row of scores
  uint32_t r[2][32];
  __device__ __forceinline__ void load(uint32_t at) {
    PAGED_LD32(at, r[0]);
    PAGED_LD32(at + 32, r[1]);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    PAGED_HOLD32(r[0]);
    PAGED_HOLD32(r[1]);
  }
  __device__ __forceinline__ float score(int i) const { return __uint_as_float(r[i >> 5][i & 31]); }
  // scores of tokens above `last` and of blocks whose byte in `there` is 0 become -infinity
  __device__ __forceinline__ void mask(int last, uint32_t there) {
#pragma unroll
    for (int i = 0; i < 64; ++i)
      if (i > last || !(there >> (8 * (i >> 4)) & 1)) r[i >> 5][i & 31] = __float_as_uint(-FBLA_INF);
  }
  __device__ __forceinline__ float largest() const {
    float top[4] = {NOTHING, NOTHING, NOTHING, NOTHING};
#pragma unroll
    for (int i = 0; i < 32; ++i) top[i & 3] = fbla::max3(top[i & 3], score(2 * i), score(2 * i + 1));
    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  }
  // 2^(score mult - m) as 32 words of FP16 pairs in r[0]; their sum, and the largest exponent.
  __device__ __forceinline__ float exponentials(float mult, float m, float &high) {
    float2 sum[2] = {};
    float top[2] = {NOTHING, NOTHING};
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float2 e = __ffma2_rn(make_float2(score(2 * i), score(2 * i + 1)), make_float2(mult, mult), make_float2(-m, -m));
      top[i & 1] = fbla::max3(top[i & 1], e.x, e.y);
      const float2 f = make_float2(ex2(e.x), ex2(e.y));
      sum[i & 1] = __fadd2_rn(sum[i & 1], f);
      r[0][i] = from_floats<MLOPS_PAGED_FP16>(f.x, f.y);
    }
    high = fmaxf(top[0], top[1]);
    return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
  }
};

// a thread's part of a row of queries
struct Line {
  float m, l, mult;
  int limit;     // the last token that the row sees
  bool started;  // O holds sums
};

// one tile of half X: scores in tensor memory at s become P there
__device__ __forceinline__ bool take_tile(Smem &sm, Line &q, uint32_t s, uint32_t o, int first_token, int low, uint2 there, uint64_t *o_done, uint32_t o_parity,
                                          int line, int half, int turn) {
  const int quarter = line >> 5, in_half = q.limit - first_token - 64 * half;
  const bool mask = first_token + TOKENS - 1 > low || (there.x & there.y) != 0x01010101u;  // some row does not see all of the tile
  const uint32_t blocks = half ? there.y : there.x;
  Half x;
  bool ok = true;
  float high, sum = 0.f;
  bool over = true;
  x.load(s + 64 * half);
  if (mask) x.mask(in_half, blocks);
  if (q.started) {  // as if m' may stay where it is; the pair finds out together whether it may
    sum = x.exponentials(q.mult, q.m, high);
    over = __any_sync(FULL, high > TOP);
    if ((line & 31) == 0) sm.over[turn & 1][half][quarter] = over;
    pair_meet(quarter);
    over |= sm.over[turn & 1][half ^ 1][quarter];
  }
  if (over) {
    if (q.started) {
      x.load(s + 64 * half);
      if (mask) x.mask(in_half, blocks);
    }
    const float own = x.largest() * q.mult;  // (mult is positive)
    sm.exchange[half][line] = own;
    pair_meet(quarter);
    high = fmaxf(own, sm.exchange[half ^ 1][line]);
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
      for (int i = 0; i < 4; ++i) {
        uint32_t y[16];
        tc::tmem_ld16(o + 64 * half + 16 * i, y);
        tc::tmem_ld_wait(y);
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * keep);
        tc::tmem_st8(o + 64 * half + 16 * i, reinterpret_cast<const uint32_t(&)[8]>(y[0]));
        tc::tmem_st8(o + 64 * half + 16 * i + 8, reinterpret_cast<const uint32_t(&)[8]>(y[8]));
      }
      tc::tmem_st_wait();
    }
    sum = x.exponentials(q.mult, q.m, high);
    pair_meet(quarter);  // (the exchanged maxima have been read)
  }
  q.l += sum;
  tc::tmem_st32(s + 64 * half, x.r[0]);  // (in the place of the thread's own scores)
  return ok;
}

template <int TYPE> __device__ __forceinline__ void soften(const Call &k, Smem &sm, long long hi, int warp, int lane) {
  const int half = warp >> 2, line = 32 * (warp & 3) + lane;
  const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
  uint32_t mine[2] = {0, 0}, at = 0;
  bool ok = true;
  Row &w = sm.row[warp];  // (not in registers: they are all needed)
  if (lane == 0) w = sm.begin;
  __syncwarp();
  bool more;
  do {
    const bool shared = w.halves(k);
    asm volatile("bar.sync 5, 256;" ::: "memory");  // (the last row of work's outputs have left Q's place)
    load_q<TYPE>(k, w, 0, sm.q[0], sm.down[0], warp, lane);
    if (!shared) load_q<TYPE>(k, w, ROWS, sm.q[1], sm.down[1], warp, lane);
    fbla::fence_async_smem();
    asm volatile("bar.sync 5, 256;" ::: "memory");
    if (lane == 0) {
      tc::mbar_arrive(&sm.q_ready[0]);
      tc::mbar_arrive(&sm.q_ready[1]);
    }
    Line q[2];
    int low[2];
    bool warp_live[2];
    const float base = k.sl * __ldg(k.c.k_scale + w.head);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int c = line + (shared ? 0 : ROWS * x), col = 2 * ROWS * w.pair + c;  // of the row of work, of the request
      const bool live = c < w.rows(k);
      warp_live[x] = c - lane < w.rows(k);
      q[x] = Line{NOTHING, 0.f, fmaxf(base * sm.down[shared ? 0 : x][line], 1e-37f), live ? w.r.at + query_of(k, col) : -1, false};  // (mult is not 0: masked scores are -infinity)
      low[x] = w.r.at + query_of(k, col - lane);  // the smallest limit of the warp's rows
    }
    const int tiles0 = tiles_of_half(k, w, 0), tiles1 = tiles_of_half(k, w, 1), n0 = w.n0, n1 = w.n1;
#pragma unroll 1
    for (int n = n0; n < n1; ++n, ++at) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (!Part{shared, x ? tiles1 : tiles0}.has(n, x)) continue;
        ok = __all_sync(FULL, ok && wait(sm, &sm.s_ready[x], mine[x] & 1));
        tc::tc_fence_after();
        if (warp_live[x])  // (after a wait that gave up too: the warps of a pair meet)
          ok &= take_tile(sm, q[x], sm.tmem + 128 * x + lanes, sm.tmem + 256 + 128 * x + lanes, TOKENS * n, low[x], *reinterpret_cast<const uint2 *>(sm.there[at & 3]),
                         &sm.o_done[x], (mine[x] - 1) & 1, line, half, (int)(mine[0] + mine[1]));
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sm.p_ready[x]);
        q[x].started = true;
        ++mine[x];
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (q[x].started) ok = __all_sync(FULL, ok && wait(sm, &sm.o_done[x], (mine[x] - 1) & 1));
    tc::tc_fence_after();
    const bool whole = w.n0 == 0 && w.n1 == w.tiles;
    const float v_scale = __ldg(k.c.v_scale + w.head);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (!warp_live[x] || (x == 1 && shared)) continue;
      float m = q[x].m, l = q[x].l, keep = q[x].started ? 1.f : 0.f, other = 0.f;
      if (shared) {  // both halves' sums are of these rows
        m = fmaxf(q[0].m, q[1].m);
        l = q[0].l * ex2(q[0].m - m) + q[1].l * ex2(q[1].m - m);
        keep = q[0].started ? ex2(q[0].m - m) : 0.f;
        other = q[1].started ? ex2(q[1].m - m) : 0.f;
      }
      pair_meet(line >> 5);
      sm.exchange[half][line] = l;
      pair_meet(line >> 5);
      l = half ? sm.exchange[0][line] + l : l + sm.exchange[1][line];
      if (!ok) l = __int_as_float(0x7fc00000);  // (a wait that gave up: the rows are NaN)
      const int c = line + ROWS * x;
      const float f = l == 0.f ? 0.f : v_scale / l;
      float *const slot = k.tile_part + (((size_t)blockIdx.x * 2 + (w.n0 ? 0 : 1)) * 2 * ROWS + c) * PSTRIDE;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const int ch = 64 * half + 16 * i;
        uint32_t r[16], y[16];
        tc::tmem_ld16(sm.tmem + 256 + 128 * x + lanes + ch, r);
        tc::tmem_ld_wait(r);
        float o[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = keep == 0.f ? 0.f : __uint_as_float(r[e]) * keep;  // (a half without tiles has nothing in its accumulator)
        if (shared) {
          tc::tmem_ld16(sm.tmem + 256 + 128 + lanes + ch, y);
          tc::tmem_ld_wait(y);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = other == 0.f ? o[e] : fmaf(__uint_as_float(y[e]), other, o[e]);
        }
        if (whole) {  // through Q's place, from where whole rows are stored
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<uint4 *>(sm.q[x] + half * SLAB + line * 128 + (((2 * i + e) ^ (line & 7)) << 4)) =
                pack8<TYPE>(make_float4(o[8 * e] * f, o[8 * e + 1] * f, o[8 * e + 2] * f, o[8 * e + 3] * f),
                            make_float4(o[8 * e + 4] * f, o[8 * e + 5] * f, o[8 * e + 6] * f, o[8 * e + 7] * f));
        } else if (c < w.rows(k)) {
#pragma unroll
          for (int e = 0; e < 4; ++e) __stcg(reinterpret_cast<float4 *>(slot + ch) + e, make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]));
        }
      }
      if (half == 0 && c < w.rows(k)) {
        int query, head;
        split_column(k, 2 * ROWS * w.pair + c, query, head);
        if (!whole) __stcg(reinterpret_cast<float2 *>(slot + D), make_float2(m, l));
        else if (k.a.lse) k.a.lse[(size_t)(w.r.start + query) * k.a.q_heads + w.head * k.group + head] = lse_of(m, l);
      }
    }
    if (whole) {
      asm volatile("bar.sync 5, 256;" ::: "memory");
      const int rows = w.rows(k), ch = lane & 15;
#pragma unroll 4
      for (int c = 2 * warp + (lane >> 4); c < rows; c += 16) {
        const int at = c & (ROWS - 1);
        int query, head;
        split_column(k, 2 * ROWS * w.pair + c, query, head);
        reinterpret_cast<uint4 *>(out_row(k, w.r.start + query, w.head * k.group + head))[ch] =
            *reinterpret_cast<const uint4 *>(sm.q[c >> 7] + (ch >> 3) * SLAB + at * 128 + (((ch & 7) ^ (at & 7)) << 4));
      }
    }
    tc::tc_fence_before();
    __syncwarp();
    more = lane == 0 && next_row(k, sm.before, hi, w);
    more = __shfl_sync(FULL, (int)more, 0);
  } while (more);
}

// CTA of unit u when `ctas` CTAs share `total` units: CTA c has [total c / ctas, total (c + 1) / ctas)
__device__ __forceinline__ int cta_of(long long u, long long total, int ctas) { return (int)(((u + 1) * ctas - 1) / total); }

// the partial rows of row of work w, joined by the CTA that comes last
template <int TYPE> __device__ __forceinline__ void join_row(const Call &k, Smem &sm, const Row &w, long long total, int tid) {
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
__device__ __forceinline__ void spoil_rows(const Call &k, Smem &sm, long long hi, int tid) {
  Row w = sm.begin;
  do {
    if (tid < 8) sm.nan_from[tid] = INT_MAX;
    __syncthreads();
    const int end = min(w.n1 * TOKENS, w.r.tokens);
    for (int t = w.n0 * TOKENS + tid; t < end; t += THREADS) {
      const int column = t / k.c.page_size, at = t - column * k.c.page_size, page = __ldg(k.a.table + (size_t)w.b * k.a.table_stride + column);
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
      if (w.r.at + query < sm.nan_from[j]) continue;
      if (whole) {
        uint4 *const dst = reinterpret_cast<uint4 *>(out_row(k, w.r.start + query, w.head * k.group + head)) + 2 * j;
        dst[0] = dst[1] = make_uint4(0x7fff7fff, 0x7fff7fff, 0x7fff7fff, 0x7fff7fff);
      } else {
        float4 *const dst = reinterpret_cast<float4 *>(k.tile_part + (((size_t)blockIdx.x * 2 + (w.n0 ? 0 : 1)) * 2 * ROWS + c) * PSTRIDE) + 4 * j;
        const float x = __int_as_float(0x7fc00000);
        for (int i = 0; i < 4; ++i) __stcg(dst + i, make_float4(x, x, x, x));
      }
    }
    __syncthreads();
  } while (next_row(k, sm.before, hi, w));
}

template <int TYPE> __global__ void __launch_bounds__(THREADS, 1) tile_kernel(const Call k) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem &sm = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      fbla::mbar_init(&sm.q_ready[i], PRODUCER0);
      fbla::mbar_init(&sm.s_ready[i], 1);
      fbla::mbar_init(&sm.p_ready[i], PRODUCER0);
      fbla::mbar_init(&sm.o_done[i], 1);
      fbla::mbar_init(&sm.k_full[i], PRODUCERS);
      fbla::mbar_init(&sm.v_full[i], PRODUCERS);
      fbla::mbar_init(&sm.k_empty[i], 2);
      fbla::mbar_init(&sm.v_empty[i], 2);
      fbla::mbar_init(&sm.drained[i], 1);
      fbla::mbar_init(&sm.places_full[i], 1);
      fbla::mbar_init(&sm.places_empty[i], PRODUCERS);
    }
    sm.abort = sm.v_nan = 0;
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
        for (int p = 0; 2 * ROWS * p < rows_of(k, r); ++p) n += HEAD + tiles_of(k, r, p);
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
  __syncthreads();
  const int ctas = (int)min(total, (long long)gridDim.x);  // (each has a unit at least: a row's CTAs are consecutive)
  if ((int)blockIdx.x >= ctas) return;
  const long long lo = total * blockIdx.x / ctas, hi = total * (blockIdx.x + 1) / ctas;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(fbla::smem_u32(&sm.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 1) {
    const Row w = first_row(k, sm.before, lo, hi, lane);
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
    if (tiles) soften<TYPE>(k, sm, hi, warp, lane);
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
  if (!tiles) return;
  if (sm.v_nan) spoil_rows(k, sm, hi, tid);

  // the run's first and last rows of work, where they are cut
  const Row w = sm.begin;
  if (w.n0 > 0 || w.n1 < w.tiles) join_row<TYPE>(k, sm, w, total, tid);
  const Row end = sm.row[0];
  if (end.unit0 > w.unit0 && end.n1 < end.tiles) join_row<TYPE>(k, sm, end, total, tid);
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
