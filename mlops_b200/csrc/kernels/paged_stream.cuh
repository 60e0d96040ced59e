// Attention over the paged cache for few queries per request (mlops_paged_attend, mlops_paged_cross_attend, mlops_paged_attend_shared: paged_stream*.cu): the pages are streamed once, bound by their bytes.
//
// A row of work is (item, KV head, tile of 8 NT columns; an item is a request, or a group's common tokens); a column is one of the item's queries with one of the KV head's query heads. A row's
// unit is a pair of blocks, 32 tokens, 2304 contiguous bytes each. All rows' units form one list, which the grid's warps share out in equal contiguous runs,
// so that ragged lengths cost nothing; a warp brings its run's blocks through a ring of its own in shared memory with bulk copies.
//
// Per block, tokens on the M axis: S^T[16 tokens x 8] = K Q^T and O^T[128 channels x 8] += V^T P^T with mma.sync m16n8k16, FP16 operands, FP32 sums.
// K and V: code * scale is exact in FP16. Q: FP16 after a power of two per column (q_factor). P: 2^(s - m') with m' between 9 and 15 below the column's
// largest score so far, rounded to FP16: relative 2^-11 down to 2^-14, which is 2^-23 of the column's largest weight or less, and absolute 2^-25 (2^-34 of the largest)
// below, where weights are lost from 2^-34 of the largest on; 2^17 tokens of such weights are 2^-17 of the sum. m' moves, and O and l are rescaled, only where a score
// would pass 2^15. l sums the unrounded P.
//
// Channels and tokens are dealt to the fragments so that a lane's operands are whole words: for K lane (g, t) takes channels 32 t .. 32 t + 31 of its two
// tokens (the order of the K extent of a product is free as long as Q has the same); for V it takes channels 16 g .. 16 g + 15 of four tokens, and two
// tokens' nibbles of a channel are put beside each other before the conversion, so that a converted pair is a register of V^T.
//
// Rows that several warps share are joined in shared memory, those that several CTAs share by the CTA that comes last (a counter per CTA) or by merge_kernel (mlops_paged_attend_shared), always in
// the order of the tokens: the result does not depend on who that is.
//
// Bound by instructions beside the bytes: some 290 per block and tile of columns, of which a conversion and a scaling of every pair of codes are 128; no pipe is full
// (issue 0.60 per cycle and scheduler, the ALU pipe 57 % active, shared memory 25 %), warps wait for results of a fixed time and for one another. On the device (a graph of
// calls with a scratch of their own), 32 / 8 heads: 64 requests of 1K-64K tokens 174 us = 5.25 TB/s, 0.80 of the copy rate; 131 072 tokens 41 us, of which 28 are the
// loop, 6.5 what comes before (lengths, table, queries: five dependent reads) and some 7 the joining; 4096 tokens 12 us. Without the products and conversions the 64
// requests took 0.83 of the time, with units of one block instead of two (and rows shared out by 64-bit products) 1.18 times; twelve warps instead of sixteen: the same.
#pragma once
#include "fbla_launch.h"
#include "paged_attend.cuh"

namespace paged {
namespace {

// One tile of columns: sixteen warps of 128 registers (12 bytes of them spilled, 40 in cross attention). Two: eight of 240 or 241; with twelve of 168 the registers do not hold a block's words (1.04 times
// the time of drafted tokens of 16 requests). Three do not pay: requests of 24 columns take 0.85 of the time, but those of 16 columns 1.14 and of 32 1.15.
template <int NT> constexpr int WARPS = NT == 1 ? 16 : 8;
template <int NT> constexpr int STAGES = NT == 1 ? 2 : 3;
template <int NT> constexpr int THREADS = 32 * WARPS<NT>;
constexpr uint32_t DRAIN = 1u << 20;  // polls for a copy after a wait that gave up
constexpr float TOP = 15.f, REST = 9.f;  // log2 of the largest P, and of a column's largest when m' is set

// a row of work
template <int NT, int MODE> struct Row {
  Request<MODE> r;
  int b, head, tile, columns, units;
  int unit0;  // its first unit
};

template <int NT> struct Piece {  // a warp's partial rows of one row of work
  float o[8 * NT][PSTRIDE];        // (o[128], m', l)
};
template <int NT, int MODE> struct __align__(128) Smem {
  uint8_t ring[WARPS<NT>][STAGES<NT>][2][BLOCK_BYTES];
  Piece<NT> first[WARPS<NT>];      // of a run's first row; the last row's piece takes the ring's place when that is through
  uint64_t full[WARPS<NT>][STAGES<NT>];
  int tag[32];                     // pieces in the order of the tokens, two per warp: the first unit of the piece's row, -1: none
  Row<NT, MODE> row[32];           // the pieces' rows
  float2 total[8 * NT];            // (m', l) of a row that CTAs share
  int warp_sum[WARPS<NT>], share;
  long long tiles;  // SHARED: units of the tile kernel
  int last[2];
  int before[];                    // [items + 1]: the items' first units
};
template <int NT, int MODE> constexpr size_t shared_bytes(size_t items) {
  using S = Smem<NT, MODE>;
  return offsetof(S, before) + (items + 1) * sizeof(int);
}
template <int NT> constexpr bool fits = sizeof(Piece<NT>) <= STAGES<NT> * 2 * BLOCK_BYTES;

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
// token of the block in row r < 8 of the S^T fragment: two even and two odd tokens wherever four or two lanes read at once
__device__ __forceinline__ int token_of(int r) { return ((r >> 1) ^ (r & 1)) + 4 * (r & 1); }

// How the units are dealt: warp w has units [first(w), first(w + 1)), whole + 1 of them for w < more and `whole` for the others (one for each of the first
// warps where there are fewer units than warps).
struct Deal {
  int total, whole, more;
  __device__ __forceinline__ Deal(int total, int warps) : total(total) {
    whole = total < warps ? 1 : total / warps;
    more = total < warps ? 0 : total - whole * warps;
  }
  __device__ __forceinline__ int first(int w) const { return min(w * whole + min(w, more), total); }
  __device__ __forceinline__ int warp_of(int u) const { return u < more * (whole + 1) ? u / (whole + 1) : (u - more) / whole; }
};

template <int NT> __device__ __forceinline__ int tiles_of(const Call &k, const Plain &r) { return (r.n * k.group + 8 * NT - 1) / (8 * NT); }
// the item that unit u belongs to: before[b] <= u < before[b + 1]
__device__ __forceinline__ int item_at(const int *before, int items, int u) {
  int a = 0;
  for (int b = items; b - a > 1;) {
    const int mid = (a + b) >> 1;
    if (before[mid] <= u) a = mid; else b = mid;
  }
  return a;
}
// the row that unit u (of item b) belongs to
template <int NT, int MODE> __device__ __forceinline__ Row<NT, MODE> row_at(const Call &k, const int *before, int b, int u) {
  Row<NT, MODE> w;
  w.b = b;
  w.r = request<MODE>(k, b);
  w.units = units_of(w.r);
  const int tiles = tiles_of<NT>(k, w.r), row = (u - before[b]) / w.units;
  w.head = tiles == 1 ? row : row / tiles;
  w.tile = row - w.head * tiles;
  w.columns = min(w.r.n * k.group - w.tile * 8 * NT, 8 * NT);
  w.unit0 = before[b] + row * w.units;
  return w;
}

template <int TYPE, int NT> struct Columns {  // a row's queries, as B fragments
  uint32_t q[NT][16];
  float mult[NT][2];   // of the lane's two columns of the sums: scores in log2 units per unit of S
  int limit[NT][2];    // the last token that the column sees, -1: none
  int low;             // the smallest limit of the row's columns

  // q[j] takes the column's 32 channels as they are; `convert` follows
  template <int MODE> __device__ __forceinline__ void fetch(const Call &k, const Row<NT, MODE> &w, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int c = 8 * j + g;
      int query, head;
      split_column(k, w.tile * 8 * NT + c, query, head);
      const uint16_t *const src = static_cast<const uint16_t *>(k.a.q) + (int64_t)(w.r.start + query) * k.a.q_token_stride +
                                  (int64_t)(w.head * k.group + head) * k.a.q_head_stride + 32 * t;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint4 raw = c < w.columns ? __ldg(reinterpret_cast<const uint4 *>(src) + e) : make_uint4(0, 0, 0, 0);
        q[j][4 * e] = raw.x; q[j][4 * e + 1] = raw.y; q[j][4 * e + 2] = raw.z; q[j][4 * e + 3] = raw.w;
      }
    }
  }
  template <int MODE> __device__ __forceinline__ void convert(const Call &k, const Row<NT, MODE> &w, int lane) {
    const int t = lane & 3;
    const float base = k.sl * __ldg(k.c.k_scale + w.head);
    low = limit_of<MODE>(w.r, query_of(k, w.tile * 8 * NT));
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 x = to_floats<TYPE>(q[j][i]);
        top = max(top, max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu));
      }
      top = max(top, __shfl_xor_sync(FULL, top, 1));
      top = max(top, __shfl_xor_sync(FULL, top, 2));
      float down;
      const float up = q_factor(top, down);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 x = to_floats<TYPE>(q[j][i]);
        q[j][i] = from_floats<MLOPS_PAGED_FP16>(x.x * up, x.y * up);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mult[j][i] = fmaxf(base * __shfl_sync(FULL, down, (2 * t + i) * 4), 1e-37f);  // (not 0: masked scores are -infinity)
        const int cc = 8 * j + 2 * t + i;
        limit[j][i] = cc < w.columns ? limit_of<MODE>(w.r, query_of(k, w.tile * 8 * NT + cc)) : -1;
      }
    }
  }
};

// running sums of a row: O^T, m' and l of the lane's columns (l of its own tokens until `fold`)
template <int NT> struct Sums {
  float o[NT][8][4], m[NT][2], l[NT][2];
  __device__ __forceinline__ void clear(const int (&limit)[NT][2]) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][i][e] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[j][i] = limit[j][i] < 0 ? 0.f : NOTHING;  // (a column that sees nothing never waits for its first score)
        l[j][i] = 0.f;
      }
    }
  }
  __device__ __forceinline__ void fold() {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[j][i] += __shfl_xor_sync(FULL, l[j][i], x);
  }
};

// S^T of the unit's blocks, in score units of the product
template <int TYPE, int NT> __device__ __forceinline__ void scores(const uint8_t (&block)[2][BLOCK_BYTES], const Columns<TYPE, NT> &Q, float (&acc)[2][NT][4], int lane) {
  const int t = lane & 3, row = token_of(lane >> 2);
  uint32_t w[2][2][4], s[2][2];  // [block][token row, row + 8]
#pragma unroll
  for (int n = 0; n < 2; ++n) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint4 x = fbla::lds128(block[n] + (row + 8 * r) * CODE_BYTES + 16 * t);
      w[n][r][0] = x.x; w[n][r][1] = x.y; w[n][r][2] = x.z; w[n][r][3] = x.w;
      s[n][r] = scales_to_half2(*reinterpret_cast<const uint16_t *>(block[n] + K_SCALES + (row + 8 * r) * SCALE_BYTES + 2 * t));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      uint32_t h[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        codes_to_half2(w[n][r][i], h[r]);
        const uint32_t x = __byte_perm(s[n][r], 0, i < 2 ? 0x1010 : 0x3232);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[r][e] = times(h[r][e], x);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma(acc[n][j], h[0][0], h[1][0], h[0][1], h[1][1], Q.q[j][4 * i], Q.q[j][4 * i + 1]);
        mma(acc[n][j], h[0][2], h[1][2], h[0][3], h[1][3], Q.q[j][4 * i + 2], Q.q[j][4 * i + 3]);
      }
    }
}
// O^T += V^T P^T of a block whose first token is `token`; of its tokens only the first `tokens` count (EDGE: they may be fewer than 16, and columns may see fewer).
// A weight of 0 times NaN is NaN: at an edge NaN scales are taken as 0, and NaN goes into the sums of the columns that see such a token. The lane's sixteen
// channels have one scale per token, and a column sees all tokens up to its limit, so that the first such token decides.
template <int NT, bool EDGE>
__device__ __forceinline__ void values(const uint8_t *block, const uint32_t (&p)[NT][2], const int (&limit)[NT][2], Sums<NT> &s, int token, int tokens, int lane) {
  const int g = lane >> 2, t = lane & 3;
  // rows 2 t, 2 t + 1 (and + 8) of the K extent are tokens t, (t ^ 1) + 4 (and + 8)
  const int at[4] = {t, (t ^ 1) + 4, t + 8, (t ^ 1) + 12};
  uint2 v[4];
  uint32_t sv[4];
  int nan = BT;  // the block's first token with a NaN scale
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = fbla::lds64(block + V_CODES + at[i] * CODE_BYTES + 8 * g);
    sv[i] = block[V_SCALES + at[i] * SCALE_BYTES + g];
    if (EDGE && at[i] >= tokens) sv[i] = 0;  // (what is stored behind the last token may be anything, NaN too)
    if (EDGE && (sv[i] & 0x7f) == 0x7f) sv[i] = 0, nan = min(nan, at[i]);
  }
  if (EDGE && __any_sync(FULL, nan < BT)) {
    nan = min(nan, __shfl_xor_sync(FULL, nan, 1));
    nan = min(nan, __shfl_xor_sync(FULL, nan, 2));
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (nan < BT && token + nan <= limit[j][i])
#pragma unroll
          for (int n = 0; n < 8; ++n) s.o[j][n][i] = s.o[j][n][2 + i] = __int_as_float(0x7fc00000);
  }
  const uint32_t s01 = scales_to_half2(sv[0] | sv[1] << 8), s23 = scales_to_half2(sv[2] | sv[3] << 8);
#pragma unroll
  for (int half = 0; half < 2; ++half) {  // the even channels of the lane's sixteen, then the odd ones
    uint32_t a[4][4];  // word of channels 0-7 with tokens 0, 1; 8-15 with 0, 1; 0-7 with 2, 3; 8-15 with 2, 3
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = i & 1 ? v[i & 2].y : v[i & 2].x, y = i & 1 ? v[(i & 2) + 1].y : v[(i & 2) + 1].x;
      const uint32_t w = half ? ((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u) : (x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u);
      codes_to_half2(w, a[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[i][e] = times(a[i][e], i < 2 ? s01 : s23);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < NT; ++j) mma(s.o[j][2 * e + half], a[0][e], a[1][e], a[2][e], a[3][e], p[j][0], p[j][1]);
  }
}

// a unit: two blocks of 16 tokens, the first token of which is `token`, of a request of `tokens`; EDGE: some column does not see all of them, or a block is
// not `there` (bits 0, 1)
template <int TYPE, int NT, bool EDGE>
__device__ __forceinline__ void take_unit(const uint8_t (&block)[2][BLOCK_BYTES], const Columns<TYPE, NT> &Q, Sums<NT> &s, int token, int tokens, int there, int lane) {
  const int row = token_of(lane >> 2);
  float x[2][NT][4];
  scores<TYPE, NT>(block, Q, x, lane);
  // exponents, element e of the fragment: token row + 8 (e / 2) of the block, column 2 t + e % 2. A column that has no m' yet takes 0 for it.
  float high = NOTHING;
  bool open = false;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const float m[2] = {s.m[j][0] == NOTHING ? 0.f : s.m[j][0], s.m[j][1] == NOTHING ? 0.f : s.m[j][1]};
    open |= s.m[j][0] == NOTHING || s.m[j][1] == NOTHING;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (EDGE && (token + 16 * n + row + 8 * (e >> 1) > Q.limit[j][e & 1] || !(there >> n & 1))) x[n][j][e] = -FBLA_INF;
        x[n][j][e] = fmaf(x[n][j][e], Q.mult[j][e & 1], -m[e & 1]);
      }
      high = fbla::max3(fbla::max3(high, x[n][j][0], x[n][j][1]), x[n][j][2], x[n][j][3]);
    }
  }
  if (__any_sync(FULL, open || high > TOP)) {  // m' moves for the columns that need it
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = fmaxf(fmaxf(x[0][j][i], x[0][j][2 + i]), fmaxf(x[1][j][i], x[1][j][2 + i]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, d));
        const bool none = s.m[j][i] == NOTHING;
        if (top > (none ? -FBLA_INF : TOP)) {
          const float shift = top - REST, keep = none ? 0.f : ex2(-shift);
          s.m[j][i] = none ? shift : s.m[j][i] + shift;
          s.l[j][i] *= keep;
#pragma unroll
          for (int n = 0; n < 8; ++n) s.o[j][n][i] *= keep, s.o[j][n][2 + i] *= keep;
#pragma unroll
          for (int n = 0; n < 2; ++n) x[n][j][i] -= shift, x[n][j][2 + i] -= shift;
        }
      }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    uint32_t p[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][j][e] = ex2(x[n][j][e]);
      s.l[j][0] += x[n][j][0] + x[n][j][2];
      s.l[j][1] += x[n][j][1] + x[n][j][3];
      p[j][0] = transpose8(from_floats<MLOPS_PAGED_FP16>(x[n][j][0], x[n][j][1]));
      p[j][1] = transpose8(from_floats<MLOPS_PAGED_FP16>(x[n][j][2], x[n][j][3]));
    }
    values<NT, EDGE>(block[n], p, Q.limit, s, token + 16 * n, there >> n & 1 ? tokens - token - 16 * n : 0, lane);
  }
}

// a finished row to the output: by the warp that has all of it
template <int TYPE, int NT, int MODE> __device__ __forceinline__ void store_row(const Call &k, const Row<NT, MODE> &w, Sums<NT> &s, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const float vs = __ldg(k.c.v_scale + w.head);
  s.fold();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = 8 * j + 2 * t + i, col = w.tile * 8 * NT + c;
      if (c >= w.columns) continue;
      int query, head;
      split_column(k, col, query, head);
      const int row = w.r.start + query;
      head += w.head * k.group;
      if constexpr (MODE == SHARED) {
        float *const to = sums_row(k, w.r.common, row, head);
#pragma unroll
        for (int h = 0; h < 4; ++h)
          reinterpret_cast<float4 *>(to + 16 * g)[h] = make_float4(s.o[j][4 * (h & 1)][2 * (h >> 1) + i], s.o[j][4 * (h & 1) + 1][2 * (h >> 1) + i],
                                                                   s.o[j][4 * (h & 1) + 2][2 * (h >> 1) + i], s.o[j][4 * (h & 1) + 3][2 * (h >> 1) + i]);
        if (g == 0) *reinterpret_cast<float4 *>(to + D) = row_end(w.r, s.m[j][i], s.l[j][i]);
        continue;
      }
      const float f = s.l[j][i] == 0.f ? 0.f : vs / s.l[j][i];
      uint4 *const dst = reinterpret_cast<uint4 *>(out_row(k, row, head) + 16 * g);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        dst[h] = pack8<TYPE>(make_float4(s.o[j][0][2 * h + i] * f, s.o[j][1][2 * h + i] * f, s.o[j][2][2 * h + i] * f, s.o[j][3][2 * h + i] * f),
                             make_float4(s.o[j][4][2 * h + i] * f, s.o[j][5][2 * h + i] * f, s.o[j][6][2 * h + i] * f, s.o[j][7][2 * h + i] * f));
      if (k.a.lse && g == 0) k.a.lse[(size_t)row * k.a.q_heads + head] = lse_of(s.m[j][i], s.l[j][i]);
    }
}
template <int NT> __device__ __forceinline__ void store_piece(Piece<NT> &p, Sums<NT> &s, int lane) {
  const int g = lane >> 2, t = lane & 3;
  s.fold();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float *const dst = p.o[8 * j + 2 * t + i];
#pragma unroll
      for (int h = 0; h < 4; ++h)
        *reinterpret_cast<float4 *>(dst + 16 * g + 4 * h) = make_float4(s.o[j][4 * (h & 1)][2 * (h >> 1) + i], s.o[j][4 * (h & 1) + 1][2 * (h >> 1) + i],
                                                                        s.o[j][4 * (h & 1) + 2][2 * (h >> 1) + i], s.o[j][4 * (h & 1) + 3][2 * (h >> 1) + i]);
      if (g == 0) dst[D] = s.l[j][i] == 0.f ? NOTHING : s.m[j][i], dst[D + 1] = s.l[j][i];
    }
}

template <int TYPE, int NT, int MODE> __global__ void __launch_bounds__(THREADS<NT>, 1) stream_kernel(const Call k) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<NT, MODE> &sm = *reinterpret_cast<Smem<NT, MODE> *>(smem_raw);
  static_assert(fits<NT>, "a run's last piece lies in the ring");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (lane < STAGES<NT>) fbla::mbar_init(&sm.full[warp][lane], 1);
  fbla::mbar_init_fence();
  if (MODE != SHARED || !k.wait_last) fbla::wait_previous_pass();
  fbla::allow_next_pass();

  // the items' units
  const int items = items_of<MODE>(k);
  int total = 0;
  long long tiles = 0;
  for (int b0 = 0; b0 < items; b0 += THREADS<NT>) {
    const int b = b0 + tid;
    int n = 0;
    if (b < items) {
      const Request<MODE> r = request<MODE>(k, b);
      n = stream_units(k, r, 8 * NT);
      if (MODE == SHARED && k.wait_last) tiles += tile_units<MODE>(k, r);
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(FULL, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) sm.warp_sum[warp] = sum;
    __syncthreads();
    int base = total;
#pragma unroll
    for (int w = 0; w < WARPS<NT>; ++w) {
      if (w < warp) base += sm.warp_sum[w];
      total += sm.warp_sum[w];
    }
    if (b < items) sm.before[b] = base + sum - n;
    __syncthreads();
  }
  if (tid == 0) sm.before[items] = total;
  if (tid < 32) sm.tag[tid] = -1;
  int ctas = gridDim.x;  // that have units
  if (MODE == SHARED && k.wait_last && total) {
    if (tid == 0) sm.tiles = 0;
    __syncthreads();
    if (tiles) atomicAdd(reinterpret_cast<unsigned long long *>(&sm.tiles), (unsigned long long)tiles);
    __syncthreads();
    if (warp == 0) {
      const int share = tile_share(k, sm.tiles, total, gridDim.x, lane);
      if (lane == 0) sm.share = share;
    }
    __syncthreads();
    if (sm.share < ctas) ctas -= sm.share;  // (a device of two multiprocessors runs one kernel after the other)
    if (blockIdx.x >= ctas) return;  // (they begin when the tile kernel's CTAs are through; those with units wait for all of them)
  }
  __syncthreads();

  const int me = blockIdx.x * WARPS<NT> + warp, all = ctas * WARPS<NT>;
  const Deal deal(total, all);
  const int lo = deal.first(me), hi = deal.first(me + 1), count = hi - lo;
  if (count > 0) {
    // addresses of the run's blocks, 32 units at a time: lane i has those of unit 32 w + i of the run in window w, null where the table names no page or the
    // request has no such block
    struct Place {
      const uint8_t *block[2];
    };
    int b = item_at(sm.before, items, lo), lane_b = b;
    Row<NT, MODE> w = row_at<NT, MODE>(k, sm.before, b, lo);
    Columns<TYPE, NT> Q;
    Q.fetch(k, w, lane);
    const int per_page = k.c.page_size / BT;
    auto look_up = [&](int i) {
      Place p{{nullptr, nullptr}};
      const int u = lo + i;
      if (u >= hi) return p;
      while (sm.before[lane_b + 1] <= u) ++lane_b;
      const Row<NT, MODE> w = row_at<NT, MODE>(k, sm.before, lane_b, u);
      const int number = 2 * (u - w.unit0);
      const int in_row = number + first_token<MODE>(w.r) / BT;
      int column = in_row / per_page, at = in_row - column * per_page;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        if ((number + n) * BT < w.r.tokens) {
          const int page = __ldg(table_row<MODE>(k, w.r, lane_b) + column);
          if ((unsigned)page < (unsigned)k.c.pages)
            p.block[n] = k.c.units + (size_t)page * k.c.page_stride + (size_t)w.head * k.c.head_stride + (size_t)at * BLOCK_BYTES;
        }
        if (++at == per_page) at = 0, ++column;
      }
      return p;
    };
    Place now = look_up(lane), next;
    uint32_t there[2] = {__ballot_sync(FULL, now.block[0] != nullptr), __ballot_sync(FULL, now.block[1] != nullptr)};
    auto issue = [&](int i, const Place &from) {  // by the lane that has unit i's addresses
      uint64_t *const bar = &sm.full[warp][i % STAGES<NT>];
      fbla::fence_async_smem();
      fbla::mbar_expect_tx(bar, (from.block[0] ? BLOCK_BYTES : 0) + (from.block[1] ? BLOCK_BYTES : 0));
#pragma unroll
      for (int n = 0; n < 2; ++n)
        if (from.block[n]) fbla::bulk_g2s(sm.ring[warp][i % STAGES<NT>][n], from.block[n], BLOCK_BYTES, bar);
    };
    if (lane < STAGES<NT> && lane < count) issue(lane, now);

    bool first = true, alive = true;
    Sums<NT> s;
    for (int i = 0; i < count;) {
      if (i) {
        while (sm.before[b + 1] <= lo + i) ++b;
        w = row_at<NT, MODE>(k, sm.before, b, lo + i);
        Q.fetch(k, w, lane);
      }
      const int end = min(w.unit0 + w.units - lo, count);
      Q.convert(k, w, lane);
      if (i == 0 && count > 32) next = look_up(32 + lane);
      s.clear(Q.limit);
      int token = (lo + i - w.unit0) * UNIT;
#pragma unroll 1
      for (; i < end; ++i, token += UNIT) {
        const int stage = i % STAGES<NT>, here = (there[0] >> (i & 31) & 1) | (there[1] >> (i & 31) & 1) << 1;
        if (alive && !__all_sync(FULL, fbla::mbar_wait_bounded(&sm.full[warp][stage], (i / STAGES<NT>) & 1))) {
          alive = false;  // (for the rest of the run, which asks for nothing more; what it has asked for ends, if it does, before its places are used again)
          for (int n = i; n < min(i + STAGES<NT>, count); ++n) fbla::mbar_wait_bounded(&sm.full[warp][n % STAGES<NT>], (n / STAGES<NT>) & 1, DRAIN);
        }
        if (alive) {
          if (token + UNIT - 1 <= Q.low && here == 3) take_unit<TYPE, NT, false>(sm.ring[warp][stage], Q, s, token, w.r.tokens, 3, lane);
          else if (here) take_unit<TYPE, NT, true>(sm.ring[warp][stage], Q, s, token, w.r.tokens, here, lane);
          __syncwarp();
          const int ahead = i + STAGES<NT>;
          if (ahead < count && lane == (ahead & 31)) issue(ahead, (ahead >> 5) == (i >> 5) ? now : next);
        }
        if ((i & 31) == 31) {
          now = next;
          there[0] = __ballot_sync(FULL, now.block[0] != nullptr);
          there[1] = __ballot_sync(FULL, now.block[1] != nullptr);
          next = look_up(i + 33 + lane);
        }
      }
      if (!alive) {  // (a wait that gave up: the row is NaN)
#pragma unroll
        for (int j = 0; j < NT; ++j) s.l[j][0] = s.l[j][1] = __int_as_float(0x7fc00000);
      }
      const bool whole = w.unit0 >= lo && w.unit0 + w.units <= hi;
      if (whole) {
        store_row<TYPE, NT, MODE>(k, w, s, lane);
      } else {
        store_piece<NT>(first ? sm.first[warp] : *reinterpret_cast<Piece<NT> *>(sm.ring[warp][0][0]), s, lane);
        if (lane == 0) {
          sm.tag[2 * warp + (first ? 0 : 1)] = w.unit0;
          sm.row[2 * warp + (first ? 0 : 1)] = w;
        }
      }
      first = false;
    }
  }
  __syncthreads();

  // Rows that several of the CTA's warps share, or that go on in other CTAs, a warp per row and column. A row's pieces are its first one, p, and the first
  // pieces of the warps behind p's; lane i has the weight of piece i.
  const int cta_lo = deal.first(blockIdx.x * WARPS<NT>), cta_hi = deal.first((blockIdx.x + 1) * WARPS<NT>), my_tag = sm.tag[lane];
  const uint32_t same = __match_any_sync(FULL, my_tag);  // pieces of the row of piece `lane`
  const uint32_t leaders = __ballot_sync(FULL, my_tag >= 0 && __ffs(same) - 1 == lane);
  auto piece = [&](int p, int i) -> const Piece<NT> & { return i == 0 && (p & 1) ? *reinterpret_cast<const Piece<NT> *>(sm.ring[p >> 1][0][0]) : sm.first[(p >> 1) + i]; };
  auto is_cut = [&](const Row<NT, MODE> &w) { return w.unit0 < cta_lo || w.unit0 + w.units > cta_hi; };
  auto store = [&](const Row<NT, MODE> &w, int c, const float4 &o, float m, float l) {  // column c, a lane's four channels
    int query, head;
    split_column(k, w.tile * 8 * NT + c, query, head);
    store_joined<TYPE, MODE>(k, w.r, w.r.start + query, w.head, w.head * k.group + head, lane, o, m, l);
  };
  const int live = leaders >> lane & 1 ? sm.row[lane].columns : 0;  // columns of the row that piece `lane` leads
  int through = live;                                               // of all rows up to it
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(FULL, through, d);
    if (lane >= d) through += x;
  }
  const int columns = __shfl_sync(FULL, through, 31);
  for (int f = warp; f < columns; f += WARPS<NT>) {
    const int p = __popc(__ballot_sync(FULL, through <= f)), c = f - __shfl_sync(FULL, through - live, p);
    const int pieces = __popc(__shfl_sync(FULL, same, p));
    const Row<NT, MODE> &w = sm.row[p];
    float m, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (pieces <= 4) {  // (most rows lie in two warps: all that they are joined from is read at once, by every lane)
      float2 y[4];
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = i < pieces ? *reinterpret_cast<const float2 *>(piece(p, i).o[c] + D) : make_float2(NOTHING, 0.f);
        v[i] = i < pieces ? *reinterpret_cast<const float4 *>(piece(p, i).o[c] + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      m = fmaxf(fmaxf(y[0].x, y[1].x), fmaxf(y[2].x, y[3].x));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float g = ex2(y[i].x - m);
        l = fmaf(y[i].y, g, l);
        o = make_float4(fmaf(v[i].x, g, o.x), fmaf(v[i].y, g, o.y), fmaf(v[i].z, g, o.z), fmaf(v[i].w, g, o.w));
      }
    } else {
      const float2 y = lane < pieces ? *reinterpret_cast<const float2 *>(piece(p, lane).o[c] + D) : make_float2(NOTHING, 0.f);
      m = y.x;
#pragma unroll
      for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, d));
      const float weight = ex2(y.x - m);
      l = fbla::warp_sum(y.y * weight);
#pragma unroll 4
      for (int i = 0; i < pieces; ++i) {
        const float g = __shfl_sync(FULL, weight, i);
        const float4 v = *reinterpret_cast<const float4 *>(piece(p, i).o[c] + 4 * lane);
        o = make_float4(fmaf(v.x, g, o.x), fmaf(v.y, g, o.y), fmaf(v.z, g, o.z), fmaf(v.w, g, o.w));
      }
    }
    if (is_cut(w)) {
      float *const slot = k.stream_part + (((size_t)blockIdx.x * 2 + (w.unit0 < cta_lo ? 0 : 1)) * 8 * NT + c) * PSTRIDE;
      __stcg(reinterpret_cast<float4 *>(slot) + lane, o);
      if (lane == 0) __stcg(reinterpret_cast<float2 *>(slot + D), make_float2(m, l));
      if constexpr (MODE == SHARED)
        if (lane == 0 && w.unit0 >= cta_lo) {
          int query, head;
          split_column(k, w.tile * 8 * NT + c, query, head);
          const int slots = deal.warp_of(w.unit0 + w.units - 1) / WARPS<NT> - blockIdx.x + 1;
          *reinterpret_cast<float4 *>(sums_row(k, w.r.common, w.r.start + query, w.head * k.group + head) + D) = pieces_end(w.r, (blockIdx.x * 2 + 1) * 8 * NT + c, 8 * NT, slots);
        }
    } else {
      store(w, c, o, m, l);
    }
  }
  // rows that go on in other CTAs, this one's first and last at most: the CTA that comes last joins their slots (SHARED: merge_kernel)
  const int ends[2] = {__ffs(leaders) - 1, 31 - __clz(leaders)};
  if (MODE != SHARED && leaders && (is_cut(sm.row[ends[0]]) || is_cut(sm.row[ends[1]]))) {
    __threadfence();
    __syncthreads();
    if (tid < 2) {
      const Row<NT, MODE> &w = sm.row[ends[tid]];
      sm.last[tid] = -1;
      if (is_cut(w) && !(tid && ends[0] == ends[1])) {
        const int c0 = deal.warp_of(w.unit0) / WARPS<NT>, c1 = deal.warp_of(w.unit0 + w.units - 1) / WARPS<NT>;
        if (atomicAdd(k.stream_counters + c0, 1) == c1 - c0) {
          k.stream_counters[c0] = 0;
          sm.last[tid] = c0;
        }
      }
    }
    __syncthreads();
    for (int side = 0; side < 2; ++side) {
      const int c0 = sm.last[side];
      if (c0 < 0) continue;
      __threadfence();
      const Row<NT, MODE> &w = sm.row[ends[side]];
      const int slots = deal.warp_of(w.unit0 + w.units - 1) / WARPS<NT> - c0 + 1;
      // a warp per column and slice of the slots, every slices-th one; everything it reads is on its way before the first value is used. The slices' sums
      // meet in shared memory.
      const int slices = max(WARPS<NT> / w.columns, 1);
      float4(*const sums)[32] = reinterpret_cast<float4(*)[32]>(sm.ring);  // [column * slices + slice][lane]
      float *const weights = reinterpret_cast<float *>(sm.first[warp].o);  // of the slots
      for (int f = warp; f < w.columns * slices; f += WARPS<NT>) {
        const int c = f / slices, slice = f - c * slices;
        const float *const slot0 = k.stream_part + ((size_t)c0 * 2 * 8 * NT + c) * PSTRIDE;
        auto slot = [&](int i) { return slot0 + (i ? i * 2 : 1) * (8 * NT * PSTRIDE); };
        float2 y[4];
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = 32 * i + lane < slots ? __ldcg(reinterpret_cast<const float2 *>(slot(32 * i + lane) + D)) : make_float2(NOTHING, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = slice + i * slices < slots ? __ldcg(reinterpret_cast<const float4 *>(slot(slice + i * slices)) + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        float m = fmaxf(fmaxf(y[0].x, y[1].x), fmaxf(y[2].x, y[3].x)), l = 0.f;
        for (int i = 128 + lane; i < slots; i += 32) m = fmaxf(m, __ldcg(slot(i) + D));
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, d));
        __syncwarp();
        for (int i = lane; i < slots; i += 32) {
          const float2 z = i < 32 ? y[0] : i < 64 ? y[1] : i < 96 ? y[2] : i < 128 ? y[3] : __ldcg(reinterpret_cast<const float2 *>(slot(i) + D));
          weights[i] = ex2(z.x - m);
          l += z.y * weights[i];
        }
        __syncwarp();
        l = fbla::warp_sum(l);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = slice;;) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float g = i0 + i * slices < slots ? weights[i0 + i * slices] : 0.f;
            o = make_float4(fmaf(v[i].x, g, o.x), fmaf(v[i].y, g, o.y), fmaf(v[i].z, g, o.z), fmaf(v[i].w, g, o.w));
          }
          i0 += 8 * slices;
          if (i0 >= slots) break;
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = i0 + i * slices < slots ? __ldcg(reinterpret_cast<const float4 *>(slot(i0 + i * slices)) + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (slices == 1) {
          store(w, c, o, m, l);
        } else {
          sums[f][lane] = o;
          if (lane == 0 && slice == 0) sm.total[c] = make_float2(m, l);
        }
      }
      __syncthreads();
      if (slices > 1 && warp < w.columns) {
        float4 o = sums[warp * slices][lane];
        for (int i = 1; i < slices; ++i) {
          const float4 v = sums[warp * slices + i][lane];
          o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
        }
        store(w, warp, o, sm.total[warp].x, sm.total[warp].y);
      }
      __syncthreads();
    }
  }

  // rows of requests without tokens (a group's common rows are looked at only where it has some), rows of no request
  for (int b = (MODE == SHARED ? k.common.groups : 0) + me; b < items; b += all) {
    const Request<MODE> r = request<MODE>(k, b);
    if (r.tokens == 0)
      for (int i = 0; i < r.n; ++i) clear_row<MODE>(k, r, r.start + i, lane);
  }
  if (k.a.starts) {
    const int first = min(max(__ldg(k.a.starts), 0), k.a.tokens), end = min(max(__ldg(k.a.starts + k.a.batch), first), k.a.tokens);
    for (int i = me; i < first + k.a.tokens - end; i += all) clear_row<MODE>(k, Request<MODE>{}, i < first ? i : i - first + end, lane);
  }
  if (MODE == SHARED && k.wait_last) fbla::wait_previous_pass();
}

}  // namespace

template <int TYPE, int NT, int MODE> cudaError_t launch_stream(const Call &k, int sms, cudaStream_t stream) {
  static thread_local bool ready[64] = {false};
  const cudaError_t e = allow_shared(stream_kernel<TYPE, NT, MODE>, ready);
  if (e != cudaSuccess) return e;
  const size_t items = (size_t)k.a.batch + (MODE == SHARED ? k.common.groups : 0);
  const int pair = MODE == SHARED && k.wait_last && sms > 1 ? PAIR : 1;
  return fbla::launch(true, pair, stream_kernel<TYPE, NT, MODE>, dim3(sms / pair * pair), THREADS<NT>, shared_bytes<NT, MODE>(items), stream, k);
}
template <int NT, int MODE> constexpr bool holds = shared_bytes<NT, MODE>(PAGED_K_MAX_ATTENDED) <= 232448;
#define PAGED_STREAM(mode)                                                                                   \
  static_assert(holds<1, mode> && holds<2, mode>, "the rings and the largest batch fit");                    \
  template cudaError_t launch_stream<MLOPS_PAGED_BF16, 1, mode>(const Call &, int, cudaStream_t);            \
  template cudaError_t launch_stream<MLOPS_PAGED_FP16, 1, mode>(const Call &, int, cudaStream_t);            \
  template cudaError_t launch_stream<MLOPS_PAGED_BF16, 2, mode>(const Call &, int, cudaStream_t);            \
  template cudaError_t launch_stream<MLOPS_PAGED_FP16, 2, mode>(const Call &, int, cudaStream_t)

}  // namespace paged
