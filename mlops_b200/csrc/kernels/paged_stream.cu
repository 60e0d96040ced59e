// Attention over the paged cache for few queries per request (mlops_paged_attend): the pages are streamed once, bound by their bytes.
//
// A row of work is (request, KV head, tile of 8 NT columns); a column is one of the request's queries with one of the KV head's query heads. A row's
// unit is a block of 16 tokens, 2304 contiguous bytes. All rows' units form one list, which the grid's warps share out in equal contiguous runs, so that
// ragged lengths cost nothing; a warp brings its run's blocks through a ring of its own in shared memory with bulk copies.
//
// Per block, tokens on the M axis: S^T[16 tokens x 8] = K Q^T and O^T[128 channels x 8] += V^T P^T with mma.sync m16n8k16, FP16 operands, FP32 sums.
// K and V: code * scale is exact in FP16. Q: FP16 after a power of two per column (q_factor). P: 2^(s - m') with m' between 9 and 15 below the column's largest score so far, rounded to
// FP16 (relative 2^-11, the only rounding of the operands); m' moves, and O and l are rescaled, only where a score would pass 2^15. l sums the
// unrounded P. Weights below 2^-33 of the largest are lost, 2^17 of them are 2^-16 of the sum.
//
// Channels and tokens are dealt to the fragments so that a lane's operands are whole words: for K lane (g, t) takes channels 32 t .. 32 t + 31 of its two
// tokens (the order of the K extent of a product is free as long as Q has the same); for V it takes channels 16 g .. 16 g + 15 of four tokens, and two
// tokens' nibbles of a channel are put beside each other before the conversion, so that a converted pair is a register of V^T.
//
// Rows that several warps share are joined in shared memory, those that several CTAs share by the CTA that comes last (a counter per CTA), always in the
// order of the tokens: the result does not depend on who that is.
#include "fbla_launch.h"
#include "paged_attend.cuh"

namespace paged {
namespace {

template <int NT> constexpr int WARPS = NT == 1 ? 16 : 10;   // what the shared memory has room for beside the rings
template <int NT> constexpr int STAGES = NT == 1 ? 3 : 4;
template <int NT> constexpr int THREADS = 32 * WARPS<NT>;
constexpr int MIN_SHARE = 4;  // units of a warp, at least, where the work allows a choice
constexpr float TOP = 15.f, REST = 9.f;  // log2 of the largest P, and of a column's largest when m' is set

template <int NT> struct Piece {  // a warp's partial rows of one row of work
  float o[8 * NT][PSTRIDE];        // (o[128], m', l)
};
template <int NT> struct __align__(128) Smem {
  uint8_t ring[WARPS<NT>][STAGES<NT>][BLOCK_BYTES];
  Piece<NT> first[WARPS<NT>];          // of a run's first row; the last row's piece takes the ring's place when that is through
  uint64_t full[WARPS<NT>][STAGES<NT>];
  long long tag[2 * WARPS<NT>];        // pieces in the order of the tokens: the first unit of the piece's row, -1: none
  long long warp_sum[WARPS<NT>];
  int last;
  long long before[];              // [batch + 1]: the requests' first units
};
template <int NT> constexpr bool fits = sizeof(Piece<NT>) <= STAGES<NT> * BLOCK_BYTES;

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

// How the units are dealt: warp w has units [first(w), first(w + 1)).
struct Deal {
  long long total;
  int warps;
  __device__ __forceinline__ bool even() const { return total >= (long long)MIN_SHARE * warps; }
  __device__ __forceinline__ long long first(int w) const { return even() ? total * w / warps : min(total, (long long)MIN_SHARE * w); }
  __device__ __forceinline__ int warp_of(long long u) const { return even() ? (int)(((u + 1) * warps - 1) / total) : (int)(u / MIN_SHARE); }
};

// a row of work
template <int NT> struct Row {
  Request r;
  int b, head, tile, columns, blocks;
  long long unit0;  // its first unit
};

template <int NT> __device__ __forceinline__ int blocks_of(const Request &r) { return (r.tokens + BT - 1) / BT; }
template <int NT> __device__ __forceinline__ int tiles_of(const Call &k, const Request &r) { return (r.n * k.group + 8 * NT - 1) / (8 * NT); }
template <int NT> __device__ __forceinline__ long long units_of(const Call &k, const Request &r) {
  return r.n * k.group > k.wide ? 0 : (long long)k.c.kv_heads * tiles_of<NT>(k, r) * blocks_of<NT>(r);
}

// the row that unit u (of request b) belongs to
template <int NT> __device__ __forceinline__ Row<NT> row_at(const Call &k, const long long *before, int b, long long u) {
  Row<NT> w;
  w.b = b;
  w.r = request(k, b);
  w.blocks = blocks_of<NT>(w.r);
  const int tiles = tiles_of<NT>(k, w.r), row = (int)((u - before[b]) / w.blocks);
  w.head = row / tiles;
  w.tile = row % tiles;
  w.columns = min(w.r.n * k.group - w.tile * 8 * NT, 8 * NT);
  w.unit0 = before[b] + (long long)row * w.blocks;
  return w;
}

template <int TYPE, int NT> struct Columns {  // a row's queries, as B fragments
  uint32_t q[NT][16];
  float mult[NT][2];   // of the lane's two columns of the sums: scores in log2 units per unit of S
  int limit[NT][2];    // the last token that the column sees, -1: none
  int low;             // the smallest limit of the row's columns

  __device__ __forceinline__ void load(const Call &k, const Row<NT> &w, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const float base = k.sl * __ldg(k.c.k_scale + w.head);
    low = w.r.length - w.r.n + w.tile * 8 * NT / k.group;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int c = 8 * j + g, col = w.tile * 8 * NT + c;
      uint4 raw[4] = {};
      if (c < w.columns) {
        const uint16_t *const src = static_cast<const uint16_t *>(k.a.q) + (int64_t)(w.r.start + col / k.group) * k.a.q_token_stride +
                                    (int64_t)(w.head * k.group + col % k.group) * k.a.q_head_stride + 32 * t;
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[e] = __ldg(reinterpret_cast<const uint4 *>(src) + e);
      }
      float2 x[16];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t word[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[4 * e + i] = to_floats<TYPE>(word[i]);
          top = max(top, max(__float_as_uint(x[4 * e + i].x) & 0x7fffffffu, __float_as_uint(x[4 * e + i].y) & 0x7fffffffu));
        }
      }
      top = max(top, __shfl_xor_sync(FULL, top, 1));
      top = max(top, __shfl_xor_sync(FULL, top, 2));
      float down;
      const float up = q_factor(top, down);
#pragma unroll
      for (int i = 0; i < 16; ++i) q[j][i] = from_floats<MLOPS_PAGED_FP16>(x[i].x * up, x[i].y * up);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mult[j][i] = base * __shfl_sync(FULL, down, (2 * t + i) * 4);
        const int cc = 8 * j + 2 * t + i;
        limit[j][i] = cc < w.columns ? w.r.length - w.r.n + (w.tile * 8 * NT + cc) / k.group : -1;
      }
    }
  }
};

// running sums of a row: O^T, m' and l of the lane's columns (l of its own tokens until `fold`)
template <int NT> struct Sums {
  float o[NT][8][4], m[NT][2], l[NT][2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][i][e] = 0.f;
      m[j][0] = m[j][1] = NOTHING;
      l[j][0] = l[j][1] = 0.f;
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

// one block of 16 tokens, the first of which is `token`; EDGE: some column does not see all of it
template <int TYPE, int NT, bool EDGE>
__device__ __forceinline__ void take_block(const uint8_t *block, const Columns<TYPE, NT> &Q, Sums<NT> &s, int token, int tokens, int lane) {
  const int g = lane >> 2, t = lane & 3, row = token_of(g);
  float acc[NT][4], odd[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = odd[j][e] = 0.f;
  {
    const uint4 ka = fbla::lds128(block + row * CODE_BYTES + 16 * t), kb = fbla::lds128(block + (row + 8) * CODE_BYTES + 16 * t);
    const uint32_t sa = scales_to_half2(*reinterpret_cast<const uint16_t *>(block + K_SCALES + row * SCALE_BYTES + 2 * t));
    const uint32_t sb = scales_to_half2(*reinterpret_cast<const uint16_t *>(block + K_SCALES + (row + 8) * SCALE_BYTES + 2 * t));
    const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t ha[4], hb[4];
      codes_to_half2(wa[i], ha);
      codes_to_half2(wb[i], hb);
      const uint32_t xa = __byte_perm(sa, 0, i < 2 ? 0x1010 : 0x3232), xb = __byte_perm(sb, 0, i < 2 ? 0x1010 : 0x3232);
#pragma unroll
      for (int e = 0; e < 4; ++e) ha[e] = times(ha[e], xa), hb[e] = times(hb[e], xb);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma(acc[j], ha[0], hb[0], ha[1], hb[1], Q.q[j][4 * i], Q.q[j][4 * i + 1]);
        mma(odd[j], ha[2], hb[2], ha[3], hb[3], Q.q[j][4 * i + 2], Q.q[j][4 * i + 3]);
      }
    }
  }
  // scores in log2 units, element e of the fragment: token row + 8 (e / 2), column 2 t + e % 2
  float high = NOTHING;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = (acc[j][e] + odd[j][e]) * Q.mult[j][e & 1];
      if (EDGE && token + row + 8 * (e >> 1) > Q.limit[j][e & 1]) x = -FBLA_INF;
      acc[j][e] = x;
      high = fmaxf(high, x - s.m[j][e & 1]);
    }
  if (__any_sync(FULL, high > TOP)) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fmaxf(acc[j][i], acc[j][2 + i]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(FULL, x, d));
        if (x - s.m[j][i] > TOP) {
          const float m = x - REST, keep = ex2(s.m[j][i] - m);
          s.m[j][i] = m;
          s.l[j][i] *= keep;
#pragma unroll
          for (int n = 0; n < 8; ++n) s.o[j][n][i] *= keep, s.o[j][n][2 + i] *= keep;
        }
      }
  }
  uint32_t p[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[j][e] = ex2(acc[j][e] - s.m[j][e & 1]);
      s.l[j][e & 1] += acc[j][e];
    }
    p[j][0] = transpose8(from_floats<MLOPS_PAGED_FP16>(acc[j][0], acc[j][1]));
    p[j][1] = transpose8(from_floats<MLOPS_PAGED_FP16>(acc[j][2], acc[j][3]));
  }
  // V: rows 2 t, 2 t + 1 (and + 8) of the K extent are tokens t, (t ^ 1) + 4 (and + 8)
  const int at[4] = {t, (t ^ 1) + 4, t + 8, (t ^ 1) + 12};
  uint2 v[4];
  uint32_t sv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = fbla::lds64(block + V_CODES + at[i] * CODE_BYTES + 8 * g);
    sv[i] = block[V_SCALES + at[i] * SCALE_BYTES + g];
    if (EDGE && token + at[i] >= tokens) sv[i] = 0;  // (what is stored behind the last token may be anything, NaN too)
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

// a finished row to the output: by the warp that has all of it
template <int TYPE, int NT> __device__ __forceinline__ void store_row(const Call &k, const Row<NT> &w, Sums<NT> &s, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const float vs = __ldg(k.c.v_scale + w.head);
  s.fold();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = 8 * j + 2 * t + i, col = w.tile * 8 * NT + c;
      if (c >= w.columns) continue;
      const int row = w.r.start + col / k.group, head = w.head * k.group + col % k.group;
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
      if (g == 0) dst[D] = s.m[j][i], dst[D + 1] = s.l[j][i];
    }
}

template <int TYPE, int NT> __global__ void __launch_bounds__(THREADS<NT>, 1) stream_kernel(const Call k) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<NT> &sm = *reinterpret_cast<Smem<NT> *>(smem_raw);
  static_assert(fits<NT>, "a run's last piece lies in the ring");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (lane < STAGES<NT>) fbla::mbar_init(&sm.full[warp][lane], 1);
  fbla::mbar_init_fence();
  fbla::wait_previous_pass();
  fbla::allow_next_pass();

  // the requests' units
  long long total = 0;
  for (int b0 = 0; b0 < k.a.batch; b0 += THREADS<NT>) {
    const int b = b0 + tid;
    const long long n = b < k.a.batch ? units_of<NT>(k, request(k, b)) : 0;
    long long sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(FULL, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) sm.warp_sum[warp] = sum;
    __syncthreads();
    long long base = total;
#pragma unroll
    for (int w = 0; w < WARPS<NT>; ++w) {
      if (w < warp) base += sm.warp_sum[w];
      total += sm.warp_sum[w];
    }
    if (b < k.a.batch) sm.before[b] = base + sum - n;
    __syncthreads();
  }
  if (tid == 0) sm.before[k.a.batch] = total;
  if (lane < 2) sm.tag[2 * warp + lane] = -1;
  __syncthreads();

  const Deal deal{total, (int)gridDim.x * WARPS<NT>};
  const int me = blockIdx.x * WARPS<NT> + warp;
  const long long lo = deal.first(me), hi = deal.first(me + 1);
  const int count = (int)(hi - lo);
  if (count > 0) {
    // addresses of the run's blocks, 32 at a time: lane i has that of block 32 w + i of the run in window w, 0 where the table names no page
    const int per_page = k.c.page_size / BT;
    auto request_at = [&](long long u) {  // before[b] <= u < before[b + 1]
      int a = 0, b = k.a.batch;
      while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (sm.before[mid] <= u) a = mid; else b = mid;
      }
      return a;
    };
    int lane_b = request_at(min(lo + lane, hi - 1));
    auto address = [&](int i) -> const uint8_t * {
      const long long u = lo + i;
      if (u >= hi) return nullptr;
      while (sm.before[lane_b + 1] <= u) ++lane_b;
      const Row<NT> w = row_at<NT>(k, sm.before, lane_b, u);
      const int block = (int)(u - w.unit0), column = block / per_page, page = __ldg(k.a.table + (size_t)lane_b * k.a.table_stride + column);
      if ((unsigned)page >= (unsigned)k.c.pages) return nullptr;
      return k.c.units + (size_t)page * k.c.page_stride + (size_t)w.head * k.c.head_stride + (size_t)(block - column * per_page) * BLOCK_BYTES;
    };
    const uint8_t *now = address(lane), *next = address(32 + lane);
    uint32_t now_there = __ballot_sync(FULL, now != nullptr);
    auto issue = [&](int i, const uint8_t *from) {  // by the lane that has block i's address
      uint64_t *const bar = &sm.full[warp][i % STAGES<NT>];
      if (from) {
        fbla::fence_async_smem();
        fbla::mbar_expect_tx(bar, BLOCK_BYTES);
        fbla::bulk_g2s(sm.ring[warp][i % STAGES<NT>], from, BLOCK_BYTES, bar);
      } else {
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(fbla::smem_u32(bar)) : "memory");
      }
    };
    if (lane < STAGES<NT> && lane < count) issue(lane, now);

    int b = request_at(lo);
    bool first = true, alive = true;
    Columns<TYPE, NT> Q;
    Sums<NT> s;
    for (int i = 0; i < count;) {
      while (sm.before[b + 1] <= lo + i) ++b;
      const Row<NT> w = row_at<NT>(k, sm.before, b, lo + i);
      const int end = (int)min(w.unit0 + w.blocks - lo, (long long)count);
      Q.load(k, w, lane);
      s.clear();
      int token = (int)(lo + i - w.unit0) * BT;
      for (; i < end; ++i, token += BT) {
        const int stage = i % STAGES<NT>;
        if (alive) alive = fbla::mbar_wait_bounded(&sm.full[warp][stage], (i / STAGES<NT>) & 1);
        alive = __all_sync(FULL, alive);
        if (alive && (now_there >> (i & 31) & 1)) {
          if (token + BT - 1 <= Q.low) take_block<TYPE, NT, false>(sm.ring[warp][stage], Q, s, token, w.r.tokens, lane);
          else take_block<TYPE, NT, true>(sm.ring[warp][stage], Q, s, token, w.r.tokens, lane);
        }
        __syncwarp();
        const int ahead = i + STAGES<NT>;
        if (alive && ahead < count && lane == (ahead & 31)) issue(ahead, (ahead >> 5) == (i >> 5) ? now : next);
        if ((i & 31) == 31) {
          now = next;
          now_there = __ballot_sync(FULL, now != nullptr);
          next = address(i + 33 + lane);
        }
      }
      if (!alive) {  // (a wait that gave up: the row is NaN)
#pragma unroll
        for (int j = 0; j < NT; ++j) s.l[j][0] = s.l[j][1] = __int_as_float(0x7fc00000);
      }
      const bool whole = w.unit0 >= lo && w.unit0 + w.blocks <= hi;
      if (whole) {
        store_row<TYPE, NT>(k, w, s, lane);
      } else {
        store_piece<NT>(first ? sm.first[warp] : *reinterpret_cast<Piece<NT> *>(sm.ring[warp][0]), s, lane);
        if (lane == 0) sm.tag[2 * warp + (first ? 0 : 1)] = w.unit0;
      }
      first = false;
    }
  }
  __syncthreads();

  // rows that this CTA's warps share
  const long long cta_lo = deal.first(blockIdx.x * WARPS<NT>), cta_hi = deal.first((blockIdx.x + 1) * WARPS<NT>);
  auto piece = [&](int p) -> Piece<NT> & { return p & 1 ? *reinterpret_cast<Piece<NT> *>(sm.ring[p >> 1][0]) : sm.first[p >> 1]; };
  for (int p = 0; p < 2 * WARPS<NT>;) {
    const long long tag = sm.tag[p];
    if (tag < 0) { ++p; continue; }
    int list[WARPS<NT> + 1], pieces = 0;  // (a row's pieces in this CTA are one per warp)
    for (; p < 2 * WARPS<NT> && (sm.tag[p] == tag || sm.tag[p] < 0); ++p)
      if (sm.tag[p] == tag && pieces <= WARPS<NT>) list[pieces++] = p;
    int b = 0;
    for (int e = k.a.batch; e - b > 1;) {
      const int mid = (b + e) >> 1;
      if (sm.before[mid] <= tag) b = mid; else e = mid;
    }
    const Row<NT> w = row_at<NT>(k, sm.before, b, tag);
    const bool whole = tag >= cta_lo && tag + w.blocks <= cta_hi;
    float *const slot = k.stream_part + ((size_t)blockIdx.x * 2 + (tag < cta_lo ? 0 : 1)) * 8 * NT * PSTRIDE;
    for (int e = tid; e < w.columns * 32; e += THREADS<NT>) {
      const int c = e >> 5, x = e & 31, col = w.tile * 8 * NT + c;
      float m, l;
      const float4 o = join(pieces, [&](int i) { return (const float *)piece(list[i]).o[c]; }, x, m, l);
      if (whole) {
        store_joined<TYPE>(k, w.r.start + col / k.group, w.head, w.head * k.group + col % k.group, x, o, m, l);
      } else {
        __stcg(reinterpret_cast<float4 *>(slot + c * PSTRIDE) + x, o);
        if (x == 0) __stcg(reinterpret_cast<float2 *>(slot + c * PSTRIDE + D), make_float2(m, l));
      }
    }
    if (!whole) {  // the last of the row's CTAs joins their slots
      const int c0 = deal.warp_of(tag) / WARPS<NT>, c1 = deal.warp_of(tag + w.blocks - 1) / WARPS<NT>;
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        sm.last = atomicAdd(k.stream_counters + c0, 1) == c1 - c0;
        if (sm.last) k.stream_counters[c0] = 0;
      }
      __syncthreads();
      if (sm.last) {
        __threadfence();
        for (int e = tid; e < w.columns * 32; e += THREADS<NT>) {
          const int c = e >> 5, x = e & 31, col = w.tile * 8 * NT + c;
          float m, l;
          const float4 o = join(c1 - c0 + 1, [&](int i) { return k.stream_part + ((size_t)(c0 + i) * 2 + (i ? 0 : 1)) * 8 * NT * PSTRIDE + c * PSTRIDE; }, x, m, l);
          store_joined<TYPE>(k, w.r.start + col / k.group, w.head, w.head * k.group + col % k.group, x, o, m, l);
        }
      }
    }
  }

  // rows of requests without tokens, rows of no request
  for (int b = me; b < k.a.batch; b += deal.warps) {
    const Request r = request(k, b);
    if (r.tokens == 0)
      for (int i = 0; i < r.n; ++i) clear_row(k, r.start + i, lane);
  }
  if (k.a.starts)
    for (int row = max(__ldg(k.a.starts + k.a.batch), 0) + me; row < k.a.tokens; row += deal.warps) clear_row(k, row, lane);
}

}  // namespace

template <int TYPE, int NT> cudaError_t launch_stream(const Call &k, int sms, cudaStream_t stream) {
  static thread_local bool ready[64] = {false};
  const cudaError_t e = allow_shared(stream_kernel<TYPE, NT>, ready);
  if (e != cudaSuccess) return e;
  return fbla::launch(true, 1, stream_kernel<TYPE, NT>, dim3(sms), THREADS<NT>, offsetof(Smem<NT>, before) + ((size_t)k.a.batch + 1) * sizeof(long long), stream, k);
}
template cudaError_t launch_stream<MLOPS_PAGED_BF16, 1>(const Call &, int, cudaStream_t);
template cudaError_t launch_stream<MLOPS_PAGED_FP16, 1>(const Call &, int, cudaStream_t);
template cudaError_t launch_stream<MLOPS_PAGED_BF16, 2>(const Call &, int, cudaStream_t);
template cudaError_t launch_stream<MLOPS_PAGED_FP16, 2>(const Call &, int, cudaStream_t);

}  // namespace paged

