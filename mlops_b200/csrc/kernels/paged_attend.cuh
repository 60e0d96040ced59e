// What the attention kernels of the paged cache share: the call, the requests' share of a kernel's work, joining of partial rows.
#pragma once
#include "paged_format.cuh"

namespace paged {
using fbla::ex2;
using fbla::lg2;

constexpr int PSTRIDE = 132;           // floats of a partial row: o[128], m, l, two unused
constexpr float NOTHING = -3e38f;      // the running maximum before the first score: finite, so that no difference of maxima is NaN
constexpr float LN2 = 0.6931471805599453f;

// What a query sees: its request's tokens up to its own (mlops_paged_attend), all of its request's (mlops_paged_cross_attend), or as the first with the tokens that
// groups of requests have in common taken apart (mlops_paged_attend_shared)
enum { CAUSAL, WHOLE, SHARED };

struct Call {
  mlops_paged_attend_args a;
  mlops_paged_cache c;
  float sl;        // softmax scale times log2(e)
  int group;       // query heads per KV head
  Divisor by_group;
  int wide;        // requests with more than so many columns (queries times group) are the tile kernel's
  int narrow;      // columns of the stream's rows of work
  int room;        // tokens that a row of the table can name; at most 2^31 - 256, so that they can be rounded up to units and tiles
  float *stream_part, *tile_part;          // partial rows, see the kernels
  int *stream_counters, *tile_counters;    // one per CTA, zeros before and after every call
  // SHARED: the groups, and the sums of every row of q and head over common and own tokens (row_end, pieces_end); rows of both kernels' parts
  mlops_paged_common common;
  float *common_rows, *own_rows;
  int part_rows;
  bool wait_last;  // the kernel before in the stream is of the same call and leaves nothing that this one reads: waited for at the end
};

// a column's query and its query head among the KV head's: column / group, column % group
__device__ __forceinline__ int query_of(const Call &k, int column) { return k.by_group.divide(column); }
__device__ __forceinline__ void split_column(const Call &k, int column, int &query, int &head) {
  query = query_of(k, column);
  head = column - query * k.group;
}

// An item of a call is a request; SHARED: a group's common tokens (items 0 .. groups - 1), then the requests with their own.
template <int MODE> __device__ __forceinline__ int items_of(const Call &k) { return MODE == SHARED ? k.common.groups + k.a.batch : k.a.batch; }

// an item's queries and tokens, as far as q's rows and the table's width go. Rows that q does not have move no other: row i of request b is its token
// lengths[b] - starts[b + 1] + i.
struct Plain {
  int start, n, at, tokens;  // first row of q, queries, the first one's token (negative: before the item's), tokens that a table row can name
};
struct Apart {
  int start, n, at, tokens;
  int row, skip;  // row of the table; the item's first token in it
  bool common;    // a group's: all of them are seen by all
  __device__ __forceinline__ operator Plain() const { return Plain{start, n, at, tokens}; }
};
template <int MODE> struct RequestOf { using type = Plain; };
template <> struct RequestOf<SHARED> { using type = Apart; };
template <int MODE> using Request = typename RequestOf<MODE>::type;

__device__ __forceinline__ Plain plain_request(const Call &k, int b) {
  Plain r;
  int e = b + 1;
  if (k.a.starts) {
    const int s = __ldg(k.a.starts + b);
    e = __ldg(k.a.starts + b + 1);
    r.start = min(max(s, 0), k.a.tokens);
    r.n = max(min(e, k.a.tokens) - r.start, 0);
  } else {
    r.start = b;
    r.n = 1;
  }
  const int length = max(__ldg(k.a.lengths + b), 0);
  r.at = length - e + r.start;
  r.tokens = min(length, k.room);
  return r;
}
// group g's requests, and their common tokens: whole pages of the table, none for a single request, nor for requests of more than LONE columns on average, which fill rows of work by
// themselves: they take their tokens in one row instead of two that are joined (16 requests behind 6 000 common tokens, us by themselves and together: 132 columns each 136 and 107, 260 216 and
// 185, 384 235 and 247, 512 282 and 322, 1024 526 and 609). The average of mixed groups: a chunk of 2 048 queries of four heads
// and 15 decodes behind 16 384 tokens (516 columns) take 702 in mlops_paged_attend and 735 here, the chunk and 31 decodes (260) 780 and 707. Whether a request's first query sees them all, so that it takes part, is asked for each.
constexpr int LONE = 320;
struct Group {
  int first, end, tokens;
};
__device__ __forceinline__ Group group_at(const Call &k, int g) {
  Group x{0, k.a.batch, 0};
  if (k.common.starts) {
    x.first = min(max(__ldg(k.common.starts + g), 0), k.a.batch);
    x.end = min(max(__ldg(k.common.starts + g + 1), x.first), k.a.batch);
  }
  if (x.end - x.first > 1) {
    const int pages = max(__ldg(k.common.tokens + g), 0) / k.c.page_size;
    if (pages <= k.a.width) x.tokens = pages * k.c.page_size;  // (no request has more than its row of the table can name)
    if (k.a.starts && (long long)(__ldg(k.a.starts + x.end) - __ldg(k.a.starts + x.first)) * k.group > (long long)LONE * (x.end - x.first)) x.tokens = 0;
  }
  return x;
}
__device__ __forceinline__ bool takes_part(const Plain &r, int tokens) { return r.n > 0 && tokens > 0 && r.at >= tokens - 1; }

template <int MODE> __device__ __forceinline__ Request<MODE> request(const Call &k, int item) {
  Request<MODE> r;
  if constexpr (MODE != SHARED) {
    r = plain_request(k, item);
    if (MODE == WHOLE) r.at = max(__ldg(k.a.lengths + item), 0) - 1;
  } else if (item < k.common.groups) {
    const Group x = group_at(k, item);
    r.row = 0;
    r.start = r.n = r.skip = r.tokens = 0;
    r.at = -1;
    r.common = true;
    const int start = k.a.starts ? min(max(__ldg(k.a.starts + x.first), 0), k.a.tokens) : x.first, end = k.a.starts ? min(__ldg(k.a.starts + x.end), k.a.tokens) : x.end;
    Plain p = x.end > x.first ? plain_request(k, x.first) : Plain{0, 0, -1, 0};  // (its loads beside those of the group; mostly it is the one)
    for (int b = x.first; b < x.end && x.tokens > 0; ++b) {
      if (b > x.first) p = plain_request(k, b);
      if (!takes_part(p, x.tokens)) continue;
      // (the rows of requests that do not take part are computed with the others' and not used)
      r.row = b;
      r.tokens = x.tokens;
      r.at = x.tokens - 1;
      r.start = start;
      r.n = max(end - start, 0);
      break;
    }
  } else {
    const int b = item - k.common.groups;
    const Plain p = plain_request(k, b);  // (its loads beside those of the groups)
    r.start = p.start;
    r.n = p.n;
    r.at = p.at;
    r.tokens = p.tokens;
    r.row = b;
    r.skip = 0;
    r.common = false;
    int g = 0;
    if (k.common.starts)
      for (int e = k.common.groups; e - g > 1;) {
        const int mid = (g + e) >> 1;
        if (__ldg(k.common.starts + mid) <= b) g = mid; else e = mid;
      }
    const Group x = group_at(k, g);
    if (b >= x.first && b < x.end && takes_part(r, x.tokens)) {
      r.skip = x.tokens;
      r.at -= x.tokens;
      r.tokens -= x.tokens;
    }
  }
  return r;
}
// the last of the item's tokens that its query sees
template <int MODE> __device__ __forceinline__ int limit_of(const Request<MODE> &r, int query) {
  if constexpr (MODE == SHARED) return r.common ? r.at : r.at + query;
  else return MODE == WHOLE ? r.at : r.at + query;
}
template <int MODE> __device__ __forceinline__ const int *table_row(const Call &k, const Request<MODE> &r, int item) {
  if constexpr (MODE == SHARED) return k.a.table + (size_t)r.row * k.a.table_stride;
  else return k.a.table + (size_t)item * k.a.table_stride;
}
template <int MODE> __device__ __forceinline__ int first_token(const Request<MODE> &r) {
  if constexpr (MODE == SHARED) return r.skip;
  else return 0;
}

// a row of the output in 16 bits: eight channels from ch on
template <int TYPE> __device__ __forceinline__ uint4 pack8(const float4 &x, const float4 &y) {
  return make_uint4(from_floats<TYPE>(x.x, x.y), from_floats<TYPE>(x.z, x.w), from_floats<TYPE>(y.x, y.y), from_floats<TYPE>(y.z, y.w));
}
__device__ __forceinline__ uint16_t *out_row(const Call &k, int row, int head) {
  return static_cast<uint16_t *>(k.a.out) + (int64_t)row * k.a.out_token_stride + (int64_t)head * k.a.out_head_stride;
}
// the log-sum-exp of a row with running maximum m (log2 units) and sum l
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -FBLA_INF : (m + lg2(l)) * LN2; }

// SHARED: where the sums of q's row `row` and query head `head` go, by the item
__device__ __forceinline__ float *sums_row(const Call &k, bool common, int row, int head) {
  return (common ? k.common_rows : k.own_rows) + ((size_t)row * k.a.q_heads + head) * PSTRIDE;
}
// What stands behind a row's sums o[128], which merge_kernel joins: m (anything where l is 0), l, whether the common row counts too, 0. Where CTAs share the row: the first of its
// pieces as a row of stream_part, the rows of a CTA's slot, whether the common row counts too, how many pieces.
__device__ __forceinline__ float4 row_end(const Apart &r, float m, float l) { return make_float4(m, l, __int_as_float(r.skip > 0), __int_as_float(0)); }
__device__ __forceinline__ float4 pieces_end(const Apart &r, int first, int rows, int pieces) {
  return make_float4(__int_as_float(first), __int_as_float(rows), __int_as_float(r.skip > 0), __int_as_float(pieces));
}
// CTA c has two slots of `rows` rows: pieces of rows that other CTAs begin, and that it begins. Piece i of a row that CTA c begins, relative to piece 0
__device__ __forceinline__ int piece_row(int rows, int i) { return i ? (2 * i - 1) * rows : 0; }

// Units of work. The stream's: two blocks of a row of work of `narrow` columns. The tile kernel's: a tile of 128 tokens of a row of work of 256 rows, and HEAD for the row.
constexpr int UNIT = 2 * BT, TILE_ROWS = 256, TOKENS = 128;
constexpr int HEAD = 4;  // what a further row of work costs beside its tiles, as tiles (us with 3, 4, 5, 6, 7: two prompts of 8192 tokens 1 302, 1 240, 1 246, 1 256, 1 261; a mixed step of eight
                         // 312, 305, 308, 301, 309; drafted tokens of 24 requests behind two prompts 60, 56, 59, 62, 68)
__device__ __forceinline__ int units_of(const Plain &r) { return (r.tokens + UNIT - 1) / UNIT; }  // of each of the item's rows of work
__device__ __forceinline__ int stream_units(const Call &k, const Plain &r, int columns) {
  return r.n * k.group > k.wide ? 0 : k.c.kv_heads * ((r.n * k.group + columns - 1) / columns) * units_of(r);
}
__device__ __forceinline__ int rows_of(const Call &k, const Plain &r) { return r.n * k.group; }
// tiles of tokens that rows up to 256 (pair + 1) of an item see
template <int MODE> __device__ __forceinline__ int tiles_of(const Call &k, const Request<MODE> &r, int pair) {
  const int last = min(TILE_ROWS * (pair + 1), rows_of(k, r)) - 1, seen = min(limit_of<MODE>(r, query_of(k, last)) + 1, r.tokens);
  return max((seen + TOKENS - 1) / TOKENS, 1);  // (rows that see nothing have a tile all the same: their zeros are written like the others' sums)
}
template <int MODE> __device__ __forceinline__ long long tile_units(const Call &k, const Request<MODE> &r) {
  long long n = 0;
  if (r.tokens > 0 && r.n * k.group > k.wide) {
    const int pairs = (rows_of(k, r) + TILE_ROWS - 1) / TILE_ROWS;
    bool alike = MODE == WHOLE;  // all of the item's rows see the same tokens
    if constexpr (MODE == SHARED) alike = r.common;
    if (alike) n = (long long)pairs * (HEAD + tiles_of<MODE>(k, r, 0));
    else
      for (int p = 0; p < pairs; ++p) n += HEAD + tiles_of<MODE>(k, r, p);
    n *= k.c.kv_heads;
  }
  return n;
}

// SHARED: both kernels have work that does not wait for the other's, one bound by its products, the other by memory, on multiprocessors of their own: how many of `sms` are the tile
// kernel's, so that both end together. Cycles of a unit and beside the units, as measured: 4 100 and 45 000; 280 or 450 (tiles of 8 or 16 columns) and 32 000, with the start behind the
// tile kernel's CTAs that have nothing to do. In pairs: both kernels are launched in clusters of two, which lie on two neighbouring multiprocessors; one of each kernel there slow each other
// down, the tile kernel's to 0.78 and the stream's to 0.7 of their rate (256 requests behind 32 768 common tokens, us: 306, in pairs 230). By one warp; any number is right.
constexpr int PAIR = 2;
__device__ __forceinline__ int tile_share(const Call &k, long long tiles, int units, int sms, int lane) {
  if (tiles == 0 || units == 0 || sms < 2 * PAIR) return tiles ? sms : 0;
  uint32_t best = ~0u;
  for (int n = PAIR * (1 + lane); n < sms; n += 32 * PAIR) {
    const float a = 45e3f + 4100.f * ceilf(__fdividef((float)tiles, n)), b = 32e3f + (k.narrow == 8 ? 280.f : 450.f) * __fdividef((float)units, sms - n);
    best = min(best, (uint32_t)fminf(fmaxf(a, b) * 0.0625f, 2097151.f) << 11 | n);
  }
  return __reduce_min_sync(FULL, best) & 2047;
}

// zeros (and -infinity) for q's row `row`, by one warp; SHARED: no sums, for the item r or for no request (skip 0)
template <int MODE> __device__ __forceinline__ void clear_row(const Call &k, const Request<MODE> &r, int row, int lane) {
  if constexpr (MODE == SHARED) {
    for (int i = lane; i < k.a.q_heads; i += 32) *reinterpret_cast<float4 *>(sums_row(k, false, row, i) + D) = row_end(r, NOTHING, 0.f);
  } else {
    for (int i = lane; i < k.a.q_heads * 16; i += 32) reinterpret_cast<uint4 *>(out_row(k, row, i >> 4))[i & 15] = make_uint4(0, 0, 0, 0);
    if (k.a.lse)
      for (int i = lane; i < k.a.q_heads; i += 32) k.a.lse[(size_t)row * k.a.q_heads + i] = -FBLA_INF;
  }
}

template <int TYPE, int MODE>
__device__ __forceinline__ void store_joined(const Call &k, const Request<MODE> &r, int row, int kv_head, int head, int x, const float4 &o, float m, float l) {
  if constexpr (MODE == SHARED) {
    float *const to = sums_row(k, r.common, row, head);
    reinterpret_cast<float4 *>(to)[x] = l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : o;
    if (x == 0) *reinterpret_cast<float4 *>(to + D) = row_end(r, m, l);
  } else {
    const float f = l == 0.f ? 0.f : __ldg(k.c.v_scale + kv_head) / l;
    *reinterpret_cast<uint2 *>(out_row(k, row, head) + 4 * x) = make_uint2(from_floats<TYPE>(o.x * f, o.y * f), from_floats<TYPE>(o.z * f, o.w * f));
    if (k.a.lse && x == 0) k.a.lse[(size_t)row * k.a.q_heads + head] = lse_of(m, l);
  }
}

// the power of two that puts a query's largest element (its bits: `top`) into [2^8, 2^9), and its inverse; 1 where that is infinite or NaN. As FP16
// elements down to 2^-22 of the largest are exact, the others are rounded to 2^-33 of it.
__device__ __forceinline__ float q_factor(uint32_t top, float &inverse) {
  const uint32_t e = top >> 23, field = e == 255 ? 127 : min(262 - e, 253u);
  inverse = __uint_as_float((254 - field) << 23);
  return __uint_as_float(field << 23);
}

// a kernel's shared memory is above the default limit: asked for once per device and host thread
template <class K> cudaError_t allow_shared(K *kernel, bool (&ready)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && ready[dev])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
  if (e == cudaSuccess && dev < 64) ready[dev] = true;
  return e;
}
// 8 NT: columns of a row of work
template <int TYPE, int NT, int MODE> cudaError_t launch_stream(const Call &k, int sms, cudaStream_t stream);
template <int TYPE, int MODE> cudaError_t launch_tile(const Call &k, int sms, cudaStream_t stream);
// SHARED: the outputs from the sums over common and own tokens
template <int TYPE> cudaError_t launch_merge(const Call &k, int sms, cudaStream_t stream);

}  // namespace paged
