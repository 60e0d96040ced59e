// What the attention kernels of the paged cache share: the call, the requests' share of a kernel's work, joining of partial rows.
#pragma once
#include "paged_format.cuh"

namespace paged {
using fbla::ex2;
using fbla::lg2;

constexpr int PSTRIDE = 132;           // floats of a partial row: o[128], m, l, two unused
constexpr float NOTHING = -3e38f;      // the running maximum before the first score: finite, so that no difference of maxima is NaN
constexpr float LN2 = 0.6931471805599453f;

struct Call {
  mlops_paged_attend_args a;
  mlops_paged_cache c;
  float sl;        // softmax scale times log2(e)
  int group;       // query heads per KV head
  Divisor by_group;
  int wide;        // requests with more than so many columns (queries times group) are the tile kernel's
  float *stream_part, *tile_part;          // partial rows, see the kernels
  int *stream_counters, *tile_counters;    // one per CTA, zeros before and after every call
};

// a column's query and its query head among the KV head's: column / group, column % group
__device__ __forceinline__ int query_of(const Call &k, int column) { return k.by_group.divide(column); }
__device__ __forceinline__ void split_column(const Call &k, int column, int &query, int &head) {
  query = query_of(k, column);
  head = column - query * k.group;
}

// request b's queries and tokens, as far as q's rows and the table's width go. Rows that q does not have move no other: row i is the request's token
// lengths[b] - starts[b + 1] + i.
struct Request {
  int start, n, at, tokens;  // first row of q, queries, the first one's token (negative: before the request), tokens that a table row can name
};
__device__ __forceinline__ Request request(const Call &k, int b) {
  Request r;
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
  r.tokens = (int)min((long long)length, (long long)k.a.width * k.c.page_size);
  return r;
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

// zeros (and -infinity) for q's row `row`, by one warp
__device__ __forceinline__ void clear_row(const Call &k, int row, int lane) {
  for (int i = lane; i < k.a.q_heads * 16; i += 32) reinterpret_cast<uint4 *>(out_row(k, row, i >> 4))[i & 15] = make_uint4(0, 0, 0, 0);
  if (k.a.lse)
    for (int i = lane; i < k.a.q_heads; i += 32) k.a.lse[(size_t)row * k.a.q_heads + i] = -FBLA_INF;
}

template <int TYPE> __device__ __forceinline__ void store_joined(const Call &k, int row, int kv_head, int head, int x, const float4 &o, float m, float l) {
  const float f = l == 0.f ? 0.f : __ldg(k.c.v_scale + kv_head) / l;
  *reinterpret_cast<uint2 *>(out_row(k, row, head) + 4 * x) = make_uint2(from_floats<TYPE>(o.x * f, o.y * f), from_floats<TYPE>(o.z * f, o.w * f));
  if (k.a.lse && x == 0) k.a.lse[(size_t)row * k.a.q_heads + head] = lse_of(m, l);
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
template <int TYPE, int NT> cudaError_t launch_stream(const Call &k, int sms, cudaStream_t stream);
template <int TYPE> cudaError_t launch_tile(const Call &k, int sms, cudaStream_t stream);

}  // namespace paged
