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
  int group;       // queries heads per KV head
  float *part;     // partial rows, see the kernels
  int *counters;   // zeros before and after every call
};

// request b's queries and tokens, as far as q's rows and the table's width go
struct Request {
  int start, n, length, tokens;  // first row of q, queries, lengths[b], tokens that a table row can name
};
__device__ __forceinline__ Request request(const Call &k, int b) {
  Request r;
  if (k.a.starts) {
    const int s = __ldg(k.a.starts + b), e = __ldg(k.a.starts + b + 1);
    r.start = min(max(s, 0), k.a.tokens);
    r.n = max(min(e, k.a.tokens) - r.start, 0);
  } else {
    r.start = b;
    r.n = 1;
  }
  r.length = max(__ldg(k.a.lengths + b), 0);
  r.tokens = (int)min((long long)r.length, (long long)k.a.width * k.c.page_size);
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

}  // namespace paged
