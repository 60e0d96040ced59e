// Quantise-on-write and read-back of the paged cache (mlops_paged_append, mlops_paged_read): a thread per 16 channels of one token, head and tensor.
#include "fbla_launch.h"
#include "paged_format.cuh"

namespace paged {
namespace {

constexpr int THREADS = 256;
constexpr int PER_ROW = 2 * D / 16;  // threads of a (token, head): 8 of K, 8 of V

// fl(x / s) from r = fl(1 / s): one Newton step on the product is the rounded quotient wherever nothing under- or overflows (the residual of a
// product within an ulp of it is exact in an FMA), and a code only asks on which side of a halfway case the quotient lies. (The step would take -0 to +0.)
__device__ __forceinline__ float quotient(float x, float s, float r) {
  const float q = __fmul_rn(x, r);
  return copysignf(fmaf(fmaf(-q, s, x), r, q), x);
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS) append_kernel(const mlops_paged_cache c, int tokens, const uint16_t *k, int64_t k_ts, int64_t k_hs, const uint16_t *v,
                                                         int64_t v_ts, int64_t v_hs, const int *slots) {
  fbla::wait_previous_pass();
  fbla::allow_next_pass();
  const int64_t total = (int64_t)tokens * c.kv_heads * PER_ROW;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * THREADS) {
    const int part = (int)(i % PER_ROW), j = part & 7;  // the channels' number among the row's eight
    const int64_t row = i / PER_ROW;
    const int token = (int)(row / c.kv_heads), head = (int)(row % c.kv_heads), slot = __ldg(slots + token);
    if (!is_slot(c, slot)) continue;
    const bool is_v = part >= 8;
    const uint16_t *const src = is_v ? v + token * v_ts + head * v_hs : k + token * k_ts + head * k_hs;
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>(src + 16 * j)), b = __ldg(reinterpret_cast<const uint4 *>(src + 16 * j) + 1);
    const float inverse = __fdiv_rn(1.f, __ldg((is_v ? c.v_scale : c.k_scale) + head));
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    float y[16];
    uint32_t top = 0;  // of the bits of |y|: in their order NaN is above infinity, infinity above the numbers
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 f = to_floats<TYPE>(w[e]);
      y[2 * e] = __fmul_rn(f.x, inverse);
      y[2 * e + 1] = __fmul_rn(f.y, inverse);
      top = max(top, max(__float_as_uint(y[2 * e]) & 0x7fffffffu, __float_as_uint(y[2 * e + 1]) & 0x7fffffffu));
    }
    uint32_t scale = scale_of(__fmul_rn(__uint_as_float(top), 0.1666666716337204f));
    uint2 codes = make_uint2(0, 0);
    if (top >= 0x7f800000u) {
      scale = 0x7f;
    } else if (scale) {
      const float s = half2_floats(scales_to_half2(scale)).x, r = __frcp_rn(s);
      float lo[8], hi[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[e] = quotient(y[e], s, r), hi[e] = quotient(y[8 + e], s, r);
      codes = make_uint2(codes_of(lo), codes_of(hi));
    }
    uint8_t *const block = block_of(c, slot, head);
    const int at = slot % BT;
    *reinterpret_cast<uint2 *>(block + (is_v ? V_CODES : 0) + at * CODE_BYTES + 8 * j) = codes;
    block[(is_v ? V_SCALES : K_SCALES) + at * SCALE_BYTES + j] = (uint8_t)scale;
  }
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS) read_kernel(const mlops_paged_cache c, int tokens, const int *slots, uint16_t *k, uint16_t *v) {
  fbla::wait_previous_pass();
  fbla::allow_next_pass();
  const int64_t total = (int64_t)tokens * c.kv_heads * PER_ROW;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * THREADS) {
    const int part = (int)(i % PER_ROW), j = part & 7;
    const int64_t row = i / PER_ROW;
    const int token = (int)(row / c.kv_heads), head = (int)(row % c.kv_heads), slot = __ldg(slots + token);
    const bool is_v = part >= 8;
    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (is_slot(c, slot)) {
      const uint8_t *const block = block_of(c, slot, head);
      const int at = slot % BT;
      const uint2 codes = *reinterpret_cast<const uint2 *>(block + (is_v ? V_CODES : 0) + at * CODE_BYTES + 8 * j);
      const float s = half2_floats(scales_to_half2(block[(is_v ? V_SCALES : K_SCALES) + at * SCALE_BYTES + j])).x;
      const float g = __ldg((is_v ? c.v_scale : c.k_scale) + head);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t h[4];
        codes_to_half2(half ? codes.y : codes.x, h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = half2_floats(h[e]);  // (code * scale is exact: one rounding by the factor, one to the type)
          w[4 * half + e] = from_floats<TYPE>(__fmul_rn(f.x * s, g), __fmul_rn(f.y * s, g));
        }
      }
    }
    uint4 *const dst = reinterpret_cast<uint4 *>((is_v ? v : k) + row * D + 16 * j);
    dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

dim3 grid_of(int tokens, int kv_heads) {
  const int64_t ctas = ((int64_t)tokens * kv_heads * PER_ROW + THREADS - 1) / THREADS;
  return dim3((unsigned)(ctas < 148 * 64 ? ctas : 148 * 64));
}

}  // namespace
}  // namespace paged

extern "C" cudaError_t paged_k_append_launch(const mlops_paged_cache *c, int tokens, int type, const void *k, int64_t k_ts, int64_t k_hs, const void *v, int64_t v_ts,
                                             int64_t v_hs, const int *slots, cudaStream_t stream) {
  return fbla::launch(true, 1, type == MLOPS_PAGED_BF16 ? paged::append_kernel<MLOPS_PAGED_BF16> : paged::append_kernel<MLOPS_PAGED_FP16>,
                      paged::grid_of(tokens, c->kv_heads), paged::THREADS, 0, stream, *c, tokens, static_cast<const uint16_t *>(k), k_ts, k_hs,
                      static_cast<const uint16_t *>(v), v_ts, v_hs, slots);
}

extern "C" cudaError_t paged_k_read_launch(const mlops_paged_cache *c, int tokens, int type, const int *slots, void *k, void *v, cudaStream_t stream) {
  return fbla::launch(true, 1, type == MLOPS_PAGED_BF16 ? paged::read_kernel<MLOPS_PAGED_BF16> : paged::read_kernel<MLOPS_PAGED_FP16>,
                      paged::grid_of(tokens, c->kv_heads), paged::THREADS, 0, stream, *c, tokens, slots, static_cast<uint16_t *>(k), static_cast<uint16_t *>(v));
}
