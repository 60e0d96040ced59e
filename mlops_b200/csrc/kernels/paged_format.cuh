// The paged cache's block format (include/mlops_paged.h) and its conversions: E2M1 codes, E4M3 scales of 16 channels.
#pragma once
#include "fbla_device.cuh"
#include "paged_kernels.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace paged {
using fbla::D;
using fbla::FULL;

constexpr int BT = MLOPS_PAGED_BLOCK;              // tokens of a block
constexpr int BLOCK_BYTES = MLOPS_PAGED_BLOCK_BYTES;
constexpr int CODE_BYTES = D / 2, SCALE_BYTES = D / 16;  // a token's, of one tensor
constexpr int V_CODES = BT * CODE_BYTES, K_SCALES = 2 * V_CODES, V_SCALES = K_SCALES + BT * SCALE_BYTES;
static_assert(V_SCALES + BT * SCALE_BYTES == BLOCK_BYTES, "the block's four arrays fill it");

// x / d for 0 <= x < 2^31 from inverse = 2^32 / d, rounded up (0 for d = 1): the product's high word is at most one too large
struct Divisor {
  int d;
  uint32_t inverse;
  __host__ explicit Divisor(int d) : d(d), inverse(d == 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d)) {}
  Divisor() = default;
  __device__ __forceinline__ int divide(int x) const {
    if (d == 1) return x;
    const int q = (int)__umulhi((uint32_t)x, inverse);
    return q - ((int64_t)q * d > x);
  }
};

__device__ __forceinline__ bool is_slot(const mlops_paged_cache &c, int slot) { return (unsigned)slot < (unsigned)(c.pages * c.page_size); }

// eight codes of a word as four pairs of FP16 (exact): pair i is channels 2 i, 2 i + 1
__device__ __forceinline__ void codes_to_half2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
// eight FP32 values as a word of codes, to the nearest, halfway to the even code, at most 6 in magnitude
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w) : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return w;
}
// two scale bytes (low, high) as a pair of FP16 (exact; 0x7f and 0xff are NaN)
__device__ __forceinline__ uint32_t scales_to_half2(uint32_t two_bytes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)two_bytes));
  return h;
}
// an FP32 value as a scale byte: to the nearest even, at most 448
__device__ __forceinline__ uint32_t scale_of(float x) {
  unsigned short h;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(0.f), "f"(x));
  return h & 0xffu;
}
__device__ __forceinline__ float2 half2_floats(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2 *>(&h)); }

// a word of two 16-bit values as floats and back, by type
template <int TYPE> __device__ __forceinline__ float2 to_floats(uint32_t w) {
  return TYPE == MLOPS_PAGED_BF16 ? make_float2(fbla::bf_lo(w), fbla::bf_hi(w)) : half2_floats(w);
}
template <int TYPE> __device__ __forceinline__ uint32_t from_floats(float lo, float hi) {
  if (TYPE == MLOPS_PAGED_BF16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&p);
  }
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}

}  // namespace paged
