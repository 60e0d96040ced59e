// What the kernels that write into the paged cache or read it back share: where a token's channels lie, 16 channels of a thread, the quantiser.
#pragma once
#include "fbla_launch.h"
#include "paged_format.cuh"

namespace paged {

constexpr int PER_ROW = D / 16;  // blocks of 16 channels of a (token, head)

struct Store {
  mlops_paged_cache c;
  const int *slots;
  Divisor by_heads, by_page;
  int rows;  // tokens * heads
};
// where the thread's channels of slot `slot` lie
__device__ __forceinline__ uint8_t *block_of(const Store &a, int slot, int head, int &at) {
  const int page = a.by_page.divide(slot), in_page = slot - page * a.c.page_size;
  at = in_page % BT;
  return a.c.units + (size_t)page * a.c.page_stride + (size_t)head * a.c.head_stride + (size_t)(in_page / BT) * BLOCK_BYTES;
}

struct Channels {  // sixteen, of 16 bits
  uint32_t w[8];
};
// WIDE: the 32 bytes lie on a boundary of 32
template <bool WIDE> __device__ __forceinline__ Channels load_channels(const uint16_t *p) {
  Channels x;
  if (WIDE) {
    asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(x.w[0]), "=r"(x.w[1]), "=r"(x.w[2]), "=r"(x.w[3]), "=r"(x.w[4]), "=r"(x.w[5]), "=r"(x.w[6]), "=r"(x.w[7]) : "l"(p));
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p)), b = __ldg(reinterpret_cast<const uint4 *>(p) + 1);
    x = Channels{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  }
  return x;
}
template <bool WIDE> __device__ __forceinline__ void store_channels(uint16_t *p, const Channels &x) {
  if (WIDE) {
    asm volatile("st.global.v8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(x.w[0]), "r"(x.w[1]), "r"(x.w[2]), "r"(x.w[3]), "r"(x.w[4]), "r"(x.w[5]), "r"(x.w[6]), "r"(x.w[7]), "l"(p) : "memory");
  } else {
    reinterpret_cast<uint4 *>(p)[0] = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
    reinterpret_cast<uint4 *>(p)[1] = make_uint4(x.w[4], x.w[5], x.w[6], x.w[7]);
  }
}

// fl(x / s) from r = fl(1 / s): one Newton step on the product is the rounded quotient wherever nothing under- or overflows (the residual of a
// product within an ulp of it is exact in an FMA: P. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990), and a
// code only asks on which side of a halfway case the quotient lies. (The step would take -0 to +0.)
__device__ __forceinline__ float quotient(float x, float s, float r) {
  const float q = __fmul_rn(x, r);
  return copysignf(fmaf(fmaf(-q, s, x), r, q), x);
}

// the codes of sixteen channels and their scale byte; inverse: 1 / the head's factor
template <int TYPE> __device__ __forceinline__ uint2 quantise(const Channels &x, float inverse, uint32_t &scale) {
  float y[16];
  uint32_t top = 0;  // of the bits of |y|: in their order NaN is above infinity, infinity above the numbers
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 f = to_floats<TYPE>(x.w[e]);
    y[2 * e] = __fmul_rn(f.x, inverse);
    y[2 * e + 1] = __fmul_rn(f.y, inverse);
    top = max(top, max(__float_as_uint(y[2 * e]) & 0x7fffffffu, __float_as_uint(y[2 * e + 1]) & 0x7fffffffu));
  }
  scale = scale_of(__fmul_rn(__uint_as_float(top), 0.1666666716337204f));
  if (top >= 0x7f800000u) {
    scale = 0x7f;
    return make_uint2(0, 0);
  }
  if (scale == 0) return make_uint2(0, 0);
  const float s = half2_floats(scales_to_half2(scale)).x, r = __frcp_rn(s);
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) lo[e] = quotient(y[e], s, r), hi[e] = quotient(y[8 + e], s, r);
  return make_uint2(codes_of(lo), codes_of(hi));
}
inline bool on_32(const void *p, int64_t by_token, int64_t by_head) { return reinterpret_cast<uintptr_t>(p) % 32 == 0 && by_token % 16 == 0 && by_head % 16 == 0; }

}  // namespace paged
