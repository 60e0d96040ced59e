// Quantise-on-write and read-back of the paged cache (mlops_paged_append, mlops_paged_read): a thread has 16 channels of a token and head, of K and of V, so
// that 64 bytes of a thread's are on their way at once and a slot is looked up once for both. Bound by memory: 65 536 tokens of 8 heads are read back in 56 us =
// 6.1 TB/s (0.94 of the copy rate), 32 768 appended in 37 to 39 us = 4.4 to 4.7 TB/s (0.68 to 0.71; the codes leave in pieces of 8 bytes). With a thread per tensor and two 16-byte
// accesses for 32 bytes 70 and 50 us.
#include "fbla_launch.h"
#include "paged_format.cuh"

namespace paged {
namespace {

constexpr int THREADS = 256;
constexpr int PER_ROW = D / 16;  // threads of a (token, head)
// CTAs per SM, which stay and take one row after the other: as many as are resident at once (us for 32 768 tokens of 8 heads, appended: 4 36.7, 6 39, 64 44; 65 536
// read: 4 69.7, 5 59, 6 56, 8 66, 64 59)
constexpr int APPEND_CTAS = 4, READ_CTAS = 6;

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
// the values of sixteen codes: code * scale is exact, one rounding by the factor, one to the type
template <int TYPE> __device__ __forceinline__ Channels values_of(uint2 codes, uint32_t scale, float factor) {
  Channels x;
  const float s = half2_floats(scales_to_half2(scale)).x;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t h[4];
    codes_to_half2(half ? codes.y : codes.x, h);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = half2_floats(h[e]);
      x.w[4 * half + e] = from_floats<TYPE>(__fmul_rn(f.x * s, factor), __fmul_rn(f.y * s, factor));
    }
  }
  return x;
}

template <int TYPE, bool WIDE>
__global__ void __launch_bounds__(THREADS, APPEND_CTAS) append_kernel(const Store a, const uint16_t *k, int64_t k_ts, int64_t k_hs, const uint16_t *v, int64_t v_ts, int64_t v_hs) {
  fbla::wait_previous_pass();
  fbla::allow_next_pass();
  const int j = threadIdx.x % PER_ROW;  // the channels' number among the row's eight
  for (int64_t row = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / PER_ROW; row < a.rows; row += (int64_t)gridDim.x * (THREADS / PER_ROW)) {
    const int token = a.by_heads.divide((int)row), head = (int)row - token * a.c.kv_heads, slot = __ldg(a.slots + token);
    const Channels x = load_channels<WIDE>(k + token * k_ts + head * k_hs + 16 * j), y = load_channels<WIDE>(v + token * v_ts + head * v_hs + 16 * j);
    if (!is_slot(a.c, slot)) continue;
    uint32_t k_scale, v_scale;
    const uint2 k_codes = quantise<TYPE>(x, __fdiv_rn(1.f, __ldg(a.c.k_scale + head)), k_scale), v_codes = quantise<TYPE>(y, __fdiv_rn(1.f, __ldg(a.c.v_scale + head)), v_scale);
    int at;
    uint8_t *const block = block_of(a, slot, head, at);
    *reinterpret_cast<uint2 *>(block + at * CODE_BYTES + 8 * j) = k_codes;
    *reinterpret_cast<uint2 *>(block + V_CODES + at * CODE_BYTES + 8 * j) = v_codes;
    block[K_SCALES + at * SCALE_BYTES + j] = (uint8_t)k_scale;
    block[V_SCALES + at * SCALE_BYTES + j] = (uint8_t)v_scale;
  }
}

template <int TYPE, bool WIDE> __global__ void __launch_bounds__(THREADS, READ_CTAS) read_kernel(const Store a, uint16_t *k, uint16_t *v) {
  fbla::wait_previous_pass();
  fbla::allow_next_pass();
  const int j = threadIdx.x % PER_ROW;
  for (int64_t row = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / PER_ROW; row < a.rows; row += (int64_t)gridDim.x * (THREADS / PER_ROW)) {
    const int token = a.by_heads.divide((int)row), head = (int)row - token * a.c.kv_heads, slot = __ldg(a.slots + token);
    Channels x{}, y{};
    if (is_slot(a.c, slot)) {
      int at;
      const uint8_t *const block = block_of(a, slot, head, at);
      const uint2 k_codes = *reinterpret_cast<const uint2 *>(block + at * CODE_BYTES + 8 * j), v_codes = *reinterpret_cast<const uint2 *>(block + V_CODES + at * CODE_BYTES + 8 * j);
      const uint32_t k_scale = block[K_SCALES + at * SCALE_BYTES + j], v_scale = block[V_SCALES + at * SCALE_BYTES + j];
      x = values_of<TYPE>(k_codes, k_scale, __ldg(a.c.k_scale + head));
      y = values_of<TYPE>(v_codes, v_scale, __ldg(a.c.v_scale + head));
    }
    store_channels<WIDE>(k + row * D + 16 * j, x);
    store_channels<WIDE>(v + row * D + 16 * j, y);
  }
}

Store store_of(const mlops_paged_cache *c, int tokens, const int *slots) {
  return Store{*c, slots, Divisor(c->kv_heads), Divisor(c->page_size), tokens * c->kv_heads};
}
dim3 grid_of(const Store &a, int most) {
  const int64_t ctas = ((int64_t)a.rows * PER_ROW + THREADS - 1) / THREADS;
  return dim3((unsigned)(ctas < most ? ctas : most));
}
bool on_32(const void *p, int64_t by_token, int64_t by_head) { return reinterpret_cast<uintptr_t>(p) % 32 == 0 && by_token % 16 == 0 && by_head % 16 == 0; }

}  // namespace
}  // namespace paged

extern "C" cudaError_t paged_k_append_launch(const mlops_paged_cache *c, int tokens, int type, const void *k, int64_t k_ts, int64_t k_hs, const void *v, int64_t v_ts,
                                             int64_t v_hs, const int *slots, int sms, cudaStream_t stream) {
  const paged::Store a = paged::store_of(c, tokens, slots);
  const bool wide = paged::on_32(k, k_ts, k_hs) && paged::on_32(v, v_ts, v_hs), bf16 = type == MLOPS_PAGED_BF16;
  const auto kernel = bf16 ? wide ? paged::append_kernel<MLOPS_PAGED_BF16, true> : paged::append_kernel<MLOPS_PAGED_BF16, false>
                           : wide ? paged::append_kernel<MLOPS_PAGED_FP16, true> : paged::append_kernel<MLOPS_PAGED_FP16, false>;
  return fbla::launch(true, 1, kernel, paged::grid_of(a, sms * paged::APPEND_CTAS), paged::THREADS, 0, stream, a, static_cast<const uint16_t *>(k), k_ts, k_hs, static_cast<const uint16_t *>(v), v_ts, v_hs);
}

extern "C" cudaError_t paged_k_read_launch(const mlops_paged_cache *c, int tokens, int type, const int *slots, void *k, void *v, int sms, cudaStream_t stream) {
  const paged::Store a = paged::store_of(c, tokens, slots);
  const bool wide = paged::on_32(k, 0, 0) && paged::on_32(v, 0, 0), bf16 = type == MLOPS_PAGED_BF16;
  const auto kernel = bf16 ? wide ? paged::read_kernel<MLOPS_PAGED_BF16, true> : paged::read_kernel<MLOPS_PAGED_BF16, false>
                           : wide ? paged::read_kernel<MLOPS_PAGED_FP16, true> : paged::read_kernel<MLOPS_PAGED_FP16, false>;
  return fbla::launch(true, 1, kernel, paged::grid_of(a, sms * paged::READ_CTAS), paged::THREADS, 0, stream, a, static_cast<uint16_t *>(k), static_cast<uint16_t *>(v));
}
