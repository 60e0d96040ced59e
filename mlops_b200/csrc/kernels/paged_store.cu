// Quantise-on-write and read-back of the paged cache (mlops_paged_append, mlops_paged_read): a thread has 16 channels of a token and head, of K and of V, so
// that 64 bytes of a thread's are on their way at once and a slot is looked up once for both. Bound by memory: 65 536 tokens of 8 heads are read back in 56 us =
// 6.1 TB/s (0.94 of the copy rate), 32 768 appended in 37 to 39 us = 4.4 to 4.7 TB/s (0.68 to 0.71; the codes leave in pieces of 8 bytes). With a thread per tensor and two 16-byte
// accesses for 32 bytes 70 and 50 us.
#include "paged_store.cuh"

namespace paged {
namespace {

constexpr int THREADS = 256;
// CTAs per SM, which stay and take one row after the other: as many as are resident at once (us for 32 768 tokens of 8 heads, appended: 4 36.7, 6 39, 64 44; 65 536
// read: 4 69.7, 5 59, 6 56, 8 66, 64 59)
constexpr int APPEND_CTAS = 4, READ_CTAS = 6;

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
