// Attention over the paged cache (mlops_paged_attend): a warp per query and head, one pass over the tokens with the running maximum and sum of
// the softmax. A lane has four channels.
#include "fbla_launch.h"
#include "paged_format.cuh"

namespace paged {
namespace {

constexpr int WARPS = 4;

// the lane's four codes of a token as floats (a word is two lanes')
__device__ __forceinline__ float4 four(const uint8_t *codes, int lane) {
  uint32_t h[4];
  codes_to_half2(reinterpret_cast<const uint32_t *>(codes)[lane / 2], h);
  const float2 a = half2_floats(lane & 1 ? h[2] : h[0]), b = half2_floats(lane & 1 ? h[3] : h[1]);
  return make_float4(a.x, a.y, b.x, b.y);
}

template <int TYPE> __global__ void __launch_bounds__(32 * WARPS) attend_kernel(const mlops_paged_attend_args a, const mlops_paged_cache c, float sl) {
  fbla::wait_previous_pass();
  fbla::allow_next_pass();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (row >= (int64_t)a.tokens * a.q_heads) return;
  const int t = (int)(row / a.q_heads), hq = (int)(row % a.q_heads), head = hq / (a.q_heads / c.kv_heads);
  int b = t, last = -1;  // the request and the last token that is seen
  bool mine = true;
  if (a.starts) {
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(a.starts + mid) <= t) lo = mid; else hi = mid;
    }
    b = lo;
    mine = __ldg(a.starts + b) <= t && t < __ldg(a.starts + b + 1);
  }
  if (mine) {
    const int n = a.starts ? __ldg(a.starts + b + 1) - __ldg(a.starts + b) : 1, i = a.starts ? t - __ldg(a.starts + b) : 0;
    last = __ldg(a.lengths + b) - n + i;
    last = (int)min((long long)last, (long long)a.width * c.page_size - 1);
  }
  const uint16_t *const q = static_cast<const uint16_t *>(a.q) + t * a.q_token_stride + hq * a.q_head_stride;
  const uint2 w = __ldg(reinterpret_cast<const uint2 *>(q) + lane);
  const float2 q0 = to_floats<TYPE>(w.x), q1 = to_floats<TYPE>(w.y);
  const float mult = sl * __ldg(c.k_scale + head);
  float m = -FBLA_INF, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = 0; p <= last; ++p) {
    const int page = __ldg(a.table + (size_t)b * a.table_stride + p / c.page_size);
    if ((unsigned)page >= (unsigned)c.pages) continue;
    const int slot = page * c.page_size + p % c.page_size, at = slot % BT;
    const uint8_t *const block = block_of(c, slot, head);
    const float ks = half2_floats(scales_to_half2(block[K_SCALES + at * SCALE_BYTES + lane / 4])).x, vs = half2_floats(scales_to_half2(block[V_SCALES + at * SCALE_BYTES + lane / 4])).x;
    const float4 k = four(block + at * CODE_BYTES, lane), v = four(block + V_CODES + at * CODE_BYTES, lane);
    const float s = fbla::warp_sum(ks * (k.x * q0.x + k.y * q0.y + k.z * q1.x + k.w * q1.y)) * mult;
    const float top = fmaxf(m, s), keep = fbla::ex2(m - top), e = fbla::ex2(s - top);
    l = l * keep + e;
    const float p_v = e * vs;
    o = make_float4(o.x * keep + p_v * v.x, o.y * keep + p_v * v.y, o.z * keep + p_v * v.z, o.w * keep + p_v * v.w);
    m = s != s ? s : top;
  }
  const float inverse = l == 0.f ? 0.f : __ldg(c.v_scale + head) / l;
  uint16_t *const out = static_cast<uint16_t *>(a.out) + t * a.out_token_stride + hq * a.out_head_stride;
  reinterpret_cast<uint2 *>(out)[lane] = make_uint2(from_floats<TYPE>(o.x * inverse, o.y * inverse), from_floats<TYPE>(o.z * inverse, o.w * inverse));
  if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -FBLA_INF : (m + fbla::lg2(l)) * 0.6931471805599453f;
}

}  // namespace
}  // namespace paged

extern "C" cudaError_t paged_k_attend_launch(const mlops_paged_attend_args *a, const mlops_paged_cache *c, void *, cudaStream_t stream) {
  const int64_t ctas = ((int64_t)a->tokens * a->q_heads + paged::WARPS - 1) / paged::WARPS;
  return fbla::launch(true, 1, a->type == MLOPS_PAGED_BF16 ? paged::attend_kernel<MLOPS_PAGED_BF16> : paged::attend_kernel<MLOPS_PAGED_FP16>,
                      dim3((unsigned)ctas), 32 * paged::WARPS, 0, stream, *a, *c, a->scale * 1.4426950408889634f);
}
