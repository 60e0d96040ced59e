// The outputs of mlops_paged_attend_shared: a row's sums over the tokens that its group has in common, taken once for all of the group's rows, and over its request's own. With
// maxima m, m' and sums l, l' of 2^(s - m), 2^(s - m'), O and O':   M = max(m, m'),   out = (2^(m - M) O + 2^(m' - M) O') / (2^(m - M) l + 2^(m' - M) l').
// A warp per row and query head; all that it may need is on its way at once. Bound by memory: 528 bytes a part, in the L2 for decode steps.
#include "fbla_launch.h"
#include "paged_attend.cuh"

namespace paged {
namespace {

constexpr int WARPS = 8;

template <int TYPE> __global__ void __launch_bounds__(32 * WARPS) merge_kernel(const Call k, const Divisor by_heads) {
  fbla::wait_previous_pass();
  fbla::allow_next_pass();
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)k.a.tokens * k.a.q_heads;
  for (int64_t at = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); at < rows; at += (int64_t)gridDim.x * WARPS) {
    const int row = by_heads.divide((int)at), head = (int)at - row * k.a.q_heads;
    const float *const own = sums_row(k, false, row, head), *const common = sums_row(k, true, row, head);
    const float4 x = __ldcg(reinterpret_cast<const float4 *>(own) + lane), x_end = __ldcg(reinterpret_cast<const float4 *>(own + D));
    const float4 y = __ldcg(reinterpret_cast<const float4 *>(common) + lane), y_end = __ldcg(reinterpret_cast<const float4 *>(common + D));
    // (a part without sums holds anything)
    const float m = x_end.y == 0.f ? NOTHING : x_end.x, n = x_end.z == 0.f || y_end.y == 0.f ? NOTHING : y_end.x, top = fmaxf(m, n);
    const float f = x_end.y == 0.f ? 0.f : ex2(m - top), g = x_end.z == 0.f || y_end.y == 0.f ? 0.f : ex2(n - top);
    const float l = (f == 0.f ? 0.f : f * x_end.y) + (g == 0.f ? 0.f : g * y_end.y);
    float4 o = f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
    if (g != 0.f) o = make_float4(fmaf(y.x, g, o.x), fmaf(y.y, g, o.y), fmaf(y.z, g, o.z), fmaf(y.w, g, o.w));
    const float scale = l == 0.f ? 0.f : __ldg(k.c.v_scale + k.by_group.divide(head)) / l;
    *reinterpret_cast<uint2 *>(out_row(k, row, head) + 4 * lane) = make_uint2(from_floats<TYPE>(o.x * scale, o.y * scale), from_floats<TYPE>(o.z * scale, o.w * scale));
    if (k.a.lse && lane == 0) k.a.lse[at] = lse_of(top, l);
  }
}

}  // namespace

template <int TYPE> cudaError_t launch_merge(const Call &k, int sms, cudaStream_t stream) {
  const int64_t ctas = ((int64_t)k.a.tokens * k.a.q_heads + WARPS - 1) / WARPS, most = (int64_t)sms * 8;
  return fbla::launch(true, 1, merge_kernel<TYPE>, dim3((unsigned)(ctas < most ? ctas : most)), 32 * WARPS, 0, stream, k, Divisor(k.a.q_heads));
}
template cudaError_t launch_merge<MLOPS_PAGED_BF16>(const Call &, int, cudaStream_t);
template cudaError_t launch_merge<MLOPS_PAGED_FP16>(const Call &, int, cudaStream_t);

}  // namespace paged
