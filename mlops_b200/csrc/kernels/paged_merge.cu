// The outputs of mlops_paged_attend_shared: a row's sums over the tokens that its group has in common, taken once for all of the group's rows, and over its request's own. With
// maxima m, m' and sums l, l' of 2^(s - m), 2^(s - m'), O and O':   M = max(m, m'),   out = (2^(m - M) O + 2^(m' - M) O') / (2^(m - M) l + 2^(m' - M) l').
// A warp per row and query head; all that it may need is on its way at once. Bound by memory: 528 bytes a part, in the L2 for decode steps.
#include "fbla_launch.h"
#include "paged_attend.cuh"

namespace paged {
namespace {

constexpr int WARPS = 8;

struct Part {  // a lane's four channels; m is NOTHING where l is 0
  float4 o;
  float m, l;
};
__device__ __forceinline__ void add(float4 &o, const float4 &x, float f) { o = make_float4(fmaf(x.x, f, o.x), fmaf(x.y, f, o.y), fmaf(x.z, f, o.z), fmaf(x.w, f, o.w)); }
__device__ __forceinline__ void join(Part &a, float top, const Part &b) {
  const float f = a.l == 0.f ? 0.f : ex2(a.m - top), g = b.l == 0.f ? 0.f : ex2(b.m - top);
  a.o = make_float4(a.o.x * f, a.o.y * f, a.o.z * f, a.o.w * f);
  if (b.l != 0.f) add(a.o, b.o, g);
  a.l = a.l * f + (b.l == 0.f ? 0.f : b.l * g);
  a.m = top;
}
// a row's sums, from itself (x: the lane's channels) or from its pieces, in their order. (A row that starts or groups out of order have left out holds anything: it is zeros where its pieces
// are none.)
__device__ __forceinline__ Part part_of(const Call &k, const float4 &x, const float4 &end, int lane) {
  const int pieces = __float_as_int(end.w), rows = __float_as_int(end.y);
  if (!pieces) {
    if (end.y == 0.f) return Part{make_float4(0.f, 0.f, 0.f, 0.f), NOTHING, 0.f};
    return Part{x, end.x, end.y};
  }
  Part p{make_float4(0.f, 0.f, 0.f, 0.f), NOTHING, 0.f};
  const int at = __float_as_int(end.x);
  if (pieces < 0 || pieces > PAGED_K_MAX_SMS || rows <= 0 || rows > TILE_ROWS || at < 0 || at >= k.part_rows - piece_row(rows, pieces - 1)) return p;
  const float *const first = k.stream_part + (size_t)at * PSTRIDE;
  for (int i0 = 0; i0 < pieces; i0 += 32) {
    const int n = min(pieces - i0, 32);
    float2 z = make_float2(NOTHING, 0.f);
    if (lane < n) z = __ldcg(reinterpret_cast<const float2 *>(first + (size_t)piece_row(rows, i0 + lane) * PSTRIDE + D));
    if (z.y == 0.f) z.x = NOTHING;
    float top = fmaxf(z.x, p.m);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, d));
    const float weight = z.y == 0.f ? 0.f : ex2(z.x - top), keep = p.l == 0.f ? 0.f : ex2(p.m - top);
    p.l = p.l * keep + fbla::warp_sum(z.y * weight);
    p.o = make_float4(p.o.x * keep, p.o.y * keep, p.o.z * keep, p.o.w * keep);
    p.m = top;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float4 v = __ldcg(reinterpret_cast<const float4 *>(first + (size_t)piece_row(rows, i0 + i) * PSTRIDE) + lane);
      add(p.o, v, __shfl_sync(FULL, weight, i));
    }
  }
  return p;
}

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
    Part a = part_of(k, x, x_end, lane);
    if (__float_as_int(x_end.z)) {
      const Part b = part_of(k, y, y_end, lane);
      const float top = fmaxf(a.m, b.m);
      join(a, top, b);
    }
    const float l = a.l;
    const float scale = l == 0.f ? 0.f : __ldg(k.c.v_scale + k.by_group.divide(head)) / l;
    *reinterpret_cast<uint2 *>(out_row(k, row, head) + 4 * lane) = make_uint2(from_floats<TYPE>(a.o.x * scale, a.o.y * scale), from_floats<TYPE>(a.o.z * scale, a.o.w * scale));
    if (k.a.lse && lane == 0) k.a.lse[at] = lse_of(a.m, l);
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
