// A step's queries, keys and values on their way from the projection (mlops_paged_append_rotated): q and k rotated by their tokens' positions, q stored, k and v
// quantised into the cache's slots.
//
// Rotation of a pair (x, y) by (c, s): (x c - y s, y c + x s). q takes it in FP32, rounded once to its type at the end. A stored code of k asks on which side of a border a value
// lies, so k's rotation is exact before its one rounding to 16 bits: each product with its error (an FMA gives it), each sum with its (TwoSum: D. Knuth, The Art of Computer
// Programming 2, 4.2.2), and where the rounded sum is not exact its last bit is set, so that rounding it again to 16 bits never meets a halfway case that is none (rounding to odd: S. Boldo, G.
// Melquiond, Emulation of FMA and correctly rounded sums, 2008). What is stored is, bit for bit, what mlops_paged_append stores of the correctly rounded rotation.
#include "paged_store.cuh"
#include <type_traits>

namespace paged {
namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS, CTAS = 2;
constexpr int SLICE = 8;  // heads that a warp has at once: four threads of 32 channels each

struct Turn {
  mlops_paged_rotate_args a;
  Store s;
  Divisor by_parts;
  int q_slices, slices, parts, span;  // slices of 8 query heads, of 8 KV heads behind them; a warp's unit is up to `span` slices of a token, which has `parts` units
};

// channels of a thread: two blocks of 16, which hold the pairs' two halves or whole pairs
struct Two {
  Channels x[2];
};
// (not through the read-only path: the rotated rows may take the queries' place)
template <bool WIDE> __device__ __forceinline__ Channels load_shared(const uint16_t *p) {
  Channels x;
  if (WIDE) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(x.w[0]), "=r"(x.w[1]), "=r"(x.w[2]), "=r"(x.w[3]), "=r"(x.w[4]), "=r"(x.w[5]), "=r"(x.w[6]), "=r"(x.w[7]) : "l"(p));
  } else {
    const uint4 a = reinterpret_cast<const uint4 *>(p)[0], b = reinterpret_cast<const uint4 *>(p)[1];
    x = Channels{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  }
  return x;
}

// x c - y s, rounded to odd: the nearest FP32 number, or where that is not exact the one beside the exact value whose last bit is set
__device__ __forceinline__ float turned_exactly(float x, float c, float y, float s) {
  const float a = __fmul_rn(x, c), a_off = __fmaf_rn(x, c, -a), b = -__fmul_rn(y, s), b_off = -__fmaf_rn(y, s, b);
  const float sum = __fadd_rn(a, b), bb = __fsub_rn(sum, a);
  const float off = __fadd_rn(__fadd_rn(__fsub_rn(a, __fsub_rn(sum, bb)), __fsub_rn(b, bb)), __fadd_rn(a_off, b_off));
  const float r = __fadd_rn(sum, off), rest = __fsub_rn(off, __fsub_rn(r, sum));
  uint32_t bits = __float_as_uint(r);
  if (rest != 0.f && !(bits & 1) && (bits & 0x7f800000u) != 0x7f800000u) bits += (rest > 0.f) == (r > 0.f) ? 1u : ~0u;
  return __uint_as_float(bits);
}
template <bool EXACT> __device__ __forceinline__ float2 turn(float x, float y, float c, float s) {
  if (EXACT) return make_float2(turned_exactly(x, c, y, s), turned_exactly(y, c, x, -s));
  return make_float2(__fmaf_rn(x, c, -__fmul_rn(y, s)), __fmaf_rn(y, c, __fmul_rn(x, s)));
}
template <int TYPE, bool NEIGHBOURS, bool EXACT> __device__ __forceinline__ void rotate(Two &t, const float (&c)[16], const float (&s)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 a = to_floats<TYPE>(t.x[0].w[i]), b = to_floats<TYPE>(t.x[1].w[i]);
    if (NEIGHBOURS) {
      const float2 x = turn<EXACT>(a.x, a.y, c[i], s[i]), y = turn<EXACT>(b.x, b.y, c[8 + i], s[8 + i]);
      t.x[0].w[i] = from_floats<TYPE>(x.x, x.y);
      t.x[1].w[i] = from_floats<TYPE>(y.x, y.y);
    } else {
      const float2 x = turn<EXACT>(a.x, b.x, c[2 * i], s[2 * i]), y = turn<EXACT>(a.y, b.y, c[2 * i + 1], s[2 * i + 1]);
      t.x[0].w[i] = from_floats<TYPE>(x.x, y.x);
      t.x[1].w[i] = from_floats<TYPE>(x.y, y.y);
    }
  }
}

template <int TYPE, bool WIDE, bool NEIGHBOURS> __global__ void __launch_bounds__(THREADS, CTAS) rotate_kernel(const Turn k) {
  fbla::wait_previous_pass();
  fbla::allow_next_pass();
  const int lane = threadIdx.x & 31, t = lane & 3, g = lane >> 2;
  // the thread's blocks: t and its partner where the pairs are halves of the rotated channels, two beside each other elsewhere
  const int half = k.a.rotated / 32;
  const bool turns = t < half;
  const int first = !NEIGHBOURS && turns ? t : 2 * t, second = !NEIGHBOURS && turns ? t + half : 2 * t + 1;
  for (int64_t unit = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); unit < (int64_t)k.a.tokens * k.parts; unit += (int64_t)gridDim.x * WARPS) {
    const int token = k.by_parts.divide((int)unit), slice0 = ((int)unit - token * k.parts) * k.span, slice1 = min(slice0 + k.span, k.slices);
    const int position = __ldg(k.a.positions + token), slot = __ldg(k.s.slots + token);
    const bool known = (unsigned)position < (unsigned)k.a.reach;
    float c[16], s[16];
    if (turns && known) {
      const float4 *const row = reinterpret_cast<const float4 *>(k.a.angles + position * k.a.angle_stride + 16 * t);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = __ldg(row + i), y = __ldg(row + 4 * half + i);
        c[4 * i] = x.x; c[4 * i + 1] = x.y; c[4 * i + 2] = x.z; c[4 * i + 3] = x.w;
        s[4 * i] = y.x; s[4 * i + 1] = y.y; s[4 * i + 2] = y.z; s[4 * i + 3] = y.w;
      }
    }
    auto spoil = [&](Two &x) {  // no position: zeros; one behind the table: NaN
#pragma unroll
      for (int i = 0; i < 8; ++i) x.x[0].w[i] = x.x[1].w[i] = position < 0 ? 0u : 0x7fff7fffu;
    };
    for (int slice = slice0; slice < slice1; ++slice) {
      if (slice < k.q_slices) {
        const int head = SLICE * slice + g;
        if (head >= k.a.q_heads) continue;
        const uint16_t *const from = static_cast<const uint16_t *>(k.a.q) + token * k.a.q_token_stride + head * k.a.q_head_stride;
        Two x{{load_shared<WIDE>(from + 16 * first), load_shared<WIDE>(from + 16 * second)}};
        if (!known) spoil(x);
        else if (turns) rotate<TYPE, NEIGHBOURS, false>(x, c, s);
        uint16_t *const to = static_cast<uint16_t *>(k.a.q_out) + token * k.a.out_token_stride + head * k.a.out_head_stride;
        store_channels<WIDE>(to + 16 * first, x.x[0]);
        store_channels<WIDE>(to + 16 * second, x.x[1]);
      } else {
        const int head = SLICE * (slice - k.q_slices) + g;
        if (head >= k.s.c.kv_heads || position < 0 || !is_slot(k.s.c, slot)) continue;
        const uint16_t *const key = static_cast<const uint16_t *>(k.a.k) + token * k.a.k_token_stride + head * k.a.k_head_stride;
        const uint16_t *const value = static_cast<const uint16_t *>(k.a.v) + token * k.a.v_token_stride + head * k.a.v_head_stride + 32 * t;
        Two x{{load_channels<WIDE>(key + 16 * first), load_channels<WIDE>(key + 16 * second)}};
        const Two y{{load_channels<WIDE>(value), load_channels<WIDE>(value + 16)}};
        if (!known) spoil(x);
        else if (turns) rotate<TYPE, NEIGHBOURS, true>(x, c, s);
        int at;
        uint8_t *const block = block_of(k.s, slot, head, at);
        uint8_t *const codes = block + at * CODE_BYTES, *const scales = block + K_SCALES + at * SCALE_BYTES;
        uint32_t scale[2];
        const float k_inverse = __fdiv_rn(1.f, __ldg(k.s.c.k_scale + head)), v_inverse = __fdiv_rn(1.f, __ldg(k.s.c.v_scale + head));
        const uint2 k0 = quantise<TYPE>(x.x[0], k_inverse, scale[0]), k1 = quantise<TYPE>(x.x[1], k_inverse, scale[1]);
        *reinterpret_cast<uint2 *>(codes + 8 * first) = k0;
        *reinterpret_cast<uint2 *>(codes + 8 * second) = k1;
        scales[first] = (uint8_t)scale[0];
        scales[second] = (uint8_t)scale[1];
        const uint2 v0 = quantise<TYPE>(y.x[0], v_inverse, scale[0]), v1 = quantise<TYPE>(y.x[1], v_inverse, scale[1]);
        *reinterpret_cast<uint4 *>(codes + V_CODES + 16 * t) = make_uint4(v0.x, v0.y, v1.x, v1.y);
        *reinterpret_cast<uint16_t *>(scales + (V_SCALES - K_SCALES) + 2 * t) = (uint16_t)(scale[0] | scale[1] << 8);
      }
    }
  }
}

}  // namespace
}  // namespace paged

extern "C" cudaError_t paged_k_append_rotated_launch(const mlops_paged_cache *c, const mlops_paged_rotate_args *a, int sms, cudaStream_t stream) {
  paged::Turn k{};
  k.a = *a;
  k.s = paged::Store{*c, a->slots, paged::Divisor(c->kv_heads), paged::Divisor(c->page_size), a->tokens * c->kv_heads};
  k.q_slices = (a->q_heads + paged::SLICE - 1) / paged::SLICE;
  k.slices = k.q_slices + (c->kv_heads + paged::SLICE - 1) / paged::SLICE;
  k.span = a->tokens < sms * paged::CTAS * paged::WARPS ? 1 : k.slices;
  k.parts = (k.slices + k.span - 1) / k.span;
  k.by_parts = paged::Divisor(k.parts);
  const int64_t ctas = ((int64_t)a->tokens * k.parts + paged::WARPS - 1) / paged::WARPS, most = (int64_t)sms * paged::CTAS;
  const bool wide = paged::on_32(a->q, a->q_token_stride, a->q_head_stride) && paged::on_32(a->q_out, a->out_token_stride, a->out_head_stride) &&
                    paged::on_32(a->k, a->k_token_stride, a->k_head_stride) && paged::on_32(a->v, a->v_token_stride, a->v_head_stride);
  const auto pick = [&](auto type) {
    constexpr int T = decltype(type)::value;
    return a->interleaved ? wide ? paged::rotate_kernel<T, true, true> : paged::rotate_kernel<T, false, true>
                          : wide ? paged::rotate_kernel<T, true, false> : paged::rotate_kernel<T, false, false>;
  };
  const auto kernel = a->type == MLOPS_PAGED_BF16 ? pick(std::integral_constant<int, MLOPS_PAGED_BF16>{}) : pick(std::integral_constant<int, MLOPS_PAGED_FP16>{});
  return fbla::launch(true, 1, kernel, dim3((unsigned)(ctas < most ? ctas : most)), paged::THREADS, 0, stream, k);
}
