// A step's queries, keys and values on their way from the projection (mlops_paged_append_rotated): q and k rotated by their tokens' positions, q stored, k and v
// quantised into the cache's slots.
//
// Rotation of a pair (x, y) by (c, s): (x c - y s, y c + x s). q takes it in FP32, rounded once to its type at the end. A stored code of k asks on which side of a border a value
// lies, so k's rotation is correctly rounded to 16 bits: r = fl(x c - fl(y s)) is off by at most 2^-24 (|y s| + |r|), and where all numbers so near to r round to the same one, that is it. Where they do not
// (some 2^-14 of the elements), the thread takes all of its pairs in FP64, where the products are exact, and
// sets the last bit of an FP32 sum that is not exact, so that rounding it again to 16 bits never meets a halfway case that is none (rounding to odd: S. Boldo,
// G. Melquiond, Emulation of FMA and correctly rounded sums, 2008). FP16, whose numbers are eight times as close, takes all of K so: 16 384 tokens of 32 / 8 heads, halves and neighbours, 72 and
// 74 us, in BF16 68 and 71. What is stored is, bit for bit, what mlops_paged_append stores of the correctly rounded rotation.
//
// Warps have units of two kinds, dealt evenly over each other so that the ones' memory and the others' arithmetic share a multiprocessor: a token's query heads, eight at a time, with the
// token's angles in registers; eight (token, KV head), four threads each.
#include "paged_store.cuh"
#include <type_traits>

namespace paged {
namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS, CTAS = 2;
constexpr int SLICE = 8;  // heads that a warp has at once: four threads of 32 channels each
constexpr int AHEAD = 2;  // slices of queries on their way at once

struct Turn {
  mlops_paged_rotate_args a;
  Store s;
  Divisor by_parts;
  int q_slices, parts, span;   // slices of 8 query heads; a unit is up to `span` slices of a token, which has `parts` units
  int units;                   // in all
  uint64_t kv_step;            // 2^32 times the share of (token, KV head) units, rounded up: of the first u units floor(u kv_step / 2^32) are of that kind
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

// x c - y s, rounded to odd: the nearest FP32 number towards 0, with its last bit set where that is not exact. In FP64 both products are exact (x and y have 11 bits at most, c and s 24, and
// no exponent comes near FP64's ends), so that the difference rounded down and up is one number or two beside each other.
__device__ __forceinline__ float turned_exactly(double x, double c, double y, double s) {
  const double b = -__dmul_rn(y, s), below = __fma_rd(x, c, b), above = __fma_ru(x, c, b), near = above <= 0. ? above : below;
  const float r = __double2float_rz(near);
  return __uint_as_float(__float_as_uint(r) | (below != above || (double)r != near));
}
// a thread's angles, of its 16 pairs
struct Angles {
  float c[16], s[16];
  __device__ __forceinline__ void load(const float *row, int half, int t) {
    const float4 *const from = reinterpret_cast<const float4 *>(row + 16 * t);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = __ldg(from + i), y = __ldg(from + 4 * half + i);
      c[4 * i] = x.x; c[4 * i + 1] = x.y; c[4 * i + 2] = x.z; c[4 * i + 3] = x.w;
      s[4 * i] = y.x; s[4 * i + 1] = y.y; s[4 * i + 2] = y.z; s[4 * i + 3] = y.w;
    }
  }
};
// every word from the two pairs that it takes: turn(x, y, c, s of its low half, of its high half)
template <int TYPE, bool NEIGHBOURS, class F> __device__ __forceinline__ void each_pair(Two &t, const Angles &k, F turn) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 a = to_floats<TYPE>(t.x[0].w[i]), b = to_floats<TYPE>(t.x[1].w[i]);
    if (NEIGHBOURS) {
      t.x[0].w[i] = turn(a.x, a.y, k.c[i], k.s[i], a.y, a.x, k.c[i], -k.s[i]);
      t.x[1].w[i] = turn(b.x, b.y, k.c[8 + i], k.s[8 + i], b.y, b.x, k.c[8 + i], -k.s[8 + i]);
    } else {
      t.x[0].w[i] = turn(a.x, b.x, k.c[2 * i], k.s[2 * i], a.y, b.y, k.c[2 * i + 1], k.s[2 * i + 1]);
      t.x[1].w[i] = turn(b.x, a.x, k.c[2 * i], -k.s[2 * i], b.y, a.y, k.c[2 * i + 1], -k.s[2 * i + 1]);
    }
  }
}
// each word is two of x c - y s
template <int TYPE, bool NEIGHBOURS> __device__ __forceinline__ void rotate(Two &t, const Angles &k) {
  each_pair<TYPE, NEIGHBOURS>(t, k, [](float x, float y, float c, float s, float u, float v, float d, float r) {
    return from_floats<TYPE>(__fmaf_rn(x, c, -__fmul_rn(y, s)), __fmaf_rn(u, d, -__fmul_rn(v, r)));
  });
}
// the same, correctly rounded where it returns true
template <int TYPE, bool NEIGHBOURS> __device__ __forceinline__ bool rotate_surely(Two &t, const Angles &k) {
  uint32_t unsure = 0;
  each_pair<TYPE, NEIGHBOURS>(t, k, [&](float x, float y, float c, float s, float u, float v, float d, float r) {
    // (the half covers the bounds' own roundings: a - e is a number beside a at least, and within 2^-24 of itself)
    constexpr float OFF = 1.5f / (1 << 24);
    const float p = __fmul_rn(y, s), q = __fmul_rn(v, r), a = __fmaf_rn(x, c, -p), b = __fmaf_rn(u, d, -q);
    const float e = __fmul_rn(__fadd_rn(fabsf(p), fabsf(a)), OFF), f = __fmul_rn(__fadd_rn(fabsf(q), fabsf(b)), OFF);
    const uint32_t lo = from_floats<TYPE>(__fsub_rn(a, e), __fsub_rn(b, f)), hi = from_floats<TYPE>(__fadd_rn(a, e), __fadd_rn(b, f));
    unsure |= lo ^ hi;
    return lo;
  });
  return unsure == 0;
}
template <bool WIDE> __device__ __forceinline__ Two load_two(const uint16_t *p, int first, int second) { return Two{{load_channels<WIDE>(p + 16 * first), load_channels<WIDE>(p + 16 * second)}}; }
template <int TYPE, bool NEIGHBOURS> __device__ __forceinline__ void rotate_exactly(Two &t, const Angles &k) {
  each_pair<TYPE, NEIGHBOURS>(t, k, [](float x, float y, float c, float s, float u, float v, float d, float r) { return from_floats<TYPE>(turned_exactly(x, c, y, s), turned_exactly(u, d, v, r)); });
}
// all of it again, correctly rounded
template <int TYPE, bool WIDE, bool NEIGHBOURS> __device__ __noinline__ Two rotated_exactly(const uint16_t *key, const float *row, int half, int t, int first, int second) {
  Two x = load_two<WIDE>(key, first, second);
  Angles k;
  k.load(row, half, t);
  rotate_exactly<TYPE, NEIGHBOURS>(x, k);
  return x;
}

template <int TYPE, bool WIDE, bool NEIGHBOURS> __global__ void __launch_bounds__(THREADS, CTAS) rotate_kernel(const Turn k) {
  fbla::wait_previous_pass();
  fbla::allow_next_pass();
  const int lane = threadIdx.x & 31, t = lane & 3, g = lane >> 2;
  // the thread's blocks: t and its partner where the pairs are halves of the rotated channels, two beside each other elsewhere
  const int half = k.a.rotated / 32;
  const bool turns = t < half;
  const int first = !NEIGHBOURS && turns ? t : 2 * t, second = !NEIGHBOURS && turns ? t + half : 2 * t + 1;
  Angles angles;
  auto row_of = [&](int position) { return k.a.angles + position * k.a.angle_stride; };
  auto spoil = [&](Two &x, uint32_t bits) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.x[0].w[i] = x.x[1].w[i] = bits;
  };
  constexpr uint32_t NANS = 0x7fff7fffu;  // (of either type)
  for (int64_t u = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); u < k.units; u += (int64_t)gridDim.x * WARPS) {
    const int before = (int)((uint64_t)u * k.kv_step >> 32), after = (int)((uint64_t)(u + 1) * k.kv_step >> 32);
    if (after == before) {  // query heads of a token
      const int unit = (int)u - before, token = k.by_parts.divide(unit), slice0 = (unit - token * k.parts) * k.span, slice1 = min(slice0 + k.span, k.q_slices);
      const int position = __ldg(k.a.positions + token);
      const bool known = (unsigned)position < (unsigned)k.a.reach;
      if (turns && known) angles.load(row_of(position), half, t);
      for (int slice = slice0; slice < slice1; slice += AHEAD) {
        Two x[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int head = SLICE * (slice + i) + g;
          if (slice + i >= slice1 || head >= k.a.q_heads) continue;
          const uint16_t *const from = static_cast<const uint16_t *>(k.a.q) + token * k.a.q_token_stride + head * k.a.q_head_stride;
          x[i] = Two{{load_shared<WIDE>(from + 16 * first), load_shared<WIDE>(from + 16 * second)}};
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int head = SLICE * (slice + i) + g;
          if (slice + i >= slice1 || head >= k.a.q_heads) continue;
          if (!known) spoil(x[i], position < 0 ? 0u : NANS);  // no position: zeros; one behind the table: NaN
          else if (turns) rotate<TYPE, NEIGHBOURS>(x[i], angles);
          uint16_t *const to = static_cast<uint16_t *>(k.a.q_out) + token * k.a.out_token_stride + head * k.a.out_head_stride;
          store_channels<WIDE>(to + 16 * first, x[i].x[0]);
          store_channels<WIDE>(to + 16 * second, x[i].x[1]);
        }
      }
    } else {  // eight (token, KV head)
      const int row = min(SLICE * before + g, k.s.rows - 1), token = k.s.by_heads.divide(row), head = row - token * k.s.c.kv_heads;
      const int position = __ldg(k.a.positions + token), slot = __ldg(k.s.slots + token);
      const bool known = (unsigned)position < (unsigned)k.a.reach;
      const uint16_t *const key = static_cast<const uint16_t *>(k.a.k) + token * k.a.k_token_stride + head * k.a.k_head_stride;
      Two x = load_two<WIDE>(key, first, second);
      const Two y = load_two<WIDE>(static_cast<const uint16_t *>(k.a.v) + token * k.a.v_token_stride + head * k.a.v_head_stride, 2 * t, 2 * t + 1);
      if (!known) {
        spoil(x, NANS);
      } else if (turns) {
        angles.load(row_of(position), half, t);
        if (TYPE == MLOPS_PAGED_FP16) rotate_exactly<TYPE, NEIGHBOURS>(x, angles);
        else if (!rotate_surely<TYPE, NEIGHBOURS>(x, angles)) x = rotated_exactly<TYPE, WIDE, NEIGHBOURS>(key, row_of(position), half, t, first, second);
      }
      if (position < 0 || !is_slot(k.s.c, slot) || SLICE * before + g >= k.s.rows) continue;
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

}  // namespace
}  // namespace paged

extern "C" cudaError_t paged_k_append_rotated_launch(const mlops_paged_cache *c, const mlops_paged_rotate_args *a, int sms, cudaStream_t stream) {
  paged::Turn k{};
  k.a = *a;
  k.s = paged::Store{*c, a->slots, paged::Divisor(c->kv_heads), paged::Divisor(c->page_size), a->tokens * c->kv_heads};
  k.q_slices = (a->q_heads + paged::SLICE - 1) / paged::SLICE;
  // all of a token's slices in one unit where there are tokens enough for the device's warps
  k.span = a->tokens < sms * paged::CTAS * paged::WARPS ? 1 : k.q_slices > 0 ? k.q_slices : 1;
  k.parts = k.q_slices > 0 ? (k.q_slices + k.span - 1) / k.span : 1;
  k.by_parts = paged::Divisor(k.parts);
  const int64_t kv_units = ((int64_t)k.s.rows + paged::SLICE - 1) / paged::SLICE, units = kv_units + (k.q_slices > 0 ? (int64_t)a->tokens * k.parts : 0);
  k.units = (int)units;
  k.kv_step = (((uint64_t)kv_units << 32) + (uint64_t)units - 1) / (uint64_t)units;
  const int64_t ctas = (units + paged::WARPS - 1) / paged::WARPS, most = (int64_t)sms * paged::CTAS;
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
