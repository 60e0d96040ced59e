// Dispatch of the paged cache's attention: requests with few columns (queries times query heads per KV head) are streamed, the others go to the tile kernel.
#include "paged_attend.cuh"

namespace paged {
namespace {

// Columns of a request that is streamed, at most. us on the device (a graph of calls with a scratch of their own), 16 requests of 5 000 to 16 000 tokens, 32 / 8 heads: 3
// to 6 queries (12 to 24 columns) take 103 with a limit of 24 or 32 and 156 with 16; 8 queries (32 columns) 125 streamed and 148 as tiles; 10 queries (40 columns), a
// third tile of the stream, 174 and 152.
constexpr int WIDE = 32;

struct Scratch {  // offsets: the counters of both kernels (zeros at first), their partial rows; SHARED: the rows of common and own tokens
  size_t stream_counters, tile_counters, stream_part, tile_part, common_rows, own_rows, bytes;
};
static_assert(2 * (PAGED_K_MAX_SMS * sizeof(int) + 255) / 256 * 256 <= MLOPS_PAGED_SCRATCH_ZEROS, "the counters are zeros");
Scratch scratch_of(int sms, bool tiles, size_t rows) {
  Scratch s{};
  const size_t counters = ((size_t)sms * sizeof(int) + 255) / 256 * 256;
  s.tile_counters = counters;
  s.stream_part = 2 * counters;
  s.tile_part = s.stream_part + (size_t)sms * 2 * 16 * PSTRIDE * sizeof(float);
  s.common_rows = s.tile_part + (tiles ? (size_t)sms * 2 * 256 * PSTRIDE * sizeof(float) : 0);
  s.own_rows = s.common_rows + rows * PSTRIDE * sizeof(float);
  s.bytes = s.own_rows + rows * PSTRIDE * sizeof(float);
  return s;
}
// whether some request (common tokens: some group) may have more than WIDE columns
bool may_be_wide(const mlops_paged_attend_args *a, int kv_heads, bool shared) {
  const int group = a->q_heads / kv_heads;
  return shared ? (int64_t)a->tokens * group > WIDE : a->starts || group > WIDE;
}

// Streamed in tiles of 8 columns where a request has no more on average, else of 16; us on the device: 64 requests of 1K-64K tokens and 4 columns each take 176 in tiles
// of 8 and 254 in tiles of 16, 16 requests of 5 000 to 16 000 tokens with 12 to 24 columns 105 and 103, with 32 columns 153 and 125. The host knows the average only.
template <int TYPE, int MODE> cudaError_t attend(const Call &k, bool tiles, int sms, cudaStream_t stream) {
  const auto few = [&](const Call &k) { return k.narrow == 8 ? launch_stream<TYPE, 1, MODE>(k, sms, stream) : launch_stream<TYPE, 2, MODE>(k, sms, stream); };
  if constexpr (MODE == SHARED) {
    // the stream's CTAs begin where the tile kernel's end: neither reads what the other leaves
    cudaError_t e = tiles ? launch_tile<TYPE, MODE>(k, sms, stream) : cudaSuccess;
    Call second = k;
    second.wait_last = tiles;
    if (e == cudaSuccess) e = few(second);
    return e != cudaSuccess ? e : launch_merge<TYPE>(k, sms, stream);
  }
  // the tile kernel's CTAs begin where the stream's end: neither reads what the other leaves
  const cudaError_t e = few(k);
  Call second = k;
  second.wait_last = true;
  return e != cudaSuccess || !tiles ? e : launch_tile<TYPE, MODE>(second, sms, stream);
}

template <int MODE> cudaError_t call(const mlops_paged_attend_args *a, const mlops_paged_common *common, const mlops_paged_cache *c, void *scratch, int sms, cudaStream_t stream) {
  const bool tiles = may_be_wide(a, c->kv_heads, MODE == SHARED);
  const Scratch s = scratch_of(sms, tiles, MODE == SHARED ? (size_t)a->tokens * a->q_heads : 0);
  char *const base = static_cast<char *>(scratch);
  Call k{};
  k.a = *a;
  k.c = *c;
  k.sl = a->scale * 1.4426950408889634f;
  k.group = a->q_heads / c->kv_heads;
  k.by_group = Divisor(k.group);
  k.wide = WIDE;
  const int64_t room = (int64_t)a->width * c->page_size;
  k.room = (int)(room < INT32_MAX - 255 ? room : INT32_MAX - 255);
  k.narrow = (int64_t)a->tokens * k.group <= (int64_t)8 * a->batch ? 8 : 16;
  k.stream_counters = reinterpret_cast<int *>(base + s.stream_counters);
  k.tile_counters = reinterpret_cast<int *>(base + s.tile_counters);
  k.stream_part = reinterpret_cast<float *>(base + s.stream_part);
  k.tile_part = reinterpret_cast<float *>(base + s.tile_part);
  if (MODE == SHARED) {
    k.part_rows = (int)((s.common_rows - s.stream_part) / (PSTRIDE * sizeof(float)));
    k.common = *common;
    k.common_rows = reinterpret_cast<float *>(base + s.common_rows);
    k.own_rows = reinterpret_cast<float *>(base + s.own_rows);
  }
  return a->type == MLOPS_PAGED_BF16 ? attend<MLOPS_PAGED_BF16, MODE>(k, tiles, sms, stream) : attend<MLOPS_PAGED_FP16, MODE>(k, tiles, sms, stream);
}

}  // namespace
}  // namespace paged

extern "C" size_t paged_k_attend_scratch(const mlops_paged_attend_args *a, int kv_heads, int shared, int sms) {
  return paged::scratch_of(sms, paged::may_be_wide(a, kv_heads, shared), shared ? (size_t)a->tokens * a->q_heads : 0).bytes;
}
extern "C" cudaError_t paged_k_attend_launch(const mlops_paged_attend_args *a, const mlops_paged_cache *c, void *scratch, int sms, cudaStream_t stream) {
  return paged::call<paged::CAUSAL>(a, nullptr, c, scratch, sms, stream);
}
extern "C" cudaError_t paged_k_cross_attend_launch(const mlops_paged_attend_args *a, const mlops_paged_cache *c, void *scratch, int sms, cudaStream_t stream) {
  return paged::call<paged::WHOLE>(a, nullptr, c, scratch, sms, stream);
}
extern "C" cudaError_t paged_k_attend_shared_launch(const mlops_paged_attend_args *a, const mlops_paged_common *common, const mlops_paged_cache *c, void *scratch, int sms,
                                                    cudaStream_t stream) {
  return paged::call<paged::SHARED>(a, common, c, scratch, sms, stream);
}
