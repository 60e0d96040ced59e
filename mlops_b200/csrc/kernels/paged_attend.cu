// Dispatch of the paged cache's attention: requests with few columns (queries times query heads per KV head) are streamed, the others go to the tile kernel.
#include "paged_attend.cuh"

namespace paged {
namespace {

// Columns of a request that is streamed, at most. us on the device (a graph of calls with a scratch of their own), 16 requests of 5 000 to 16 000 tokens, 32 / 8 heads: 3
// to 6 queries (12 to 24 columns) take 103 with a limit of 24 or 32 and 156 with 16; 8 queries (32 columns) 125 streamed and 148 as tiles; 10 queries (40 columns), a
// third tile of the stream, 174 and 152.
constexpr int WIDE = 32;

struct Scratch {  // offsets: the counters of both kernels (zeros at first), their partial rows
  size_t stream_counters, tile_counters, stream_part, tile_part, bytes;
};
Scratch scratch_of(int sms, bool tiles) {
  Scratch s{};
  const size_t counters = ((size_t)sms * sizeof(int) + 255) / 256 * 256;
  s.tile_counters = counters;
  s.stream_part = 2 * counters;
  s.tile_part = s.stream_part + (size_t)sms * 2 * 16 * PSTRIDE * sizeof(float);
  s.bytes = s.tile_part + (tiles ? (size_t)sms * 2 * 256 * PSTRIDE * sizeof(float) : 0);
  return s;
}
// whether some request may have more than WIDE columns
bool may_be_wide(const mlops_paged_attend_args *a, int kv_heads) { return a->starts || a->q_heads / kv_heads > WIDE; }

// Streamed in tiles of 8 columns where a request has no more on average, else of 16; us on the device: 64 requests of 1K-64K tokens and 4 columns each take 176 in tiles
// of 8 and 254 in tiles of 16, 16 requests of 5 000 to 16 000 tokens with 12 to 24 columns 105 and 103, with 32 columns 153 and 125. The host knows the average only.
template <int TYPE> cudaError_t attend(const Call &k, bool tiles, int sms, cudaStream_t stream) {
  const bool narrow = (int64_t)k.a.tokens * k.group <= (int64_t)8 * k.a.batch;
  const cudaError_t e = narrow ? launch_stream<TYPE, 1>(k, sms, stream) : launch_stream<TYPE, 2>(k, sms, stream);
  return e != cudaSuccess || !tiles ? e : launch_tile<TYPE>(k, sms, stream);
}

}  // namespace
}  // namespace paged

extern "C" size_t paged_k_attend_scratch(const mlops_paged_attend_args *a, int kv_heads, int sms) { return paged::scratch_of(sms, paged::may_be_wide(a, kv_heads)).bytes; }

extern "C" cudaError_t paged_k_attend_launch(const mlops_paged_attend_args *a, const mlops_paged_cache *c, void *scratch, int sms, cudaStream_t stream) {
  const bool tiles = paged::may_be_wide(a, c->kv_heads);
  const paged::Scratch s = paged::scratch_of(sms, tiles);
  char *const base = static_cast<char *>(scratch);
  paged::Call k{};
  k.a = *a;
  k.c = *c;
  k.sl = a->scale * 1.4426950408889634f;
  k.group = a->q_heads / c->kv_heads;
  k.by_group = paged::Divisor(k.group);
  k.wide = paged::WIDE;
  k.stream_counters = reinterpret_cast<int *>(base + s.stream_counters);
  k.tile_counters = reinterpret_cast<int *>(base + s.tile_counters);
  k.stream_part = reinterpret_cast<float *>(base + s.stream_part);
  k.tile_part = reinterpret_cast<float *>(base + s.tile_part);
  return a->type == MLOPS_PAGED_BF16 ? paged::attend<MLOPS_PAGED_BF16>(k, tiles, sms, stream) : paged::attend<MLOPS_PAGED_FP16>(k, tiles, sms, stream);
}
