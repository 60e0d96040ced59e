// Host layer of the paged cache (include/mlops_paged.h): checks a call's arguments and enqueues its kernels on the caller's stream. Nothing here
// allocates or synchronises; the only state is the calling thread's last message.
#include "../kernels/paged_kernels.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>

namespace {

thread_local char g_message[256] = "";

mlops_fbla_status refuse(const char *function, const char *format, ...) {
  const int used = snprintf(g_message, sizeof g_message, "%s: ", function);
  va_list args;
  va_start(args, format);
  if (used >= 0 && (size_t)used < sizeof g_message) vsnprintf(g_message + used, sizeof g_message - (size_t)used, format, args);
  va_end(args);
  return MLOPS_FBLA_INVALID_VALUE;
}
mlops_fbla_status ended(const char *function, cudaError_t error) {
  if (error == cudaSuccess) {
    g_message[0] = '\0';
    return MLOPS_FBLA_OK;
  }
  snprintf(g_message, sizeof g_message, "%s: CUDA reports \"%s\"", function, cudaGetErrorString(error));
  return MLOPS_FBLA_CUDA_ERROR;
}
mlops_fbla_status nothing_to_do() {
  g_message[0] = '\0';
  return MLOPS_FBLA_OK;
}

bool aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool known_type(int type) { return type == MLOPS_PAGED_BF16 || type == MLOPS_PAGED_FP16; }
bool known_page_size(int n) { return n > 0 && n % MLOPS_PAGED_BLOCK == 0; }

// the reason why a pool cannot be used, or null
const char *cache_fault(const mlops_paged_cache *c) {
  if (!c || !c->units || !c->k_scale || !c->v_scale) return "the cache or one of its arrays is null";
  if (c->pages <= 0 || c->kv_heads <= 0 || !known_page_size(c->page_size)) return "a pool has pages, kv_heads > 0 and a page_size that is a multiple of 16";
  if ((int64_t)c->pages * c->page_size > INT32_MAX) return "a pool has fewer than 2^31 slots";
  const int64_t unit = (int64_t)c->page_size / MLOPS_PAGED_BLOCK * MLOPS_PAGED_BLOCK_BYTES;
  if (c->page_stride % 16 || c->head_stride % 16 || (c->pages > 1 && c->page_stride < unit) || (c->kv_heads > 1 && c->head_stride < unit))
    return "page_stride and head_stride are multiples of 16 bytes, no smaller than a unit";
  if (!aligned(c->units, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) return "the units have to start on a 16-byte boundary";
  return nullptr;
}
// rows of 128 elements whose 16-byte pieces are aligned
bool rows_usable(const void *p, int64_t token_stride, int64_t head_stride) { return aligned(p, 16) && token_stride % 8 == 0 && head_stride % 8 == 0; }

bool attend_shape_acceptable(const mlops_paged_attend_args *a, int kv_heads) {
  return a && a->batch >= 0 && a->tokens >= 0 && a->batch <= PAGED_K_MAX_ATTENDED && a->q_heads > 0 && kv_heads > 0 && a->q_heads % kv_heads == 0 &&
         (int64_t)a->tokens * a->q_heads <= INT32_MAX;
}

// the current device's multiprocessors
cudaError_t processors(int *sms) {
  static thread_local int known[64] = {0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && known[dev]) {
    *sms = known[dev];
    return cudaSuccess;
  }
  e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess && dev < 64) known[dev] = *sms;
  return e;
}

}  // namespace

extern "C" {

mlops_fbla_status mlops_paged_assign(const mlops_paged_assign_args *a, cudaStream_t stream) {
  const char *const fn = "mlops_paged_assign";
  if (!a || !a->starts || !a->moved || !a->cursor) return refuse(fn, "a required pointer is null");
  if (a->batch < 0 || a->batch > PAGED_K_MAX_ASSIGNED || a->tokens < 0 || a->width < 0 || a->ring_size < 0)
    return refuse(fn, "needs batch in 0..%d and tokens, width, ring_size >= 0", PAGED_K_MAX_ASSIGNED);
  if (!known_page_size(a->page_size)) return refuse(fn, "page_size %d is no multiple of 16", a->page_size);
  if (a->batch > 0 && (!a->held || !a->added || !a->lengths || (a->width > 0 && !a->table) || a->table_stride < a->width))
    return refuse(fn, "needs held, added, lengths and a table whose stride is at least its width");
  if (a->tokens > 0 && (!a->slots || !a->positions)) return refuse(fn, "slots and positions may not be null");
  if (a->ring_size > 0 && !a->ring) return refuse(fn, "the ring of free pages is null");
  const void *const words[] = {a->table, a->held, a->added, a->ring, a->slots, a->positions, a->starts, a->lengths};
  for (const void *p : words)
    if (!aligned(p, 4)) return refuse(fn, "arrays of int have to start on 4-byte boundaries");
  if (!aligned(a->cursor, 8) || !aligned(a->moved, 8)) return refuse(fn, "cursor and moved have to start on 8-byte boundaries");
  return ended(fn, paged_k_assign_launch(a, stream));
}

mlops_fbla_status mlops_paged_append(const mlops_paged_cache *c, int tokens, int type, const void *k, int64_t k_ts, int64_t k_hs, const void *v, int64_t v_ts,
                                     int64_t v_hs, const int *slots, cudaStream_t stream) {
  const char *const fn = "mlops_paged_append";
  if (const char *why = cache_fault(c)) return refuse(fn, "%s", why);
  if (tokens < 0 || !known_type(type)) return refuse(fn, "needs tokens >= 0 and a type of MLOPS_PAGED_BF16 or MLOPS_PAGED_FP16");
  if ((int64_t)tokens * c->kv_heads > INT32_MAX) return refuse(fn, "tokens * kv_heads has to be below 2^31: split the tokens");
  if (tokens == 0) return nothing_to_do();
  if (!k || !v || !slots) return refuse(fn, "a required pointer is null");
  if (!rows_usable(k, k_ts, k_hs) || !rows_usable(v, v_ts, v_hs) || !aligned(slots, 4))
    return refuse(fn, "k and v have to start on 16-byte boundaries and have strides that are multiples of 8 elements");
  int sms = 0;
  const cudaError_t e = processors(&sms);
  return ended(fn, e != cudaSuccess ? e : paged_k_append_launch(c, tokens, type, k, k_ts, k_hs, v, v_ts, v_hs, slots, sms, stream));
}

mlops_fbla_status mlops_paged_read(const mlops_paged_cache *c, int tokens, int type, const int *slots, void *k, void *v, cudaStream_t stream) {
  const char *const fn = "mlops_paged_read";
  if (const char *why = cache_fault(c)) return refuse(fn, "%s", why);
  if (tokens < 0 || !known_type(type)) return refuse(fn, "needs tokens >= 0 and a type of MLOPS_PAGED_BF16 or MLOPS_PAGED_FP16");
  if ((int64_t)tokens * c->kv_heads > INT32_MAX) return refuse(fn, "tokens * kv_heads has to be below 2^31: split the tokens");
  if (tokens == 0) return nothing_to_do();
  if (!k || !v || !slots) return refuse(fn, "a required pointer is null");
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 4)) return refuse(fn, "k and v have to start on 16-byte boundaries");
  int sms = 0;
  const cudaError_t e = processors(&sms);
  return ended(fn, e != cudaSuccess ? e : paged_k_read_launch(c, tokens, type, slots, k, v, sms, stream));
}

size_t mlops_paged_attend_scratch_bytes(const mlops_paged_attend_args *a, int kv_heads) {
  int sms = 0;
  return attend_shape_acceptable(a, kv_heads) && processors(&sms) == cudaSuccess ? paged_k_attend_scratch(a, kv_heads, sms) : 0;
}

mlops_fbla_status mlops_paged_attend(const mlops_paged_attend_args *a, const mlops_paged_cache *c, void *scratch, size_t scratch_bytes, cudaStream_t stream) {
  const char *const fn = "mlops_paged_attend";
  if (const char *why = cache_fault(c)) return refuse(fn, "%s", why);
  if (!attend_shape_acceptable(a, c->kv_heads))
    return refuse(fn, "needs batch in 0..%d, tokens >= 0, q_heads that kv_heads divides and fewer than 2^31 rows", PAGED_K_MAX_ATTENDED);
  if (!known_type(a->type)) return refuse(fn, "type %d is neither MLOPS_PAGED_BF16 nor MLOPS_PAGED_FP16", a->type);
  if (!(a->scale >= 0.f) || std::isinf(a->scale)) return refuse(fn, "scale has to be a number that is not negative");
  if (!a->starts && a->tokens != a->batch) return refuse(fn, "without starts there is one query per request, but there are %d for %d", a->tokens, a->batch);
  if (a->tokens == 0) return nothing_to_do();
  if (a->width < 0 || a->table_stride < a->width) return refuse(fn, "the table's stride has to be at least its width, and that not negative");
  if (a->width > 0 && (int64_t)a->batch * c->kv_heads > INT32_MAX / (4 * (((int64_t)a->width * c->page_size + 31) / 32)))
    return refuse(fn, "batch * kv_heads * width * page_size is more than a call takes: split the batch");
  if (!a->q || !a->out || !scratch || (a->batch > 0 && !a->lengths) || (a->batch > 0 && a->width > 0 && !a->table)) return refuse(fn, "a required pointer is null");
  if (!rows_usable(a->q, a->q_token_stride, a->q_head_stride) || !rows_usable(a->out, a->out_token_stride, a->out_head_stride) || !aligned(scratch, 16))
    return refuse(fn, "q, out and scratch have to start on 16-byte boundaries, q and out with strides that are multiples of 8 elements");
  if (!aligned(a->lengths, 4) || !aligned(a->starts, 4) || !aligned(a->table, 4) || !aligned(a->lse, 4)) return refuse(fn, "arrays of int and float have to start on 4-byte boundaries");
  int sms = 0;
  const cudaError_t e = scratch_bytes < 16 ? cudaSuccess : processors(&sms);
  if (e != cudaSuccess) return ended(fn, e);
  if (scratch_bytes < 16 || scratch_bytes < paged_k_attend_scratch(a, c->kv_heads, sms)) return refuse(fn, "the scratch is %zu bytes, which are too few for this call", scratch_bytes);
  mlops_paged_attend_args call = *a;
  if (call.scale == 0.f) call.scale = 1.f / std::sqrt((float)MLOPS_PAGED_HEAD_DIM);
  return ended(fn, paged_k_attend_launch(&call, c, scratch, sms, stream));
}

const char *mlops_paged_last_error(void) { return g_message; }

}  // extern "C"
