// The thin C ABI between the host layer of the paged cache (validation) and its CUDA kernels: one launcher per operator, arguments as in
// include/mlops_paged.h. The host layer checks; nothing here validates.
#pragma once
#include "../../../include/mlops_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* requests of one call: their prefix sums live in shared memory */
#define PAGED_K_MAX_ASSIGNED 16384
#define PAGED_K_MAX_ATTENDED 2048

cudaError_t paged_k_assign_launch(const mlops_paged_assign_args *a, cudaStream_t stream);
cudaError_t paged_k_append_launch(const mlops_paged_cache *c, int tokens, int type, const void *k, int64_t k_ts, int64_t k_hs, const void *v, int64_t v_ts,
                                  int64_t v_hs, const int *slots, int sms, cudaStream_t stream);
cudaError_t paged_k_read_launch(const mlops_paged_cache *c, int tokens, int type, const int *slots, void *k, void *v, int sms, cudaStream_t stream);
size_t paged_k_attend_scratch(const mlops_paged_attend_args *a, int kv_heads, int sms);
cudaError_t paged_k_attend_launch(const mlops_paged_attend_args *a, const mlops_paged_cache *c, void *scratch, int sms, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
