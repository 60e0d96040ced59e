// Pages and slots of a step's new tokens, from the requests' lengths (mlops_paged_assign).
//
// Two exclusive sums over the requests give everything: starts (of the new tokens) and before (of the new pages). Token i belongs to the request
// b with starts[b] <= i < starts[b + 1], is its token p = held[b] + i - starts[b], and lies in column p / P of its table row: in the page that is
// there, where the column was in use before, else in page ring[head + before[b] + column - columns in use]. The token that opens a page enters
// it into the table. Tokens without a row of the step (it has fewer than are added) are not added: starts end at `tokens`, and what follows from them -- lengths,
// pages that are taken -- leaves them out, so that every page that is taken is in the table. Nothing that is read is written in the same call, so no CTA waits for another: every CTA forms both sums for itself (8 bytes
// per request from L2) and serves a share of the tokens. Bound by latency, launch and two passes over the requests: 64 requests of one new token each 3.3 us on the
// device, 500 with some 40 000 new tokens 7.6.
#include "fbla_launch.h"
#include "paged_kernels.h"
#include "fbla_device.cuh"
#include <climits>

namespace paged {
namespace {

constexpr int THREADS = 256;

// columns of a table row that `tokens` tokens use
__device__ __forceinline__ int columns(long long tokens, int page_size, int width) {
  const long long n = (tokens + page_size - 1) / page_size;
  return (int)(n < width ? n : width);
}

// the request of token i: starts[b] <= i < starts[b + 1]
__device__ __forceinline__ int request_of(const int *starts, int batch, int i) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS) assign_kernel(const mlops_paged_assign_args a) {
  extern __shared__ int sums[];  // starts[batch + 1], before[batch + 1]
  __shared__ long long warp_new[THREADS / 32];
  __shared__ int warp_pages[THREADS / 32], over_all;
  int *const starts = sums, *const before = sums + a.batch + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  fbla::wait_previous_pass();
  fbla::allow_next_pass();
  if (tid == 0) over_all = 0;
  __syncthreads();
  // both sums, THREADS requests at a time
  long long all_new = 0;
  int all_pages = 0, over = 0;
  for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
    const int b = b0 + tid;
    long long n = 0;
    int pages = 0;
    if (b < a.batch) {
      const int held = max(__ldg(a.held + b), 0);
      n = max(__ldg(a.added + b), 0);
      const int have = columns(held, a.page_size, a.width);
      pages = columns(held + n, a.page_size, a.width) - have;
      // (columns that the table does not have)
      over += (int)(max((held + n + a.page_size - 1) / a.page_size, (long long)a.width) - max(((long long)held + a.page_size - 1) / a.page_size, (long long)a.width));
    }
    long long n_sum = n;
    int p_sum = pages;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(fbla::FULL, n_sum, o);
      const int y = __shfl_up_sync(fbla::FULL, p_sum, o);
      if (lane >= o) n_sum += x, p_sum += y;
    }
    if (lane == 31) warp_new[warp] = n_sum, warp_pages[warp] = p_sum;
    __syncthreads();
    long long n_base = all_new;
    int p_base = all_pages;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) n_base += warp_new[w], p_base += warp_pages[w];
      all_new += warp_new[w];
      all_pages += warp_pages[w];
    }
    if (b < a.batch) {
      starts[b] = (int)min(n_base + n_sum - n, (long long)a.tokens);
      before[b] = p_base + p_sum - pages;
    }
    __syncthreads();
  }
  if (over) atomicAdd(&over_all, over);
  if (tid == 0) starts[a.batch] = (int)min(all_new, (long long)a.tokens), before[a.batch] = all_pages;
  __syncthreads();
  const int64_t head = __ldg(reinterpret_cast<const long long *>(a.cursor)), tail = __ldg(reinterpret_cast<const long long *>(a.cursor) + 1);
  const int64_t left = min(max((long long)(tail - head), 0ll), (long long)a.ring_size);  // (never more than the ring holds)
  if (blockIdx.x == 0) {
    for (int b = tid; b <= a.batch; b += THREADS) {
      a.starts[b] = starts[b];
      if (b < a.batch) a.lengths[b] = (int)min((long long)max(__ldg(a.held + b), 0) + (starts[b + 1] - starts[b]), (long long)INT_MAX);
    }
    if (tid == 0) {
      int pages = all_pages;
      if (all_new > a.tokens) {  // cut: the pages of the requests before the last one that has rows, and those of its rows
        const int b = a.tokens ? request_of(starts, a.batch, a.tokens - 1) : 0, held = max(__ldg(a.held + b), 0);
        pages = before[b] + columns((long long)held + (starts[b + 1] - starts[b]), a.page_size, a.width) - columns(held, a.page_size, a.width);
      }
      const int64_t taken = min((long long)pages, (long long)left);
      a.moved[0] = head + taken;
      a.moved[1] = tail;
      a.moved[2] = all_pages - taken + over_all;
    }
  }
  for (int i = blockIdx.x * THREADS + tid; i < a.tokens; i += gridDim.x * THREADS) {
    int slot = -1, position = -1;
    if (i < starts[a.batch]) {
      const int lo = request_of(starts, a.batch, i);
      const int P = a.page_size;
      const uint32_t held = max(__ldg(a.held + lo), 0), p = held + (uint32_t)(i - starts[lo]);
      if (p <= INT_MAX) {  // (a position behind that is in no table)
        position = (int)p;
        const int column = position / P, have = columns(held, P, a.width);
        int *const entry = a.table + (size_t)lo * a.table_stride + column;
        int page = -1;
        if (column < have) {
          page = __ldg(entry);
        } else if (column < a.width) {
          const int64_t nth = before[lo] + column - have;
          if (nth < left) {
            const int64_t at = (head + nth) % a.ring_size;
            page = __ldg(a.ring + (at < 0 ? at + a.ring_size : at));
          }
          if (position % P == 0) *entry = page;
        }
        const int64_t in_pool = (int64_t)page * P + position % P;
        if (page >= 0 && in_pool <= INT_MAX) slot = (int)in_pool;  // (a pool has fewer than 2^31 slots)
      }
    }
    a.slots[i] = slot;
    a.positions[i] = position;
  }
}

}  // namespace
}  // namespace paged

extern "C" cudaError_t paged_k_assign_launch(const mlops_paged_assign_args *a, cudaStream_t stream) {
  const size_t smem = 2 * ((size_t)a->batch + 1) * sizeof(int);
  static thread_local bool asked[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (smem > 48 * 1024 && !(dev < 64 && asked[dev])) {
    const cudaError_t e = cudaFuncSetAttribute(paged::assign_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * (PAGED_K_MAX_ASSIGNED + 1) * (int)sizeof(int));
    if (e != cudaSuccess) return e;
    if (dev < 64) asked[dev] = true;
  }
  const int ctas = (a->tokens + 4 * paged::THREADS - 1) / (4 * paged::THREADS);
  return fbla::launch(true, 1, paged::assign_kernel, dim3(ctas < 1 ? 1 : ctas > 148 ? 148 : ctas), paged::THREADS, smem, stream, *a);
}
