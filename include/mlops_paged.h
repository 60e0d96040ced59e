/* A paged cache of K and V in 4 bits for NVIDIA B200 (sm_100a): pages and slots assigned on the device, quantise-on-write,
 * also with a position's rotation on the way, read-back, and attention over the pages: causal, to states of another length, and of requests that begin alike. An addition of this
 * library; the reference has no paged cache.
 *
 * Pool. Head dimension 128. A page holds page_size tokens (a multiple of 16) of every KV head; slot s of the pool is token
 * s % page_size of page s / page_size. The unit of (page, KV head) is page_size / 16 blocks of 2304 bytes, one after the
 * other; a block holds 16 tokens:
 *     byte    0: K codes  [16 tokens][64 bytes]      byte 1024: V codes  [16 tokens][64 bytes]
 *     byte 2048: K scales [16 tokens][ 8 bytes]      byte 2176: V scales [16 tokens][ 8 bytes]
 * A code is E2M1: bit 3 the sign, bits 2-0 the magnitude 0, 0.5, 1, 1.5, 2, 3, 4, 6; channel 2 i is the low half of byte i,
 * channel 2 i + 1 the high half. Scale byte j is E4M3 and serves channels 16 j .. 16 j + 15. With the head's factor g
 * (k_scale or v_scale, FP32) an element is   code * scale * g,   4.5 bits per element; code * scale has at most 6 significant
 * bits and is a normal FP16 or BF16 number, so that tensor cores take it without a rounding.
 *
 * Quantisation of 16 channels x, in FP32 with one rounding per operation: y = x * (1 / g); scale = E4M3(min(448,
 * max |y| * 0.16666667)); code = E2M1(y / scale), both to the nearest, halfway to the even code, |code| at most 6; codes of a
 * zero scale are zeros. A block with a y that is not finite stores scale 0x7f (NaN) and zero codes: it reads as NaN.
 *
 * Attention. The requests' pages are named by a block table: token p of request b is in page table[b][p / page_size]. A
 * request that holds length[b] tokens and has n = starts[b + 1] - starts[b] queries: query i is the request's token
 * length - n + i and sees the tokens 0 .. length - n + i (its own was appended before). A query that sees nothing (an empty
 * request; more queries than tokens) has zeros as its output and -infinity as its log-sum-exp. Tokens whose table entry names
 * no page of the pool are not seen. What a page holds behind a request's last token is never used, whatever its bytes are. A token
 * whose K holds NaN makes the KV head's rows that see it NaN, one whose V does the 16 channels of the NaN block in those rows;
 * rows that do not see it are as if it were not there.
 *
 * All functions enqueue on `stream`, allocate nothing and do not synchronise; lengths, tables and slots live on the device, so
 * a captured call follows them. Status codes as in mlops_fbla.h; mlops_paged_last_error() is the calling thread's message. */
#ifndef MLOPS_PAGED_H
#define MLOPS_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "mlops_fbla.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MLOPS_PAGED_HEAD_DIM 128
#define MLOPS_PAGED_BLOCK 16          /* tokens of a block */
#define MLOPS_PAGED_BLOCK_BYTES 2304

/* 16-bit types of K, V, queries and outputs */
enum { MLOPS_PAGED_BF16 = 0, MLOPS_PAGED_FP16 = 1 };

typedef struct mlops_paged_cache {
  uint8_t *units;              /* 16-byte aligned */
  const float *k_scale, *v_scale; /* [kv_heads], positive */
  int64_t page_stride, head_stride; /* bytes between pages, between a page's heads: multiples of 16, no smaller than a unit */
  int pages, page_size, kv_heads; /* pages * page_size < 2^31 */
} mlops_paged_cache;

/* Pages for `added[b]` new tokens of each request b, which holds held[b]: taken from the ring of free pages
 * ring[cursor[0] % ring_size] .. ring[(cursor[1] - 1) % ring_size], in the order of the requests, and entered into the table.
 * Outputs: starts[batch + 1] (exclusive sums of added), lengths[batch] = held + added, and for token i < `tokens` of the call
 * (request by request) its slot and its position in its request; tokens behind starts[batch] have slot and position -1. Where
 * more than `tokens` are added in all, those behind are left out of everything (starts[batch] = tokens, lengths without them,
 * no page taken for them); the pages that they would have needed count as missing.
 * moved = {cursor[0] + pages taken, cursor[1], pages that were missing}: where the ring runs out or a request outgrows the
 * table's width, entries and slots are -1. The ring holds cursor[1] - cursor[0] pages, at least none and at most ring_size
 * (which may be 0). It is not written: pages go back to it by storing their numbers at ring[cursor[1] % ring_size ...] and
 * advancing cursor[1]. Negative counts are taken as 0, lengths end at 2^31 - 1, a position or slot behind that is -1. No
 * output may overlap an input. */
typedef struct mlops_paged_assign_args {
  int batch, tokens, page_size, width; /* width: entries of a table row that may be used; batch at most 16384 */
  int64_t table_stride;                /* entries between rows of the table */
  int *table;
  const int *held, *added, *ring;
  int ring_size;
  const int64_t *cursor;               /* [2]: head, tail */
  int *slots, *positions, *starts, *lengths;
  int64_t *moved;                      /* [3] */
} mlops_paged_assign_args;
mlops_fbla_status mlops_paged_assign(const mlops_paged_assign_args *args, cudaStream_t stream);

/* Quantises K and V of `tokens` tokens, [tokens][kv_heads][128] with strides in elements (multiples of 8, 16-byte aligned rows),
 * into their slots; tokens whose slot is not one of the pool's are left out. The slots of the pool are distinct: nothing orders two tokens of one
 * slot, which may end with one's codes and the other's scales, other from run to run; no other slot is touched. (Those that
 * mlops_paged_assign gives are, where no page is in two places of the ring and the table's rows.) */
mlops_fbla_status mlops_paged_append(const mlops_paged_cache *cache, int tokens, int type, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                                     const void *v, int64_t v_token_stride, int64_t v_head_stride, const int *slots, cudaStream_t stream);

/* A step's tokens as the projection leaves them: q and k rotated by the tokens' positions, q stored, k and v quantised into the slots as
 * mlops_paged_append does. Rotation of a pair (x, y) of channels by position p: (x c - y s, y c + x s) with c = angles[p][i], s = angles[p][rotated / 2 + i]
 * for pair i: channels (i, i + rotated / 2), or (2 i, 2 i + 1) where `interleaved`; channels from `rotated` on stay as they are. Rotated q is rounded once to the
 * type (FP32 arithmetic); rotated k is the exact rotation rounded once to the type (BF16:
 * where that is 0 or above 2^-100 in magnitude), so that the cache's bytes are those that mlops_paged_append stores of it.
 * A token without a slot of the pool has its q rotated and is not stored. A token of a negative position (a row that is no request's) has zeros as its
 * q and is not stored; one whose position is behind the table has NaN as its q, and its K is stored as NaN. q_out may be q with the same strides, and overlaps no other input
 * or q. */
typedef struct mlops_paged_rotate_args {
  int tokens, q_heads, type;                /* q_heads: any number, 0 too */
  int rotated, interleaved;                 /* rotated: 32, 64, 96 or 128; interleaved: 0 or 1 */
  int reach;                                /* positions of the table */
  const float *angles;                      /* [reach][rotated], angle_stride floats between rows (a multiple of 4), 16-byte aligned */
  int64_t angle_stride;
  const void *q, *k, *v;                    /* [tokens][heads][128], strides in elements: multiples of 8 */
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  void *q_out;
  int64_t out_token_stride, out_head_stride;
  const int *slots, *positions;             /* [tokens]; the slots of the pool are distinct */
} mlops_paged_rotate_args;
mlops_fbla_status mlops_paged_append_rotated(const mlops_paged_cache *cache, const mlops_paged_rotate_args *args, cudaStream_t stream);

/* The values of `tokens` slots as [tokens][kv_heads][128], rounded once to `type`; zeros for a slot that is not one of the pool's. */
mlops_fbla_status mlops_paged_read(const mlops_paged_cache *cache, int tokens, int type, const int *slots, void *k, void *v, cudaStream_t stream);

typedef struct mlops_paged_attend_args {
  int batch, tokens, q_heads, type;    /* tokens: rows of q; kv_heads divides q_heads; batch at most 2048 */
  const void *q;                       /* [tokens][q_heads][128], strides in elements: multiples of 8 */
  int64_t q_token_stride, q_head_stride;
  void *out;                           /* likewise */
  int64_t out_token_stride, out_head_stride;
  float *lse;                          /* [tokens][q_heads] natural log-sum-exp of the scaled scores, or null */
  const int *table;                    /* [batch][width], table_stride entries between rows */
  int64_t table_stride;
  int width;
  const int *lengths;                  /* [batch] */
  const int *starts;                   /* [batch + 1], or null: one query per request, tokens = batch */
  float scale;                         /* 0: 1 / sqrt(128) */
} mlops_paged_attend_args;
/* Bytes of scratch a call of this shape needs (0: the arguments are refused). Of the pointers only starts is looked at: null or not. */
size_t mlops_paged_attend_scratch_bytes(const mlops_paged_attend_args *args, int kv_heads);
/* Rows of q that are no request's, before starts[0] and behind starts[batch], have zeros as their output and -infinity as their log-sum-exp:
 * a slice of a step's requests (table, lengths and starts from request b on) goes with all of the step's rows. Where starts[batch] is
 * above `tokens`, the rows that q does not have are left out and the others see what they would beside them. The first MLOPS_PAGED_SCRATCH_ZEROS bytes of the scratch (16-byte aligned; all of
 * it where it is smaller) are filled with zeros once, before its first call; what a call leaves in it serves the next one, of whatever shape. Calls that overlap need scratches of
 * their own. */
#define MLOPS_PAGED_SCRATCH_ZEROS 8192
mlops_fbla_status mlops_paged_attend(const mlops_paged_attend_args *args, const mlops_paged_cache *cache, void *scratch, size_t scratch_bytes, cudaStream_t stream);

/* Cross attention: as mlops_paged_attend, but every query of a request sees all of the request's lengths[b] tokens (the states of an encoder; queries may outnumber them, as those of
 * several beams do). For requests of one query each, with starts or without, it is mlops_paged_attend. Scratch: mlops_paged_attend_scratch_bytes; one that serves mlops_paged_attend serves this too. */
mlops_fbla_status mlops_paged_cross_attend(const mlops_paged_attend_args *args, const mlops_paged_cache *cache, void *scratch, size_t scratch_bytes, cudaStream_t stream);

/* Requests that begin with the same tokens: group g is the requests starts[g] .. starts[g + 1] - 1 (ascending; requests of no group share nothing), whose first tokens[g] tokens
 * are the same. Of these whole pages count, and these pages' entries in the table's rows of the group's requests are the same (those of any one of them may be read for all).
 * Both arrays live on the device. Where groups or the requests' starts do not ascend, rows of q that belong to two requests, or lie in the rows of two groups, hold anything; the others
 * are as they would be. */
typedef struct mlops_paged_common {
  int groups;                          /* batch + groups at most 2048 */
  const int *starts;                   /* [groups + 1], or null: all requests are one group (groups 1) */
  const int *tokens;                   /* [groups] */
} mlops_paged_common;
/* What mlops_paged_attend gives, within rounding; the pages that a group's requests have in common are read once for all of them. A request whose first query does not see all of the
 * common tokens is attended by itself; its rows are multiplied with the common tokens all the same where it stands in a group, so that one of many queries is better left out of it. So are, all of them, the requests of
 * a group whose queries times query heads per KV head are more than 320 on average, a long chunk among few decodes for instance: nothing is shared in such a group. (A group's first request that takes
 * part is looked for in their order: idle places of a batch are better at a group's end.) Scratch, what the function returns: 1056 bytes per row of q and query head, beside them what mlops_paged_attend asks
 * for, without starts too that of a call with starts where `tokens` times the query heads per KV head are more than 32. */
size_t mlops_paged_attend_shared_scratch_bytes(const mlops_paged_attend_args *args, const mlops_paged_common *common, int kv_heads);
mlops_fbla_status mlops_paged_attend_shared(const mlops_paged_attend_args *args, const mlops_paged_common *common, const mlops_paged_cache *cache, void *scratch, size_t scratch_bytes,
                                            cudaStream_t stream);

const char *mlops_paged_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* MLOPS_PAGED_H */
