/* tgai_kv_group.h -- operators over several KV caches of one layer: sequences
 * that share a prefix, packed prompts of different lengths, and forking and
 * compacting cache rows.  Additive API over include/tgai_kv_cache.h.
 *
 * A group is n caches (one per sequence) and optionally a prefix cache, the
 * K/V of a text that every sequence starts with (a system prompt, a document).
 * Sequence i's positions are the prefix's [0, P), P = tg_kv_len(prefix) at the
 * call, followed by its own cache's [0, len_i): the prefix is stored once and
 * read once per call for all sequences.  A sequence whose history changes
 * inside the prefix gets its own copy of the rows it keeps (tg_kv_fork).
 *
 * Return convention, errors and streams are those of tgai_kv_cache.h: 1 = done,
 * 0 = refused with the reason in tg_kv_last_error() and nothing launched or
 * changed; device work is asynchronous on `stream` (a cudaStream_t; NULL = the
 * legacy default stream).  Lengths live on the host and travel with each
 * launch, so a call captured into a CUDA graph replays with the lengths it was
 * captured with.  No call allocates device memory after create.  A group's
 * scratch (about 59 MB at head_dim 128, half of it at 64) is shared by its
 * calls: order calls and graph replays that use one group (or one of its caches,
 * the prefix's rows included while they change) on one stream or with events.
 * Calls of different groups may overlap.  A group's caches, and those of a fork or
 * compaction, lie on the current device.  Device waits are bounded; one that runs
 * out leaves the call's output undefined and shows in tg_cuda_kv_device_error().
 */
#ifndef TGAI_KV_GROUP_H
#define TGAI_KV_GROUP_H

#include <stdint.h>

#include "tgai_kv_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct TGKvGroup TGKvGroup;

/* A group over n caches (1..1024, all different) and a prefix cache (or NULL;
 * not one of the n), for n_heads query heads.  All caches: bf16, the same
 * n_kv_heads and head_dim (64 or 128); n_heads a multiple of n_kv_heads, up to
 * 128 query heads per KV head.  act is the element type of q, k_new, v_new and
 * out in the group's calls: TG_KV_F32 or TG_KV_BF16.  The caches must outlive
 * the group.  NULL on failure. */
TGKvGroup* tg_kv_group_create(TGKvCache* prefix, TGKvCache* const* caches, uint32_t n,
                              uint32_t n_heads, int act);
void       tg_kv_group_destroy(TGKvGroup* g);

/* One decode step: append row i of k_new / v_new ([n][kv_dim]) to cache i,
 * then attend query row i of q ([n][n_heads][head_dim]) over the prefix and
 * all of cache i, the new row included, into row i of out (same shape).  Each
 * cache's len grows by one.  With k_new and v_new NULL nothing is appended and
 * row i is the query of cache i's last position (len_i >= 1).  All pointers
 * are 16-byte aligned device addresses.  Scores are scaled by
 * mscale / sqrt(head_dim); all caches of the group have the same mscale > 0.
 * Rows behind a cache's length may hold anything.  out overlaps none of the
 * call's other arrays. */
int tg_kv_group_decode(TGKvGroup* g, const void* q, const void* k_new, const void* v_new,
                       void* out, void* stream);

/* Packed prompts: the n_new[i] new tokens of sequence i (0 is allowed), packed
 * one sequence behind the other: total = sum n_new rows of k_new / v_new
 * ([total][kv_dim]) are appended to their caches, then the queries q
 * ([total][n_heads][head_dim]) attend causally into out: token t of sequence i
 * sees the prefix and its own cache's positions up to its own.  Each cache's
 * len grows by n_new[i].  n_new is a host array.  With k_new and v_new NULL
 * nothing is appended and the queries are those of each cache's last n_new[i]
 * positions.  Otherwise as tg_kv_group_decode.
 *
 * Precision: scores, maxima and sums are fp32.  bf16 activations: q is exact, a
 * weight is rounded once to bf16 before it meets V, as the output is.  fp32
 * ones: q and the weights enter as two bf16 terms (16 mantissa bits; within
 * 5e-5 of a head's output scale), or as three (24 bits) where no sequence has
 * more than 10 query rows per KV head (most decode steps' own rows).  Values of
 * K and V that are not finite reach the queries that see them and no others (an
 * infinity of V as NaN where a weight, or with fp32 activations a lo part of one,
 * is 0). */
int tg_kv_group_prompt(TGKvGroup* g, const uint32_t* n_new, const void* q, const void* k_new,
                       const void* v_new, void* out, void* stream);

/* tg_kv_truncate of every cache of the group: cache i to len[i] positions
 * (host array).  Refused as a whole if any len[i] exceeds its cache's len.
 * The prefix is not touched. */
int tg_kv_group_truncate(TGKvGroup* g, const uint32_t* len);

/* Fork: dst[i * fan + j] gets rows [0, n_rows) of src[i] and length n_rows, for
 * i < n_src and j < fan: each source is read once for its fan copies.  Every
 * dst is a different cache and none of the sources; all caches have one
 * dtype, n_kv_heads and head_dim (kv_dim a multiple of 8), n_rows is at most
 * every source's len and every dst's capacity, n_src * fan at most 1024. */
int tg_kv_fork(TGKvCache* const* src, uint32_t n_src, TGKvCache* const* dst, uint32_t fan,
               uint32_t n_rows, void* stream);

/* Compaction, in place: each of the n caches (the layers of one sequence, all
 * of one length) keeps the positions of n_ranges ranges [start[r],
 * start[r] + count[r]) -- host arrays, ascending and disjoint, below len,
 * counts >= 1 -- moved to the front in that order; len becomes the sum of the
 * counts.  n_ranges 0 empties the caches.  Rows keep the K/V they were
 * appended with (their rotation too).  1..1024 different caches of one dtype,
 * n_kv_heads and head_dim (kv_dim a multiple of 8), at most 1024 ranges. */
int tg_kv_compact(TGKvCache* const* caches, uint32_t n, const uint32_t* start,
                  const uint32_t* count, uint32_t n_ranges, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TGAI_KV_GROUP_H */
