/* tgkv_group_plan.h -- how a group call's attention is cut into pieces and
 * dealt to CTAs.  Plain C, shared by the host planner (tgai_cuda_bridge.c) and
 * the kernels (tgkv_group.cu).
 *
 * A row tile is up to 128 query rows of one KV head: 128 / G tokens times the G
 * query heads of that KV head.  An item is one or two consecutive row tiles, or
 * (light) up to 16 query rows, with the 128-position K/V tiles they attend.
 * There are two ways to cut a call:
 *   split   (share = 1) items over the packed tokens of all sequences attend the
 *           prefix ("sequence" 0 below), items of each sequence's own tokens
 *           attend its own cache, and a merge joins the two parts of every row:
 *           the prefix is read for all rows of an item at once, whichever
 *           sequences they come from;
 *   joined  (share = 0) items of each sequence attend the prefix, then the own
 *           cache.
 * Items in order (sequence, KV head, place in the sequence) form a line of
 * tiles, which is cut into n_cta contiguous stretches of about the same cost
 * (tiles plus item_cost per item).  A CTA's stretch is a run of
 * pieces: parts of an item's tiles.  Only a stretch's first piece can continue
 * an item and only its last piece can leave one unfinished, so partial results
 * need two slots of an item's rows per CTA (and, split, one row per query row
 * and part).
 * Line 0 holds the items of tgkv_group.cu, line 1 those of tgkv_group_light.cuh:
 * the sequences' own items when none of them has more than the light rows (most
 * decode steps), and with them the prefix's when all tokens together are that
 * few.
 */
#ifndef TGKV_GROUP_PLAN_H
#define TGKV_GROUP_PLAN_H
#include <stdint.h>

#include "tgkv_launch.h"

#ifdef __CUDACC__
#define TGKV_HD __host__ __device__ __forceinline__
#else
#define TGKV_HD static inline
#endif

#define TGKV_GROUP_ROWS 128
#define TGKV_GROUP_TILE 128

/* What the cut depends on. */
typedef struct {
    uint32_t n_seq, n_kv_heads, prefix_len, share;
    uint32_t tpt;                /* tokens of a row tile: 128 / G */
    uint32_t item_tokens;        /* tokens of an item */
    uint32_t item_cost;          /* of an item beside its tiles, in tiles */
    const uint32_t* old_len;     /* [n_seq] */
    const uint32_t* tok0;        /* [n_seq + 1] */
} TGKvGroupShape;

/* A place on the line: tile `tile` of item (seq, kvh, at); seq 0: the shared
 * prefix, seq i + 1: sequence i; seq n_seq + 1: the end. */
typedef struct {
    uint32_t seq, kvh, at, tile;
} TGKvGroupPos;

TGKV_HD uint32_t tgkv_group_tokens(const TGKvGroupShape* s, uint32_t seq) {
    return seq ? s->tok0[seq] - s->tok0[seq - 1] : (s->share ? s->tok0[s->n_seq] : 0);
}
TGKV_HD uint32_t tgkv_group_items(const TGKvGroupShape* s, uint32_t seq) {
    return (tgkv_group_tokens(s, seq) + s->item_tokens - 1) / s->item_tokens;
}
/* Tiles of the prefix that an item of `seq` attends. */
TGKV_HD uint32_t tgkv_group_prefix_tiles(const TGKvGroupShape* s, uint32_t seq) {
    return (seq == 0) == (s->share != 0) ? (s->prefix_len + TGKV_GROUP_TILE - 1) / TGKV_GROUP_TILE : 0;
}
/* Own rows that item `at` of sequence `seq` (>= 1) sees at most. */
TGKV_HD uint32_t tgkv_group_own_rows(const TGKvGroupShape* s, uint32_t seq, uint32_t at) {
    const uint32_t n = tgkv_group_tokens(s, seq), e = (at + 1) * s->item_tokens;
    return s->old_len[seq - 1] + (e < n ? e : n);
}
TGKV_HD uint32_t tgkv_group_item_tiles(const TGKvGroupShape* s, uint32_t seq, uint32_t at) {
    const uint32_t pre = tgkv_group_prefix_tiles(s, seq);
    return seq ? pre + (tgkv_group_own_rows(s, seq, at) + TGKV_GROUP_TILE - 1) / TGKV_GROUP_TILE : pre;
}
/* The first sequence at or after seq that has items. */
TGKV_HD uint32_t tgkv_group_skip(const TGKvGroupShape* s, uint32_t seq) {
    while (seq <= s->n_seq && tgkv_group_tokens(s, seq) == 0) ++seq;
    return seq;
}
TGKV_HD TGKvGroupPos tgkv_group_next_item(const TGKvGroupShape* s, TGKvGroupPos a) {
    a.tile = 0;
    if (++a.at < tgkv_group_items(s, a.seq)) return a;
    a.at = 0;
    if (++a.kvh < s->n_kv_heads) return a;
    a.kvh = 0;
    a.seq = tgkv_group_skip(s, a.seq + 1);
    return a;
}
TGKV_HD int tgkv_group_same_item(TGKvGroupPos a, TGKvGroupPos b) {
    return a.seq == b.seq && a.kvh == b.kvh && a.at == b.at;
}
/* a <= b on the line */
TGKV_HD int tgkv_group_le(TGKvGroupPos a, TGKvGroupPos b) {
    if (a.seq != b.seq) return a.seq < b.seq;
    if (a.kvh != b.kvh) return a.kvh < b.kvh;
    if (a.at != b.at) return a.at < b.at;
    return a.tile <= b.tile;
}

#endif /* TGKV_GROUP_PLAN_H */
