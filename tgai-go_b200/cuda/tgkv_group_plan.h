/* tgkv_group_plan.h -- how a group call's attention is cut into pieces and
 * dealt to CTAs.  Plain C, shared by the host planner (tgai_cuda_bridge.c) and
 * the kernels (tgkv_group.cu).
 *
 * A row tile is up to 128 query rows of one KV head: TPT = 128 / G tokens times
 * the G query heads of that KV head.  An item is a row tile with the 128-
 * position K/V tiles it attends.  There are two ways to cut a call:
 *   split   (share = 1) row tiles over the packed tokens of all sequences attend
 *           the prefix (items of "sequence" 0 below), row tiles of each
 *           sequence's own tokens attend its own cache, and a merge joins the
 *           two parts of every row: the prefix is read for 128 rows at a time,
 *           whichever sequences they come from;
 *   joined  (share = 0) row tiles of each sequence attend the prefix, then the
 *           own cache.
 * Items in order (sequence, KV head, row tile) form one line of tiles, which is
 * cut into n_cta contiguous stretches of about the same number of tiles (plus
 * TGKV_GROUP_ITEM_COST per item).  A CTA's stretch is a run of pieces: parts of
 * an item's tiles.  Only a stretch's first piece can continue an item and only
 * its last piece can leave one unfinished, so partial results need two slots of
 * 128 rows per CTA (and, split, one row per query row and part).
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
#define TGKV_GROUP_ITEM_COST 1

/* A place on the line: tile `tile` of item (seq, kvh, rt); seq 0: the shared
 * prefix, seq i + 1: sequence i; seq n_seq + 1: the end. */
typedef struct {
    uint32_t seq, kvh, rt, tile;
} TGKvGroupPos;

TGKV_HD uint32_t tgkv_group_tpt(const TGKvGroupParams* p) {
    return TGKV_GROUP_ROWS / (p->n_heads / p->n_kv_heads);
}
TGKV_HD uint32_t tgkv_group_tokens(const TGKvGroupParams* p, uint32_t seq) {
    return seq ? p->tok0[seq] - p->tok0[seq - 1] : (p->share ? p->tok0[p->n_seq] : 0);
}
TGKV_HD uint32_t tgkv_group_row_tiles(const TGKvGroupParams* p, uint32_t seq) {
    const uint32_t tpt = tgkv_group_tpt(p);
    return (tgkv_group_tokens(p, seq) + tpt - 1) / tpt;
}
/* Tiles of the prefix that an item of `seq` attends. */
TGKV_HD uint32_t tgkv_group_prefix_tiles(const TGKvGroupParams* p, uint32_t seq) {
    return (seq == 0) == (p->share != 0) ? (p->prefix_len + TGKV_GROUP_TILE - 1) / TGKV_GROUP_TILE : 0;
}
/* Own rows that row tile rt of sequence `seq` (>= 1) sees at most. */
TGKV_HD uint32_t tgkv_group_own_rows(const TGKvGroupParams* p, uint32_t seq, uint32_t rt) {
    const uint32_t n = tgkv_group_tokens(p, seq), e = (rt + 1) * tgkv_group_tpt(p);
    return p->old_len[seq - 1] + (e < n ? e : n);
}
TGKV_HD uint32_t tgkv_group_item_tiles(const TGKvGroupParams* p, uint32_t seq, uint32_t rt) {
    const uint32_t pre = tgkv_group_prefix_tiles(p, seq);
    return seq ? pre + (tgkv_group_own_rows(p, seq, rt) + TGKV_GROUP_TILE - 1) / TGKV_GROUP_TILE : pre;
}
/* The first sequence at or after seq that has items. */
TGKV_HD uint32_t tgkv_group_skip(const TGKvGroupParams* p, uint32_t seq) {
    while (seq <= p->n_seq && tgkv_group_tokens(p, seq) == 0) ++seq;
    return seq;
}
TGKV_HD TGKvGroupPos tgkv_group_next_item(const TGKvGroupParams* p, TGKvGroupPos a) {
    a.tile = 0;
    if (++a.rt < tgkv_group_row_tiles(p, a.seq)) return a;
    a.rt = 0;
    if (++a.kvh < p->n_kv_heads) return a;
    a.kvh = 0;
    a.seq = tgkv_group_skip(p, a.seq + 1);
    return a;
}
TGKV_HD int tgkv_group_same_item(TGKvGroupPos a, TGKvGroupPos b) {
    return a.seq == b.seq && a.kvh == b.kvh && a.rt == b.rt;
}
/* a <= b on the line */
TGKV_HD int tgkv_group_le(TGKvGroupPos a, TGKvGroupPos b) {
    if (a.seq != b.seq) return a.seq < b.seq;
    if (a.kvh != b.kvh) return a.kvh < b.kvh;
    if (a.rt != b.rt) return a.rt < b.rt;
    return a.tile <= b.tile;
}

#endif /* TGKV_GROUP_PLAN_H */
