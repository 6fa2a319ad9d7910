/* tgai_kv_group.c -- operators over several caches: groups that share a
 * prefix, packed prompts, fork and compaction (include/tgai_kv_group.h).
 *
 * Host C: argument checks and length bookkeeping; every check comes before
 * the first launch, so a refused call changes nothing.  Device work goes
 * through tgai_cuda_bridge.c.
 */
#include "tgai_kv_group.h"
#include "tgai_cuda_bridge.h"
#include "tgai_gpu_dispatch.h"
#include "tgai_kv_internal.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>

#define set_err tgkv_kv_set_err
#define TGKV_GROUP_MAX 1024

static int on_cuda(const char* what) {
    if (tg_be_current() == &tg_backend_cuda) return 1;
    set_err("%s needs the cuda backend (tg_be_select(\"cuda\")); no fallback", what);
    return 0;
}

static TGCudaRowCache row_cache(const TGKvCache* c) {
    TGCudaRowCache r = {(uint64_t)(uintptr_t)c->dev, c->max_seq};
    return r;
}

static int ptr_less(const void* a, const void* b) {
    const uintptr_t x = (uintptr_t)*(void* const*)a, y = (uintptr_t)*(void* const*)b;
    return x < y ? -1 : x > y;
}

/* 1 if the n pointers and (if set) `other` are all different. */
static int all_different(TGKvCache* const* v, uint32_t n, const TGKvCache* const* other,
                         uint32_t n_other) {
    const void** s = (const void**)malloc(((size_t)n + n_other) * sizeof(void*));
    if (!s) return 0;
    memcpy(s, v, n * sizeof(void*));
    qsort(s, n, sizeof(void*), ptr_less);
    int ok = 1;
    for (uint32_t i = 1; i < n; i++)
        if (s[i] == s[i - 1]) ok = 0;
    for (uint32_t j = 0; ok && j < n_other; j++) {
        const void* key = other[j];
        if (bsearch(&key, s, n, sizeof(void*), ptr_less)) ok = 0;
    }
    free(s);
    return ok;
}

static int same_geometry(const TGKvCache* a, const TGKvCache* b) {
    return a->n_kv_heads == b->n_kv_heads && a->head_dim == b->head_dim && a->dtype == b->dtype;
}

/* The cuda backend, and caches that lie on the current device. */
static int on_device(const char* what, TGKvCache* const* v, uint32_t n) {
    if (!on_cuda(what)) return 0;
    const int dev = tg_cuda_kv_device();
    for (uint32_t i = 0; i < n; i++)
        if (v[i]->device != dev) {
            set_err("%s: cache %u lies on device %d, called on device %d", what, i, v[i]->device, dev);
            return 0;
        }
    return 1;
}

/* ---- groups --------------------------------------------------------------- */
struct TGKvGroup {
    uint32_t n, n_heads;
    int act, device;
    TGKvCache* prefix;
    TGKvCache** caches;
    uint32_t* old_len;                /* host [n]: own rows before the call's tokens */
    uint32_t* ones;                   /* host [n]: the n_new of a decode step */
    void* table_dev;
    void* scratch;                    /* partial rows, sized for every call of the group */
};

TGKvGroup* tg_kv_group_create(TGKvCache* prefix, TGKvCache* const* caches, uint32_t n,
                              uint32_t n_heads, int act) {
    if (!caches || n == 0 || n > TGKV_GROUP_MAX) {
        set_err("group: need 1..%d caches", TGKV_GROUP_MAX);
        return NULL;
    }
    for (uint32_t i = 0; i < n; i++)
        if (!caches[i]) { set_err("group: null cache %u", i); return NULL; }
    const TGKvCache* c0 = caches[0];
    for (uint32_t i = 1; i < n; i++)
        if (!same_geometry(c0, caches[i])) {
            set_err("group: cache %u differs in geometry or dtype", i);
            return NULL;
        }
    if (prefix && !same_geometry(c0, prefix)) {
        set_err("group: the prefix cache differs in geometry or dtype");
        return NULL;
    }
    if (act != TG_KV_F32 && act != TG_KV_BF16) { set_err("group: invalid dtype %d", act); return NULL; }
    if (c0->dtype != TG_KV_BF16 || (c0->head_dim != 64 && c0->head_dim != 128)) {
        set_err("group: no attention kernel for dtype %d head_dim %u (bf16 caches of 64 or 128)",
                c0->dtype, c0->head_dim);
        return NULL;
    }
    if (n_heads == 0 || n_heads % c0->n_kv_heads || n_heads / c0->n_kv_heads > 128) {
        set_err("group: n_heads %u is not a multiple of n_kv_heads %u, or more than 128 times it",
                n_heads, c0->n_kv_heads);
        return NULL;
    }
    const TGKvCache* pre = prefix;
    if (!all_different(caches, n, &pre, prefix ? 1 : 0)) {
        set_err("group: a cache appears twice");
        return NULL;
    }
    if (!on_device("group", caches, n)) return NULL;
    if (prefix && !on_device("group: prefix", &prefix, 1)) return NULL;
    TGKvGroup* g = (TGKvGroup*)calloc(1, sizeof(TGKvGroup));
    TGCudaRowCache* table = (TGCudaRowCache*)calloc((size_t)n + 1, sizeof(TGCudaRowCache));
    if (g) {
        g->caches = (TGKvCache**)malloc(n * sizeof(TGKvCache*));
        g->old_len = (uint32_t*)malloc(n * sizeof(uint32_t));
        g->ones = (uint32_t*)malloc(n * sizeof(uint32_t));
    }
    if (!g || !table || !g->caches || !g->old_len || !g->ones) {
        free(table);
        tg_kv_group_destroy(g);
        set_err("group: out of host memory");
        return NULL;
    }
    g->n = n;
    g->n_heads = n_heads;
    g->act = act;
    g->prefix = prefix;
    for (uint32_t i = 0; i < n; i++) {
        g->caches[i] = caches[i];
        g->ones[i] = 1;
        table[i] = row_cache(caches[i]);
    }
    if (prefix) table[n] = row_cache(prefix);
    g->device = tg_cuda_kv_device();
    g->table_dev = tg_cuda_kv_group_table(table, n, c0->n_kv_heads, c0->head_dim);
    free(table);
    if (g->table_dev)
        g->scratch = tg_cuda_kv_malloc(tg_cuda_kv_group_scratch_bytes(n, n_heads, c0->head_dim));
    if (!g->table_dev || !g->scratch) {
        set_err("group: %s", tg_cuda_kv_last_error());
        tg_kv_group_destroy(g);
        return NULL;
    }
    return g;
}

void tg_kv_group_destroy(TGKvGroup* g) {
    if (!g) return;
    tg_cuda_kv_free(g->table_dev);
    tg_cuda_kv_free(g->scratch);
    free(g->caches);
    free(g->old_len);
    free(g->ones);
    free(g);
}

int tg_kv_group_truncate(TGKvGroup* g, const uint32_t* len) {
    if (!g || !len) { set_err("null argument"); return 0; }
    for (uint32_t i = 0; i < g->n; i++)
        if (len[i] > g->caches[i]->len) {
            set_err("group: truncate cache %u to %u beyond length %u", i, len[i], g->caches[i]->len);
            return 0;
        }
    for (uint32_t i = 0; i < g->n; i++) g->caches[i]->len = len[i];
    return 1;
}

static int group_call(TGKvGroup* g, const uint32_t* n_new, const void* q, const void* k_new,
                      const void* v_new, void* out, void* stream) {
    if (!g || !n_new || !q || !out) { set_err("null argument"); return 0; }
    if (!k_new != !v_new) { set_err("group: k_new and v_new go together"); return 0; }
    const TGKvCache* c0 = g->caches[0];
    const float mscale = g->prefix ? g->prefix->mscale : c0->mscale;
    if (!(mscale > 0.0f) || !isfinite(mscale)) {
        set_err("group: mscale %g is not a positive number", (double)mscale);
        return 0;
    }
    for (uint32_t i = 0; i < g->n; i++) {
        const TGKvCache* c = g->caches[i];
        if (c->mscale != mscale) { set_err("group: cache %u has another mscale", i); return 0; }
        if (k_new ? (uint64_t)c->len + n_new[i] > c->max_seq : n_new[i] > c->len) {
            if (k_new) set_err("group: capacity exceeded at cache %u", i);
            else set_err("group: %u queries but %u rows in cache %u", n_new[i], c->len, i);
            return 0;
        }
        g->old_len[i] = k_new ? c->len : c->len - n_new[i];
    }
    if (!on_cuda("group")) return 0;
    if (tg_cuda_kv_device() != g->device) {
        set_err("group: made on device %d, called on device %d", g->device, tg_cuda_kv_device());
        return 0;
    }
    TGCudaGroupCall call;
    memset(&call, 0, sizeof(call));
    call.act = g->act;
    call.n_seq = g->n;
    call.n_heads = g->n_heads;
    call.n_kv_heads = c0->n_kv_heads;
    call.head_dim = c0->head_dim;
    call.prefix_len = g->prefix ? g->prefix->len : 0;
    call.table_dev = g->table_dev;
    call.old_len = g->old_len;
    call.n_new = n_new;
    call.q = q;
    call.k_new = k_new;
    call.v_new = v_new;
    call.out = out;
    call.scratch = g->scratch;
    call.scale = (1.0f / sqrtf((float)c0->head_dim)) * mscale;
    if (!tg_cuda_kv_group_attention(&call, stream)) {
        set_err("%s", tg_cuda_kv_last_error());
        return 0;
    }
    if (k_new)
        for (uint32_t i = 0; i < g->n; i++) g->caches[i]->len += n_new[i];
    return 1;
}

int tg_kv_group_decode(TGKvGroup* g, const void* q, const void* k_new, const void* v_new,
                       void* out, void* stream) {
    if (!g) { set_err("null argument"); return 0; }
    return group_call(g, g->ones, q, k_new, v_new, out, stream);
}

int tg_kv_group_prompt(TGKvGroup* g, const uint32_t* n_new, const void* q, const void* k_new,
                       const void* v_new, void* out, void* stream) {
    return group_call(g, n_new, q, k_new, v_new, out, stream);
}

/* ---- row moves ------------------------------------------------------------ */

/* n caches (not NULL) of c0's geometry with rows the kernels can move. */
static int movable(const char* what, TGKvCache* const* v, uint32_t n, const TGKvCache* c0) {
    for (uint32_t i = 0; i < n; i++) {
        if (!v[i]) { set_err("%s: null cache %u", what, i); return 0; }
        if (!same_geometry(c0, v[i])) {
            set_err("%s: cache %u differs in geometry or dtype", what, i);
            return 0;
        }
    }
    if (c0->kv_dim % 8) {
        set_err("%s: kv_dim %u is not a multiple of 8", what, c0->kv_dim);
        return 0;
    }
    return 1;
}

int tg_kv_fork(TGKvCache* const* src, uint32_t n_src, TGKvCache* const* dst, uint32_t fan,
               uint32_t n_rows, void* stream) {
    if (!src || !dst || n_src == 0 || fan == 0 || (uint64_t)n_src * fan > TGKV_GROUP_MAX) {
        set_err("fork: need sources and 1..%d copies in all", TGKV_GROUP_MAX);
        return 0;
    }
    const uint32_t n_dst = n_src * fan;
    if (!src[0]) { set_err("fork: null cache 0"); return 0; }
    if (!movable("fork", src, n_src, src[0]) || !movable("fork", dst, n_dst, src[0])) return 0;
    if (!all_different(dst, n_dst, (const TGKvCache* const*)src, n_src)) {
        set_err("fork: a destination appears twice or is a source");
        return 0;
    }
    for (uint32_t i = 0; i < n_src; i++)
        if (n_rows > src[i]->len) {
            set_err("fork: %u rows of source %u, which has %u", n_rows, i, src[i]->len);
            return 0;
        }
    for (uint32_t i = 0; i < n_dst; i++)
        if (n_rows > dst[i]->max_seq) { set_err("fork: capacity exceeded at copy %u", i); return 0; }
    if (!on_device("fork", src, n_src) || !on_device("fork: copies", dst, n_dst)) return 0;
    TGCudaRowCache s[TGKV_GROUP_MAX], d[TGKV_GROUP_MAX];
    for (uint32_t i = 0; i < n_src; i++) s[i] = row_cache(src[i]);
    for (uint32_t i = 0; i < n_dst; i++) d[i] = row_cache(dst[i]);
    if (!tg_cuda_kv_fork_rows(s, n_src, d, fan, (uint64_t)src[0]->kv_dim * src[0]->esize, n_rows, stream)) {
        set_err("%s", tg_cuda_kv_last_error());
        return 0;
    }
    for (uint32_t i = 0; i < n_dst; i++) dst[i]->len = n_rows;
    return 1;
}

int tg_kv_compact(TGKvCache* const* caches, uint32_t n, const uint32_t* start,
                  const uint32_t* count, uint32_t n_ranges, void* stream) {
    if (!caches || n == 0 || n > TGKV_GROUP_MAX || n_ranges > TGKV_GROUP_MAX ||
        (n_ranges && (!start || !count))) {
        set_err("compact: need 1..%d caches and up to %d ranges", TGKV_GROUP_MAX, TGKV_GROUP_MAX);
        return 0;
    }
    if (!caches[0]) { set_err("compact: null cache 0"); return 0; }
    if (!movable("compact", caches, n, caches[0])) return 0;
    if (!all_different(caches, n, NULL, 0)) { set_err("compact: a cache appears twice"); return 0; }
    for (uint32_t i = 1; i < n; i++)
        if (caches[i]->len != caches[0]->len) {
            set_err("compact: cache %u has %u rows, cache 0 has %u", i, caches[i]->len, caches[0]->len);
            return 0;
        }
    uint64_t end = 0, keep = 0;
    for (uint32_t r = 0; r < n_ranges; r++) {
        if (count[r] == 0 || start[r] < end || (uint64_t)start[r] + count[r] > caches[0]->len) {
            set_err("compact: range %u (%u rows from %u) is empty, out of order or beyond length %u",
                    r, count[r], start[r], caches[0]->len);
            return 0;
        }
        end = (uint64_t)start[r] + count[r];
        keep += count[r];
    }
    if (!on_device("compact", caches, n)) return 0;
    TGCudaRowCache t[TGKV_GROUP_MAX];
    for (uint32_t i = 0; i < n; i++) t[i] = row_cache(caches[i]);
    if (!tg_cuda_kv_compact_rows(t, n, (uint64_t)caches[0]->kv_dim * caches[0]->esize, start, count,
                                 n_ranges, stream)) {
        set_err("%s", tg_cuda_kv_last_error());
        return 0;
    }
    for (uint32_t i = 0; i < n; i++) caches[i]->len = (uint32_t)keep;
    return 1;
}
