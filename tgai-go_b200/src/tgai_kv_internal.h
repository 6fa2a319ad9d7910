/* tgai_kv_internal.h -- the cache object, shared by the host C files that
 * implement include/tgai_kv_cache.h and include/tgai_kv_group.h. */
#ifndef TGAI_KV_INTERNAL_H
#define TGAI_KV_INTERNAL_H

#include "tgai_backend.h"
#include "tgai_kv_cache.h"

#include <stddef.h>

struct TGKvCache {
    uint32_t max_seq, n_kv_heads, head_dim, kv_dim;
    int      dtype;
    uint32_t esize;
    int      device;              /* that was current at create: dev lies there */
    size_t   bytes;               /* 2 * max_seq * kv_dim * esize */
    void*    dev;                 /* device address of the buffer */
    float*   host;                /* always NULL (not mappable) */
    uint32_t len;
    TGBackend* be;                /* backend that owns dev */
    void*    scratch;             /* split-sequence partials */
    uint64_t scratch_bytes;
    uint32_t* counters;
    uint64_t counter_slots;
    float*   staging;             /* device staging of host rows (bf16 append) */
    size_t   staging_bytes;
    void*    tmap;                /* TMA tensor map of dev (NULL: no attention kernel) */
    void*    tmap_sw;             /* swizzled map for the tensor-core suffix kernel, or NULL */
    uint32_t* npos;               /* host item table for attention */
    uint32_t npos_cap;
    float    mscale;              /* YaRN temperature on the 1/sqrt(head_dim) scale */
};

/* Sets the calling thread's tg_kv_last_error(). */
__attribute__((visibility("hidden"), format(printf, 1, 2)))
void tgkv_kv_set_err(const char* fmt, ...);

#endif /* TGAI_KV_INTERNAL_H */
