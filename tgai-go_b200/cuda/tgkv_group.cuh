// tgkv_group.cuh -- device code shared by tgkv_group.cu and
// tgkv_group_light.cuh: the pieces of a CTA's stretch (tgkv_group_plan.h), TMEM
// access and the launch helper.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdlib.h>

#include "tgkv_group_plan.h"
#include "tgkv_launch.h"
#include "tgkv_ptx.cuh"

namespace tgkv {
namespace group {

constexpr int kRows = TGKV_GROUP_ROWS, kPos = TGKV_GROUP_TILE;
constexpr uint32_t kBlock = 16384;              // 128 rows x 64 bf16: one swizzled box
constexpr int kErrTimeout = 7;
constexpr int kThreads = 384;

__device__ __forceinline__ float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// A table in the parameter block as ordinary memory.  Read as parameters, entries
// would come through the constant cache one after another, each first touch a miss
// that costs as much as a trip to L2 (25 us for a merge over 148 stretches); so the
// threads of a block copy the tables they search into shared memory side by side.
__device__ __forceinline__ const uint32_t* as_memory(const uint32_t* table) {
    asm volatile("" : "+l"(table));
    return table;
}
__device__ __forceinline__ void copy_table(uint32_t* dst, const uint32_t* table, uint32_t n, int tid, int threads) {
    const uint32_t* src = as_memory(table);
    for (uint32_t i = tid; i < n; i += threads) dst[i] = src[i];
}
__device__ __forceinline__ TGKvGroupPos start_of(const TGKvGroupParams& p, int line, uint32_t b) {
    const uint4 s = *reinterpret_cast<const uint4*>(as_memory(p.line[line].start) + 4 * b);
    return TGKvGroupPos{s.x, s.y, s.z, s.w};
}
__device__ __forceinline__ TGKvGroupShape shape_of(const TGKvGroupParams& p, int line, const uint32_t* old_len,
                                                   const uint32_t* tok0) {
    return TGKvGroupShape{p.n_seq, p.n_kv_heads, p.prefix_len, p.share, kRows / (p.n_heads / p.n_kv_heads),
                          p.line[line].item_tokens, 0, old_len, tok0};
}

// The pieces of a CTA's stretch, one after another.  With `most` > 0 an item's
// tiles come in pieces of at most that many (their results add up in a slot).
struct Pieces {
    TGKvGroupPos at, end;
    uint32_t j0, j1;                             // tiles [j0, j1) of the item
    uint32_t nt, first;                          // the item's tiles; where this CTA began with it
    __device__ Pieces(const TGKvGroupShape& s, TGKvGroupPos a, TGKvGroupPos e, uint32_t most) : at(a), end(e) {
        set(s, most);
    }
    __device__ bool more() const { return j0 < j1; }
    __device__ void next(const TGKvGroupShape& s, uint32_t most) {
        const uint32_t stop = tgkv_group_same_item(at, end) ? end.tile : nt;
        if (j1 < stop) {                         // more of the same item
            j0 = j1;
            j1 = most && stop - j0 > most ? j0 + most : stop;
            return;
        }
        if (tgkv_group_same_item(at, end)) { j0 = j1; return; }
        at = tgkv_group_next_item(&s, at);
        set(s, most);
    }

private:
    __device__ void set(const TGKvGroupShape& s, uint32_t most) {
        first = j0 = at.tile;
        nt = at.seq <= s.n_seq ? tgkv_group_item_tiles(&s, at.seq, at.at) : 0;
        const uint32_t stop = tgkv_group_same_item(at, end) ? end.tile : nt;
        j1 = most && stop - j0 > most ? j0 + most : stop;
    }
};

// What an item's tiles see.
struct ItemRows {
    uint32_t npre, prefix_len, own_rows;         // prefix tiles; rows some query of the item sees of each part
    uint32_t tokens;                             // of the item
    __device__ ItemRows(const TGKvGroupShape& s, const Pieces& pc)
        : npre(tgkv_group_prefix_tiles(&s, pc.at.seq)), prefix_len(s.prefix_len),
          own_rows(pc.at.seq ? tgkv_group_own_rows(&s, pc.at.seq, pc.at.at) : 0),
          tokens(min(s.item_tokens, tgkv_group_tokens(&s, pc.at.seq) - pc.at.at * s.item_tokens)) {}
    __device__ bool own(uint32_t j) const { return j >= npre; }
    __device__ uint32_t pos(uint32_t j) const { return (j >= npre ? j - npre : j) * kPos; }
    __device__ uint32_t rows(uint32_t j) const { return j >= npre ? own_rows : prefix_len; }
};

// The sequence of packed token t: the last one whose first token is at or
// before t among those with tokens.
__device__ __forceinline__ uint32_t seq_of(const uint32_t* tok0, uint32_t n_seq, uint32_t t) {
    uint32_t lo = 0, hi = n_seq;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (tok0[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The larger of three; NaN if one is, so that a NaN score reaches the row's maximum
// and with it all its weights.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 16 consecutive columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15])::"memory");
}

// A value of V that is not finite reaches the queries that see its position and no
// other, though 0 x Inf is NaN: among the rows that only some queries of an item see,
// such values are cleared in the tile, and their sum is added to the results of
// those that do see them (cache_non_finite, off the usual path).  Looking for them
// took 2 % of the time of prompts of 2000 tokens, 8 % of ragged ones of up to 1000,
// while it was the softmax threads' work; a warp of its own ahead of them leaves 0 and 3 %.
__device__ __forceinline__ uint32_t non_finite_bits(uint4 v) {                 // 0x80008000: some
    constexpr uint32_t e = 0x7f807f80u, one = 0x00800080u;
    return ((v.x & e) + one) | ((v.y & e) + one) | ((v.z & e) + one) | ((v.w & e) + one);
}
__device__ __forceinline__ uint32_t clear_non_finite(uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
    return w;
}
// Rows [lo, rows) of a V tile in shared memory, HD / 64 boxes, by THREADS threads: what
// is not finite is cleared, and *flag becomes 1 if there was any.  (A call: the code of a
// decode step, which has no such rows, stays short.)
template <int HD, int THREADS>
__device__ __noinline__ void clear_non_finite(unsigned char* tile, uint32_t lo, uint32_t rows, int r, volatile uint32_t* flag) {
    uint4* at = reinterpret_cast<uint4*>(tile) + (r & 7);
    const uint32_t y0 = lo + ((uint32_t)r >> 3), y1 = min(rows, (uint32_t)kPos);
    uint32_t bits = 0;
#pragma unroll 4
    for (uint32_t y = y0; y < y1; y += THREADS / 8)
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) bits |= non_finite_bits(at[c * (kBlock / 16) + y * 8]);
    if (bits & 0x80008000u) {
        *flag = 1;
#pragma unroll 1
        for (uint32_t y = y0; y < y1; y += THREADS / 8)
#pragma unroll 1
            for (int c = 0; c < HD / 64; ++c) {
                uint4* x = at + c * (kBlock / 16) + y * 8;
                const uint4 v = *x;
                *x = make_uint4(clear_non_finite(v.x), clear_non_finite(v.y), clear_non_finite(v.z), clear_non_finite(v.w));
            }
    }
}
// Rows [rows, end) of the tile cleared whole, rows [lo, rows) of what is not finite.
template <int HD, int THREADS>
__device__ __forceinline__ void clear_unseen(unsigned char* tile, uint32_t lo, uint32_t rows, uint32_t end, int r,
                                             volatile uint32_t* flag) {
    for (uint32_t y = rows + ((uint32_t)r >> 3); y < end; y += THREADS / 8)
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
            *reinterpret_cast<uint4*>(tile + c * kBlock + y * 128 + (r & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
    if (lo < rows) clear_non_finite<HD, THREADS>(tile, lo, rows, r, flag);
}
// The sum of the values of V's column `col` that are not finite, rows [a, e) of a cache.
__device__ __noinline__ float cache_non_finite(const TGKvRowCache* cache, uint32_t kv_dim, uint32_t col, uint32_t a, uint32_t e) {
    const uint16_t* v = reinterpret_cast<const uint16_t*>(cache->base) + (cache->max_seq + a) * kv_dim + col;
    float s = 0.f;
    for (; a < e; ++a, v += kv_dim) {
        const uint32_t b = __ldcg(v);
        if ((b & 0x7f80u) == 0x7f80u) s += lo_f(b);
    }
    return s;
}

// 8 elements of a new row as the cache stores them.
__device__ __forceinline__ uint4 row_part(const float* src) {
    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
    return make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
}
__device__ __forceinline__ uint4 row_part(const uint16_t* src) { return *reinterpret_cast<const uint4*>(src); }

// Programmatic dependent launch (TGKV_PDL=0 turns it off): each kernel waits
// (griddepcontrol.wait) before its first access to global memory.
template <typename K>
cudaError_t launch_pdl(K kernel, dim3 grid, int threads, uint32_t smem, cudaStream_t st, const TGKvGroupParams* p) {
    static const bool pdl = [] {
        const char* e = getenv("TGKV_PDL");
        return !(e && e[0] == '0');
    }();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, *p);
}

// The kernel's shared memory size, once per device.
template <typename K>
cudaError_t allow_smem(K kernel, uint32_t bytes, bool (&done)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (done[dev]) return cudaSuccess;           // benign race: same value
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    done[dev] = e == cudaSuccess;
    return e;
}

}  // namespace group
}  // namespace tgkv
