// tgkv_rows.cu -- moving rows of KV caches: fork (the first rows of a cache
// copied into several others) and in-place compaction (ranges of positions
// moved to the front).  Pure data movement: K and V rows as 16-byte vectors,
// any dtype.
#include <cuda_runtime.h>
#include <stdint.h>

#include "tgkv_launch.h"
#include "tgkv_ptx.cuh"

namespace tgkv {
namespace rows {

constexpr int kThreads = 256;

// ------------------------------------------------------------------ fork
// A cache's first n_rows rows of K (or V) are one contiguous block of
// n_vec 16-byte vectors, so a fork copies 2 blocks per source.  Bound: HBM,
// (1 + fan) * block bytes; each CTA reads a piece of a block once and writes
// it to all fan copies.
constexpr int kForkVec = 8;                       // vectors in flight per thread

__global__ void __launch_bounds__(kThreads) fork_kernel(const __grid_constant__ TGKvForkParams p) {
    const uint32_t half = blockIdx.y & 1u, i = blockIdx.y >> 1;
    const uint4* src = reinterpret_cast<const uint4*>(p.src[i].base + half * p.src[i].max_seq * p.row_bytes);
    const uint64_t v0 = (uint64_t)blockIdx.x * (kThreads * kForkVec) + threadIdx.x;
    uint4 r[kForkVec];
#pragma unroll
    for (int u = 0; u < kForkVec; ++u)
        if (v0 + u * kThreads < p.n_vec) r[u] = __ldcs(src + v0 + u * kThreads);
    for (uint32_t j = 0; j < p.fan; ++j) {
        const TGKvRowCache c = p.dst[i * p.fan + j];
        uint4* dst = reinterpret_cast<uint4*>(c.base + half * c.max_seq * p.row_bytes);
#pragma unroll
        for (int u = 0; u < kForkVec; ++u)
            if (v0 + u * kThreads < p.n_vec) dst[v0 + u * kThreads] = r[u];
    }
}

// ------------------------------------------------------------- compaction
// Destination row d takes source row s(d) >= d, s strictly increasing.  In
// place, a row must have been read before the row that lands on it is
// written.  One cluster owns a column slice of one half (K or V) of one cache
// and walks the destination rows in waves of W rows: its CTAs read the
// wave's sources into registers, meet at a cluster barrier, then write.  The
// reads of wave w + 1 need no order against the writes of waves <= w: their
// sources lie at or behind wave w + 1's own destinations.  So one barrier per
// wave (every CTA's reads of wave w before any CTA's writes of wave w), with
// the next wave's reads in flight across it, and no flags or scratch in
// memory.  Bound: HBM, 2 * moved bytes.
constexpr int kMoveVec = 8;

__device__ __forceinline__ uint64_t source_row(const TGKvCompactParams& p, uint32_t d) {
    uint32_t lo = 0, hi = p.n_ranges;             // the last range starting at or before d
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (p.first[mid] <= d) lo = mid;
        else hi = mid;
    }
    return (uint64_t)p.start[lo] + (d - p.first[lo]);
}

__global__ void __launch_bounds__(kThreads) compact_kernel(const __grid_constant__ TGKvCompactParams p) {
    uint32_t cl;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(cl));
    const uint32_t rank = cluster_ctarank();
    const uint32_t unit = blockIdx.x / cl;        // (cache, half, slice)
    const uint32_t slice = unit % p.n_slices, half = (unit / p.n_slices) & 1u;
    const uint32_t ci = unit / p.n_slices / 2;
    const uint64_t rv = p.row_bytes / 16;         // vectors of a row
    const uint32_t sv = (uint32_t)(rv / p.n_slices);
    uint4* mem = reinterpret_cast<uint4*>(p.caches[ci].base + half * p.caches[ci].max_seq * p.row_bytes) +
                 (uint64_t)slice * sv;
    // vector v of the slice's destination vectors: row v / sv, column v % sv
    const uint64_t total = (uint64_t)(p.n_keep - p.skip) * sv;
    const uint64_t per = (uint64_t)cl * kThreads * kMoveVec;
    const uint64_t mine = (uint64_t)rank * kThreads * kMoveVec + threadIdx.x;
    uint4 a[kMoveVec];
    auto load = [&](uint64_t w) {
#pragma unroll
        for (int u = 0; u < kMoveVec; ++u) {
            const uint64_t v = w * per + mine + (uint64_t)u * kThreads;
            if (v < total) {
                const uint32_t d = p.skip + (uint32_t)(v / sv);
                a[u] = mem[source_row(p, d) * rv + v % sv];
            }
        }
    };
    auto store = [&](uint64_t w, const uint4 (&x)[kMoveVec]) {
#pragma unroll
        for (int u = 0; u < kMoveVec; ++u) {
            const uint64_t v = w * per + mine + (uint64_t)u * kThreads;
            if (v < total) mem[(uint64_t)(p.skip + (uint32_t)(v / sv)) * rv + v % sv] = x[u];
        }
    };
    const uint64_t waves = (total + per - 1) / per;
    load(0);
    for (uint64_t w = 0; w < waves; ++w) {
        uint4 b[kMoveVec];
#pragma unroll
        for (int u = 0; u < kMoveVec; ++u) b[u] = a[u];
        cluster_arrive();
        if (w + 1 < waves) load(w + 1);
        cluster_wait();
        store(w, b);
    }
}

}  // namespace rows
}  // namespace tgkv

extern "C" int tgkv_launch_fork(const TGKvForkParams* p, void* stream) {
    using namespace tgkv::rows;
    const uint64_t per = kThreads * kForkVec;
    const uint64_t gx = (p->n_vec + per - 1) / per;
    if (gx == 0 || gx > 0x7fffffffull || p->n_src == 0 || p->n_src > 32767) return (int)cudaErrorInvalidValue;
    fork_kernel<<<dim3((unsigned)gx, 2 * p->n_src), kThreads, 0, (cudaStream_t)stream>>>(*p);
    return (int)cudaGetLastError();
}

extern "C" int tgkv_launch_compact(const TGKvCompactParams* p, uint32_t cluster, void* stream) {
    using namespace tgkv::rows;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p->n_caches * 2 * p->n_slices * cluster);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, compact_kernel, *p);
}
