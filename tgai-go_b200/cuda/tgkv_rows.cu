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
// it to all fan copies.  12 layers of 2000 bf16 rows of 512 into 5 caches: 50 us,
// 5.9 TB/s.
constexpr int kForkVec = 8;                       // vectors in flight per thread

__global__ void __launch_bounds__(kThreads) fork_kernel(const __grid_constant__ TGKvForkParams p) {
    const uint32_t half = blockIdx.y & 1u, i = blockIdx.y >> 1;
    const uint4* src = reinterpret_cast<const uint4*>(p.src[i].base + half * p.src[i].max_seq * p.row_bytes);
    const uint64_t v0 = (uint64_t)blockIdx.x * (kThreads * kForkVec) + threadIdx.x;
    uint4 r[kForkVec];
#pragma unroll
    for (int u = 0; u < kForkVec; ++u)
        if (v0 + u * kThreads < p.n_vec) r[u] = __ldcs(src + v0 + u * kThreads);
    // the destinations as ordinary memory: through the constant cache each would be a miss of its own
    const TGKvRowCache* to = p.dst + i * p.fan;
    asm volatile("" : "+l"(to));
#pragma unroll 4
    for (uint32_t j = 0; j < p.fan; ++j) {
        const TGKvRowCache c = to[j];
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
// and walks the destination rows in waves: its CTAs read the wave's sources into
// registers, meet at a cluster barrier, then write.  The reads of wave w + 1
// need no order against the writes of waves <= w: their sources lie at or behind
// wave w + 1's own destinations.  So one barrier per wave (every CTA's reads of
// wave w before any CTA's writes of wave w), with the next wave's reads in
// flight across it, and no flags or scratch in memory.  Bound: HBM, 2 * moved
// bytes: 24 caches of 32768 bf16 rows of 512 to 4 + 16384 take 318 us, 5.07 TB/s.
// A thread keeps its column and steps through rows, so that there is no
// division and its place among the ranges only moves on.
constexpr int kMoveRows = 8;                      // rows in flight per thread

__global__ void __launch_bounds__(kThreads, 2) compact_kernel(const __grid_constant__ TGKvCompactParams p) {
    __shared__ uint32_t start[TGKV_MAX_ITEMS], first[TGKV_MAX_ITEMS + 1];
    {
        // side by side through ordinary loads, not one by one through the constant cache
        const uint32_t *s = p.start, *f = p.first;
        asm volatile("" : "+l"(s), "+l"(f));
        for (uint32_t i = threadIdx.x; i < p.n_ranges; i += kThreads) {
            start[i] = s[i];
            first[i] = f[i];
        }
        if (threadIdx.x == 0) first[p.n_ranges] = p.n_keep;
    }
    __syncthreads();
    uint32_t cl;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(cl));
    const uint32_t rank = cluster_ctarank();
    const uint32_t unit = blockIdx.x / cl;        // (cache, half, slice)
    const uint32_t slice = unit % p.n_slices, half = (unit / p.n_slices) & 1u;
    const uint32_t ci = unit / p.n_slices / 2;
    const uint32_t rv = (uint32_t)(p.row_bytes / 16);                     // vectors of a row
    const uint32_t width = (rv + p.n_slices - 1) / p.n_slices;            // of a slice, at most kThreads
    const uint32_t per = kThreads / width;                                // rows side by side
    const uint32_t col = slice * width + threadIdx.x % width, lane_row = threadIdx.x / width;
    const bool mine = lane_row < per && col < rv;
    uint4* mem = reinterpret_cast<uint4*>(p.caches[ci].base + half * p.caches[ci].max_seq * p.row_bytes) + col;
    // wave w of this CTA: rows d0 + w * step + u * per, u < kMoveRows
    const uint32_t rows_cta = per * kMoveRows;
    const uint64_t step = (uint64_t)cl * rows_cta;
    const uint64_t d0 = p.skip + (uint64_t)rank * rows_cta + lane_row;
    const uint32_t waves = (uint32_t)((p.n_keep - p.skip + step - 1) / step);
    uint4 a[kMoveRows];
    uint32_t ri = 0;                              // the range of the last row read
    auto load = [&](uint64_t d) {
        // the range of row d: behind the last one's, most often far behind
        uint32_t hi = p.n_ranges;
        while (hi - ri > 1) {
            const uint32_t mid = (ri + hi) >> 1;
            if (first[mid] <= d) ri = mid;
            else hi = mid;
        }
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u, d += per)
            if (mine && d < p.n_keep) {
                while (first[ri + 1] <= d) ++ri;
                a[u] = __ldcs(mem + ((uint64_t)start[ri] + (d - first[ri])) * rv);
            }
    };
    load(d0);
    for (uint32_t w = 0; w < waves; ++w) {
        uint4 b[kMoveRows];
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) b[u] = a[u];
        __syncwarp();                             // the .aligned cluster barrier wants whole warps
        cluster_arrive();
        const uint64_t d = d0 + w * step;
        if (w + 1 < waves) load(d + step);
        __syncwarp();
        cluster_wait();
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u)
            if (mine && d + (uint64_t)u * per < p.n_keep) mem[(d + (uint64_t)u * per) * rv] = b[u];
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
