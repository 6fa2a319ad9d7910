// tgkv_group.cu -- attention of several sequences of one layer that may share
// a prefix cache: token t of sequence i attends the prefix's positions [0, P)
// and its own cache's positions [0, old_i + t].  q head h reads KV head
// h * n_kv_heads / n_heads; out = softmax(q K^T * scale) V over both parts.
//
// group_kernel: persistent CTAs, one per SM, each with its stretch of the line
// of K/V tiles that tgkv_group_plan.h cuts.  A piece is a row tile (128 query
// rows of one KV head, one per TMEM lane) against a run of 128-position tiles,
// in one pass: S = Q K^T, running maximum and sum in the log2 domain, O += P V.
// Inside a CTA (320 threads):
//   warps 0-7  softmax: TMEM lane r is row r, shared by warps r/32 and r/32 + 4,
//              which take positions [0,64) and [64,128) of a tile; they exchange
//              the tile's row maximum through shared memory.  Per piece they
//              write Q into TMEM; per tile they read S, mask, exponentiate and
//              write P over S; at the end they read O and write the rows, or
//              leave them as a partial;
//   warp 8     TMA: K and V tiles (64-dim boxes, 128-byte swizzle) into two rings,
//              running ahead over the CTA's whole stretch;
//   warp 9     the MMAs (one lane), A operand from TMEM: S into one of two
//              buffers, so that the next tile's S is made while the softmax works
//              on this one; PV with V as an MN-major operand.
// TERMS is the number of bf16 terms of q and P: 1 with bf16 activations (q is
// exact, P is rounded once, 2^-8 of a weight, as the output itself is), 2 with
// fp32 ones (hi + lo, 16 mantissa bits; three terms of P would not fit the
// columns S leaves free).  Scores, maxima, sums and O are fp32.
// TMEM columns: S/P [0,128) and [128,256), O [256,256+HD), Q [384,384+TERMS*HD/2).
//
// group_merge_kernel joins the partials of rows whose tiles more than one
// piece attended: no atomics, always in the same order.
//
// Every mbarrier wait is bounded; one that runs out sets the device error word
// and the CTA ends without further waits on its own data.
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
constexpr int kSoftmaxThreads = 256, kThreads = 320;
constexpr int kTmaWarp = 8, kMmaWarp = 9;
constexpr uint32_t kBlock = 16384;              // 128 positions x 64 dims bf16: one box
constexpr uint32_t TM_S = 0, TM_O = 256, TM_Q = 384, TM_COLS = 512;
constexpr int kErrTimeout = 7;

template <int HD>
struct Cfg {
    static constexpr uint32_t kTile = (uint32_t)(HD / 64) * kBlock;    // one K or V tile
    static constexpr int kStages = HD == 128 ? 3 : 6;                  // per ring: 192 KB in all
    static constexpr uint32_t OFF_K = 0, OFF_V = kStages * kTile;
    static constexpr uint32_t OFF_BAR = 2 * kStages * kTile;
    static constexpr int B_KFULL = 0, B_KEMPTY = kStages, B_VFULL = 2 * kStages, B_VEMPTY = 3 * kStages;
    static constexpr int B_SFULL = 4 * kStages;      // [2] S of the tile in the buffer is in TMEM
    static constexpr int B_PFULL = B_SFULL + 2;      // [2] its P is written (256 arrivals)
    static constexpr int B_PVDONE = B_PFULL + 2;     // one phase per tile: its PV is complete
    static constexpr int B_QREADY = B_PVDONE + 1;    // one phase per piece: Q is in TMEM (256)
    static constexpr uint32_t OFF_X = OFF_BAR + 32 * 8;                // [2][2][128] maxima
    static constexpr uint32_t OFF_L = OFF_X + 4 * kRows * 4;           // [2][128] sums
    static constexpr uint32_t OFF_SLOT = OFF_L + 2 * kRows * 4;
    static constexpr uint32_t SMEM = OFF_SLOT + 16 + 1024;             // slack to align the base
    static_assert(B_QREADY < 32 && SMEM <= 232448, "shared memory per CTA");
};

__device__ __forceinline__ void pair_sync(int quarter) {
    asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
}
__device__ __forceinline__ float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

__device__ __forceinline__ TGKvGroupPos start_of(const TGKvGroupParams& p, uint32_t b) {
    return TGKvGroupPos{p.start[4 * b], p.start[4 * b + 1], p.start[4 * b + 2], p.start[4 * b + 3]};
}

// The pieces of a CTA's stretch, one after another.
struct Pieces {
    TGKvGroupPos at, end;
    uint32_t j0, j1, nt;                         // tiles [j0, j1) of the item's nt
    __device__ Pieces(const TGKvGroupParams& p, uint32_t cta) : at(start_of(p, cta)), end(start_of(p, cta + 1)) {
        set(p);
    }
    __device__ bool more() const { return j0 < j1; }
    __device__ void next(const TGKvGroupParams& p) {
        if (tgkv_group_same_item(at, end)) { j0 = j1; return; }
        at = tgkv_group_next_item(&p, at);
        set(p);
    }

private:
    __device__ void set(const TGKvGroupParams& p) {
        const bool last = tgkv_group_same_item(at, end);
        j0 = at.tile;
        nt = at.seq <= p.n_seq ? tgkv_group_item_tiles(&p, at.seq, at.rt) : 0;
        j1 = last ? end.tile : nt;
    }
};

// The sequence of packed token t: the last one whose first token is at or
// before t among those with tokens.
__device__ __forceinline__ uint32_t seq_of(const TGKvGroupParams& p, uint32_t t) {
    uint32_t lo = 0, hi = p.n_seq;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (p.tok0[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The packed rows of k_new / v_new into their caches, 8 elements per thread.
template <typename T>
__global__ void __launch_bounds__(256) group_append_kernel(const __grid_constant__ TGKvGroupParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t kv_dim = p.n_kv_heads * p.head_dim, vec = kv_dim / 8;
    const uint64_t x = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (x >= (uint64_t)p.tok0[p.n_seq] * vec) return;
    const uint32_t t = (uint32_t)(x / vec), e = (uint32_t)(x % vec) * 8, i = seq_of(p, t);
    const T* src = reinterpret_cast<const T*>(blockIdx.y ? p.v_new : p.k_new) + (uint64_t)t * kv_dim + e;
    const TGKvRowCache c = p.table[i];
    uint16_t* dst = reinterpret_cast<uint16_t*>(c.base) +
                    ((uint64_t)blockIdx.y * c.max_seq + p.old_len[i] + (t - p.tok0[i])) * kv_dim + e;
    uint4 w;
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
        w = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
    } else {
        w = *reinterpret_cast<const uint4*>(src);
    }
    *reinterpret_cast<uint4*>(dst) = w;
    // read by the attention's TMA loads
    asm volatile("fence.proxy.async.global;" ::: "memory");
}

// 32 or 16 32-bit TMEM columns from registers.
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&w)[32]) { tmem_st32(addr, w); }
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&w)[16]) { tmem_st16(addr, w); }

// This thread's HD / 2 head dims of its query row, as bf16 words (two dims
// each) into TMEM: term t at columns TM_Q + t * HD / 2.
template <typename T, int HD, int TERMS>
__device__ __forceinline__ void load_q(const TGKvGroupParams& p, bool valid, uint64_t row, int hf, uint32_t taddr) {
    constexpr int W = HD / 4;                    // words of half a row
    uint32_t w[TERMS][W];
    const T* src = reinterpret_cast<const T*>(p.q) + row * HD + hf * (HD / 2);
    if constexpr (TERMS == 1) {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const uint4 x = valid ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
            w[0][4 * i] = x.x; w[0][4 * i + 1] = x.y; w[0][4 * i + 2] = x.z; w[0][4 * i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
            const float4 x = valid ? reinterpret_cast<const float4*>(src)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
            const uint32_t h0 = cvt_bf16x2(x.x, x.y), h1 = cvt_bf16x2(x.z, x.w);
            w[0][2 * i] = h0;
            w[0][2 * i + 1] = h1;
            w[TERMS - 1][2 * i] = cvt_bf16x2(x.x - lo_f(h0), x.y - hi_f(h0));
            w[TERMS - 1][2 * i + 1] = cvt_bf16x2(x.z - lo_f(h1), x.w - hi_f(h1));
        }
    }
#pragma unroll
    for (int t = 0; t < TERMS; ++t) tmem_st(taddr + TM_Q + t * (HD / 2) + hf * W, w[t]);
}

// P = 2^(s * scale - msc) of 32 positions, packed as bf16 words: hi (and, with two
// terms, the rounding residuals lo); the fp32 values add up in l.  Positions at or
// behind lim get 0.
template <int TERMS, bool MASK>
__device__ __forceinline__ void exp32(const uint32_t (&v)[32], float scale, float msc, int lim, float2& l,
                                      uint32_t* ph, uint32_t* pl) {
    const float2 sc = make_float2(scale, scale), nm = make_float2(-msc, -msc);
#pragma unroll
    for (int c = 0; c < 16; ++c) {
        const float2 d = __ffma2_rn(make_float2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), sc, nm);
        float p0 = ex2_approx(d.x), p1 = ex2_approx(d.y);
        if (MASK) {
            p0 = 2 * c < lim ? p0 : 0.f;
            p1 = 2 * c + 1 < lim ? p1 : 0.f;
        }
        const float2 pp = make_float2(p0, p1);
        l = __fadd2_rn(l, pp);
        ph[c] = cvt_bf16x2(p0, p1);
        if (TERMS == 2) {
            const float2 r = __ffma2_rn(make_float2(lo_f(ph[c]), hi_f(ph[c])), make_float2(-1.f, -1.f), pp);
            pl[c] = cvt_bf16x2(r.x, r.y);
        }
    }
}

template <bool MASK>
__device__ __forceinline__ float max32(const uint32_t (&v)[32], int lim) {
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = -INFINITY;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const float x = __uint_as_float(v[i]);
        a[i & 7] = fmaxf(a[i & 7], (!MASK || i < lim) ? x : -INFINITY);
    }
#pragma unroll
    for (int w = 4; w >= 1; w >>= 1)
#pragma unroll
        for (int i = 0; i < w; ++i) a[i] = fmaxf(a[i], a[i + w]);
    return a[0];
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) group_kernel(const __grid_constant__ TGKvGroupParams p) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
    using C = Cfg<HD>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_addr(base);
    uint64_t* bar = reinterpret_cast<uint64_t*>(base + C::OFF_BAR);
    uint32_t* tslot = reinterpret_cast<uint32_t*>(base + C::OFF_SLOT);
    float* sm_x = reinterpret_cast<float*>(base + C::OFF_X);
    float* sm_l = reinterpret_cast<float*>(base + C::OFF_L);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&bar[C::B_KFULL + i], 1);
            mbar_init(&bar[C::B_KEMPTY + i], 1);
            mbar_init(&bar[C::B_VFULL + i], 1);
            mbar_init(&bar[C::B_VEMPTY + i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar[C::B_SFULL + i], 1);
            mbar_init(&bar[C::B_PFULL + i], kSoftmaxThreads);
        }
        mbar_init(&bar[C::B_PVDONE], 1);
        mbar_init(&bar[C::B_QREADY], kSoftmaxThreads);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        tmem_alloc(tslot, TM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;
    const uint32_t G = p.n_heads / p.n_kv_heads, tpt = kRows / G;
    const uint32_t total_rows = p.tok0[p.n_seq] * p.n_heads;
    // Everything above overlaps the previous kernel on the stream.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    Pieces pc(p, blockIdx.x);
    if (warp == kTmaWarp) {
        if (lane == 0) {
            uint32_t n = 0;                      // tiles issued
            bool ok = true;
            for (; ok && pc.more(); pc.next(p)) {
                const uint32_t npre = tgkv_group_prefix_tiles(&p, pc.at.seq);
                const int x = (int)(pc.at.kvh * HD);
                for (uint32_t j = pc.j0; j < pc.j1; ++j, ++n) {
                    const bool own = j >= npre;
                    const uint64_t map = p.tmaps + 128ull * (own ? pc.at.seq - 1 : p.n_seq);
                    const int y = (int)((own ? j - npre : j) * kPos);
                    const uint32_t s = n % C::kStages, ph = (n / C::kStages - 1) & 1u;
                    if (n >= C::kStages && !(ok = mbar_wait(&bar[C::B_KEMPTY + s], ph))) break;
                    mbar_arrive_expect_tx(&bar[C::B_KFULL + s], C::kTile);
                    for (int b = 0; b < HD / 64; ++b)
                        tma_load_3d(base + C::OFF_K + s * C::kTile + b * kBlock, map, x + 64 * b, y, 0,
                                    &bar[C::B_KFULL + s]);
                    if (n >= C::kStages && !mbar_wait(&bar[C::B_VEMPTY + s], ph)) {
                        // the K copy just issued lands before the CTA ends
                        mbar_wait(&bar[C::B_KFULL + s], (n / C::kStages) & 1u);
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(&bar[C::B_VFULL + s], C::kTile);
                    for (int b = 0; b < HD / 64; ++b)
                        tma_load_3d(base + C::OFF_V + s * C::kTile + b * kBlock, map, x + 64 * b, y, 1,
                                    &bar[C::B_VFULL + s]);
                }
            }
            if (!ok) atomicExch(p.err, kErrTimeout);
            // every copy has landed before the CTA may end (at once in a normal run)
            for (uint32_t i = n > C::kStages ? n - C::kStages : 0; i < n; ++i) {
                const uint32_t s = i % C::kStages, ph = (i / C::kStages) & 1u;
                if (!mbar_wait(&bar[C::B_KFULL + s], ph) || !mbar_wait(&bar[C::B_VFULL + s], ph))
                    atomicExch(p.err, kErrTimeout);
            }
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        if (lane == 0) {
            constexpr uint32_t id_s = umma_idesc_bf16(kRows, kPos, 0, 0);
            constexpr uint32_t id_pv = umma_idesc_bf16(kRows, HD, 0, 1);
            // S of tile n into buffer n % 2: head dims 16 ks .. +15 of Q term t are the 8
            // columns at t * HD / 2 + 8 ks; K is K-major
            auto issue_s = [&](uint32_t n) -> bool {
                const uint32_t s = n % C::kStages, b = n & 1u;
                if (!mbar_wait(&bar[C::B_KFULL + s], (n / C::kStages) & 1u)) return false;
                tc_fence_after();
                const uint64_t kd = umma_desc_sw128(sbase + C::OFF_K + s * C::kTile, 16, 1024);
#pragma unroll
                for (uint32_t i = 0; i < TERMS * (HD / 16); ++i) {
                    const uint32_t t = i / (HD / 16), ks = i % (HD / 16);
                    const uint32_t bo = (ks >> 2) * kBlock + (ks & 3u) * 32u;
                    umma_ts(tmem + TM_S + b * 128u, tmem + TM_Q + t * (HD / 2) + ks * 8u, kd + (bo >> 4), id_s, i != 0);
                }
                umma_commit(&bar[C::B_KEMPTY + s]);
                umma_commit(&bar[C::B_SFULL + b]);
                return true;
            };
            uint32_t n = 0, it = 0;
            bool ok = true;
            for (; ok && pc.more(); pc.next(p), ++it) {
                const uint32_t end = n + (pc.j1 - pc.j0), first = n;
                ok = mbar_wait(&bar[C::B_QREADY], it & 1u);
                tc_fence_after();
                ok = ok && issue_s(n);
                if (n + 1 < end) ok = ok && issue_s(n + 1);
                for (; ok && n < end; ++n) {
                    const uint32_t s = n % C::kStages, b = n & 1u;
                    ok = mbar_wait(&bar[C::B_PFULL + b], (n >> 1) & 1u) &&
                         mbar_wait(&bar[C::B_VFULL + s], (n / C::kStages) & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    // P of positions 16 kk .. +15: 8 columns of half kk / 4, which holds its hi
                    // words first and its lo words 32 columns behind.  V is MN-major: 64-dim
                    // blocks 16 KB apart, 8-position groups 1 KB apart.
                    const uint64_t vd = umma_desc_sw128(sbase + C::OFF_V + s * C::kTile, kBlock, 1024);
#pragma unroll
                    for (uint32_t i = 0; i < TERMS * 8; ++i) {
                        const uint32_t t = i >> 3, kk = i & 7u;
                        const uint32_t a = tmem + TM_S + b * 128u + (kk >> 2) * 64u + t * 32u + (kk & 3u) * 8u;
                        umma_ts(tmem + TM_O, a, vd + ((kk * 16u * 128u) >> 4), id_pv, n != first || i != 0);
                    }
                    umma_commit(&bar[C::B_VEMPTY + s]);
                    umma_commit(&bar[C::B_PVDONE]);
                    if (n + 2 < end) {
                        // S of tile n + 2 goes where PV of tile n reads P
                        ok = mbar_wait(&bar[C::B_PVDONE], n & 1u);
                        tc_fence_after();
                        ok = ok && issue_s(n + 2);
                    }
                }
            }
            if (!ok) atomicExch(p.err, kErrTimeout);
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, hf = warp >> 2, r = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const float scale = p.qscale;
        const uint32_t tok = (uint32_t)r / G, sub = (uint32_t)r % G;
        uint32_t n = 0;
        bool ok = true;
        // Both warps of a pair meet at a named barrier every tile, so neither
        // leaves early: after a failed wait a warp only keeps the barrier count.
        for (; pc.more(); pc.next(p)) {
            const uint32_t seq = pc.at.seq, npre = tgkv_group_prefix_tiles(&p, seq);
            const uint32_t t0 = pc.at.rt * tpt, ntok = min(tpt, tgkv_group_tokens(&p, seq) - t0);
            const uint32_t own_rows = seq ? tgkv_group_own_rows(&p, seq, pc.at.rt) : 0;
            const uint32_t own_min = seq ? p.old_len[seq - 1] + t0 + 1 : 0;      // rows its first token sees
            const bool valid = tok < ntok;
            const uint64_t row = (uint64_t)((seq ? p.tok0[seq - 1] : 0) + t0 + tok) * p.n_heads + pc.at.kvh * G + sub;
            load_q<T, HD, TERMS>(p, valid, row, hf, lanes);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bar[C::B_QREADY]);

            float m = -INFINITY;                 // running maximum of the raw scores
            float2 l2 = make_float2(0.f, 0.f);
            for (uint32_t j = pc.j0; j < pc.j1; ++j, ++n) {
                const uint32_t b = n & 1u, s = n % C::kStages;
                const bool own = j >= npre;
                const uint32_t pos = (own ? j - npre : j) * kPos;
                const uint32_t rows = own ? own_rows : p.prefix_len;             // rows some query of the tile sees
                const bool mask = pos + kPos > (own ? own_min : p.prefix_len);
                const int lim = (int)((own ? own_min + min(tok, ntok - 1) : p.prefix_len) - pos) - hf * 64;
                const uint32_t sp = lanes + TM_S + b * 128u + (uint32_t)hf * 64u;
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_SFULL + b], (n >> 1) & 1u));
                if (ok) tc_fence_after();
                if (ok && pos + kPos > rows && hf == 0) {
                    // V rows that no query of this tile sees may hold anything; P is 0 there, but
                    // 0 * Inf is NaN, so they are cleared before PV reads them
                    ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_VFULL + s], (n / C::kStages) & 1u));
                    if (ok && pos + (uint32_t)r >= rows)
#pragma unroll
                        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                *reinterpret_cast<uint4*>(base + C::OFF_V + s * C::kTile + c * kBlock + r * 128 +
                                                          q * 16) = make_uint4(0u, 0u, 0u, 0u);
                    fence_proxy_async_smem();
                }
                uint32_t va[32], vb[32];
                float tm = -INFINITY;
                if (ok) {
                    tmem_ld32(sp, va);
                    tmem_ld32(sp + 32, vb);
                    tmem_wait_ld(va, vb);
                    tm = mask ? fmaxf(max32<true>(va, lim), max32<true>(vb, lim - 32))
                              : fmaxf(max32<false>(va, 0), max32<false>(vb, 0));
                }
                float* x = sm_x + b * 2 * kRows;
                x[hf * kRows + r] = tm;
                pair_sync(quarter);
                tm = fmaxf(tm, x[(hf ^ 1) * kRows + r]);
                if (ok) {
                    // the running maximum moves only when exceeded by more than 2^8
                    const bool grow = (tm - m) * scale > 8.f;
                    float alpha = 1.f;
                    if (grow) {
                        alpha = m == -INFINITY ? 0.f : ex2_approx((m - tm) * scale);
                        m = tm;
                        l2.x *= alpha;
                        l2.y *= alpha;
                    }
                    if (j > pc.j0 && __any_sync(0xffffffffu, grow)) {
                        ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_PVDONE], (n - 1) & 1u));
                        if (ok) {
                            tc_fence_after();
#pragma unroll
                            for (int c = 0; c < HD / 64; ++c) {
                                uint32_t o[32];
                                const uint32_t oc = lanes + TM_O + (uint32_t)hf * (HD / 2) + c * 32;
                                tmem_ld32(oc, o);
                                tmem_wait_ld(o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                tmem_st32(oc, o);
                            }
                        }
                    }
                }
                if (ok) {
                    const float msc = m == -INFINITY ? 0.f : m * scale;
                    uint32_t ph[32], pl[32];
                    if (mask) {
                        exp32<TERMS, true>(va, scale, msc, lim, l2, ph, pl);
                        exp32<TERMS, true>(vb, scale, msc, lim - 32, l2, ph + 16, pl + 16);
                    } else {
                        exp32<TERMS, false>(va, scale, msc, 0, l2, ph, pl);
                        exp32<TERMS, false>(vb, scale, msc, 0, l2, ph + 16, pl + 16);
                    }
                    tmem_st32(sp, ph);
                    if (TERMS == 2) tmem_st32(sp + 32, pl);
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&bar[C::B_PFULL + b]);
            }
            // the rows' sums over both halves, and O once the last PV is complete
            sm_l[hf * kRows + r] = l2.x + l2.y;
            pair_sync(quarter);
            const float l = sm_l[r] + sm_l[kRows + r];
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_PVDONE], (n - 1) & 1u));
            if (ok) tc_fence_after();
            const bool whole = pc.j0 == 0 && pc.j1 == pc.nt && !p.share;
            uint64_t slot;
            if (pc.j0 > 0 || !p.share) slot = (uint64_t)p.cta_rows + 256u * blockIdx.x + (pc.j0 > 0 ? 0u : 128u) + r;
            else slot = (seq ? total_rows : 0u) + row;
            const float inv = 1.f / l;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                uint32_t o[32];
                if (ok) {
                    tmem_ld32(lanes + TM_O + (uint32_t)hf * (HD / 2) + c * 32, o);
                    tmem_wait_ld(o);
                }
                if (!ok || !valid) continue;
                const uint32_t col = (uint32_t)hf * (HD / 2) + c * 32;
                if (!whole) {
                    uint4* dst = reinterpret_cast<uint4*>(p.part_o + slot * HD + col);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                } else if constexpr (TERMS == 2) {
                    float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + row * HD + col);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        dst[i] = make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv,
                                             __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
                } else {
                    uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + row * HD + col);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            w[k] = cvt_bf16x2(__uint_as_float(o[8 * i + 2 * k]) * inv,
                                              __uint_as_float(o[8 * i + 2 * k + 1]) * inv);
                        dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            if (ok && valid && !whole && hf == 0)
                *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m * scale, l);
        }
        if (!ok && lane == 0) atomicExch(p.err, kErrTimeout);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, TM_COLS);
    }
}

// ------------------------------------------------------------------ merge
// A row's result from its partials (o, m, l): sum 2^(m - M) o / sum 2^(m - M) l.
// One warp per query row, HD / 32 dims per lane.
template <int HD>
struct Acc {
    static constexpr int D = HD / 32;
    float o[D], m, l;
    __device__ Acc() : m(-INFINITY), l(0.f) {
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] = 0.f;
    }
    __device__ void add(const TGKvGroupParams& p, uint64_t slot, int lane) {
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot * 2);
        float x[D];
        if constexpr (D == 4) {
            const float4 v = *reinterpret_cast<const float4*>(p.part_o + slot * HD + lane * 4);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
            const float2 v = *reinterpret_cast<const float2*>(p.part_o + slot * HD + lane * 2);
            x[0] = v.x; x[1] = v.y;
        }
        if (ml.x == -INFINITY) return;           // no position of that part was visible to the row
        const float M = fmaxf(m, ml.x), a = m == -INFINITY ? 0.f : ex2_approx(m - M), b = ex2_approx(ml.x - M);
        l = l * a + ml.y * b;
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] = o[d] * a + x[d] * b;
        m = M;
    }
    template <typename T>
    __device__ void store(const TGKvGroupParams& p, uint64_t row, int lane) const {
        const float inv = 1.f / l;
        T* dst = reinterpret_cast<T*>(p.out) + row * HD + lane * D;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int d = 0; d < D; d += 2) *reinterpret_cast<float2*>(dst + d) = make_float2(o[d] * inv, o[d + 1] * inv);
        } else {
#pragma unroll
            for (int d = 0; d < D; d += 2) *reinterpret_cast<uint32_t*>(dst + d) = cvt_bf16x2(o[d] * inv, o[d + 1] * inv);
        }
    }
};

// Adds the pieces of item `it` that continue it: those of the CTAs behind the one
// with its tile 0.
template <int HD>
__device__ __forceinline__ void add_continued(const TGKvGroupParams& p, Acc<HD>& acc, TGKvGroupPos it, uint32_t r, int lane) {
    uint32_t lo = 0, hi = p.n_cta;               // the last CTA that starts at or before the item
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (tgkv_group_le(start_of(p, mid), it)) lo = mid;
        else hi = mid;
    }
    for (uint32_t b = lo + 1; b < p.n_cta; ++b) {
        const TGKvGroupPos s = start_of(p, b);
        if (!tgkv_group_same_item(s, it)) break;
        const TGKvGroupPos e = start_of(p, b + 1);
        if (tgkv_group_same_item(s, e) && s.tile == e.tile) continue;            // an empty stretch
        acc.add(p, (uint64_t)p.cta_rows + 256u * b + r, lane);
    }
}

// share: every query row, from its prefix part and its own part.
template <typename T, int HD>
__global__ void __launch_bounds__(256) group_merge_parts_kernel(const __grid_constant__ TGKvGroupParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5), total = p.tok0[p.n_seq] * p.n_heads;
    const int lane = threadIdx.x & 31;
    if (row >= total) return;
    const uint32_t G = p.n_heads / p.n_kv_heads, tpt = kRows / G;
    const uint32_t t = row / p.n_heads, h = row % p.n_heads, kvh = h / G, sub = h % G;
    const uint32_t i = seq_of(p, t), own = t - p.tok0[i];
    Acc<HD> acc;
    acc.add(p, row, lane);
    add_continued<HD>(p, acc, TGKvGroupPos{0, kvh, t / tpt, 0}, t % tpt * G + sub, lane);
    acc.add(p, (uint64_t)total + row, lane);
    add_continued<HD>(p, acc, TGKvGroupPos{i + 1, kvh, own / tpt, 0}, own % tpt * G + sub, lane);
    acc.template store<T>(p, row, lane);
}

// joined: the rows of items that several CTAs worked on.  Block (b, y) merges
// rows 16 y .. +15 of the item that CTA b leaves unfinished and began itself.
template <typename T, int HD>
__global__ void __launch_bounds__(256) group_merge_split_kernel(const __grid_constant__ TGKvGroupParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t b = blockIdx.x;
    const TGKvGroupPos s = start_of(p, b), e = start_of(p, b + 1);
    // the item that the next CTA continues, begun in this one
    if (e.seq > p.n_seq || e.tile == 0 || (tgkv_group_same_item(s, e) && s.tile > 0)) return;
    TGKvGroupPos it = e;
    it.tile = 0;
    const uint32_t G = p.n_heads / p.n_kv_heads, tpt = kRows / G, t0 = it.rt * tpt;
    const uint32_t ntok = min(tpt, tgkv_group_tokens(&p, it.seq) - t0);
    const int lane = threadIdx.x & 31;
    for (uint32_t r = blockIdx.y * 16 + (threadIdx.x >> 5); r < blockIdx.y * 16 + 16; r += 8) {
        if (r >= ntok * G) continue;
        Acc<HD> acc;
        acc.add(p, (uint64_t)p.cta_rows + 256u * b + 128u + r, lane);
        add_continued<HD>(p, acc, it, r, lane);
        const uint64_t row = (uint64_t)(p.tok0[it.seq - 1] + t0 + r / G) * p.n_heads + it.kvh * G + r % G;
        acc.template store<T>(p, row, lane);
    }
}

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

template <typename T, int HD>
int launch(const TGKvGroupParams* p, cudaStream_t st) {
    const uint32_t total = p->tok0[p->n_seq];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    static bool configured[64];                  // benign race: same value
    if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(group_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::SMEM);
        if (e != cudaSuccess) return (int)e;
        configured[dev] = true;
    }
    if (p->k_new) {
        const uint64_t n = (uint64_t)total * (p->n_kv_heads * HD / 8);
        e = launch_pdl(group_append_kernel<T>, dim3((unsigned)((n + 255) / 256), 2), 256, 0, st, p);
        if (e != cudaSuccess) return (int)e;
    }
    e = launch_pdl(group_kernel<T, HD>, dim3(p->n_cta), kThreads, Cfg<HD>::SMEM, st, p);
    if (e != cudaSuccess) return (int)e;
    if (p->share)
        e = launch_pdl(group_merge_parts_kernel<T, HD>, dim3((total * p->n_heads + 7) / 8), 256, 0, st, p);
    else if (p->n_split)
        e = launch_pdl(group_merge_split_kernel<T, HD>, dim3(p->n_cta, 8), 256, 0, st, p);
    return (int)e;
}

}  // namespace group
}  // namespace tgkv

extern "C" int tgkv_launch_group(const TGKvGroupParams* p, int act, void* stream) {
    using namespace tgkv::group;
    cudaStream_t st = (cudaStream_t)stream;
    if (p->head_dim == 128) return act ? launch<uint16_t, 128>(p, st) : launch<float, 128>(p, st);
    if (p->head_dim == 64) return act ? launch<uint16_t, 64>(p, st) : launch<float, 64>(p, st);
    return (int)cudaErrorInvalidValue;
}
