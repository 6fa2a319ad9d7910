// tgkv_group.cu -- attention of several sequences of one layer that may share
// a prefix cache: token t of sequence i attends the prefix's positions [0, P)
// and its own cache's positions [0, old_i + t].  q head h reads KV head
// h * n_kv_heads / n_heads; out = softmax(q K^T * scale) V over both parts.
//
// group_kernel: persistent CTAs, one per SM, each with its stretch of the line
// of K/V tiles that tgkv_group_plan.h cuts.  A piece is an item (one or two row
// tiles of 128 query rows of one KV head) against a run of 128-position K/V
// tiles, in one pass: S = Q K^T, running maximum and sum in the log2 domain,
// O += P V, 64 positions (half a tile) at a time.  Two streams, each with its own
// O and two S/P buffers of 64 positions in TMEM, its own four softmax warps (one
// thread per row) and its own MMA warp, run side by side:
//   wide pieces    (two row tiles) stream h has the rows of row tile h, and both
//                  read every K/V tile: half the tile traffic per row.  The scores
//                  of the half after next are made as soon as a buffer's P has
//                  been used, while the softmax works on the other buffer;
//   narrow pieces  (one row tile) both have the same rows and take alternate
//                  tiles; their results join at the end of the piece.  A tile's
//                  scores are made at once: a 64-column product of 128 dims takes
//                  as long as one of 128 columns (about 525 cycles; reading Q from
//                  shared memory bounds both), and here the other stream fills the
//                  wait.
// A tile with at most 64 rows is one half.
// Bound, long prompts: a stream's chain scores - softmax - product.  An SM takes
// about 2400 cycles per 128 rows x 128 positions of 128 dims, the starts and ends of
// items included; with two streams side by side that is about 4800 for a stream's
// own, of which the tensor core has work for 1024.  4 prompts of 2000 tokens behind
// 2048 (32/8 heads of 128): 488 us, 820 TFLOP/s with bf16 activations, 719 us with
// fp32 ones.  Measured slower in the first case: both halves' scores at once (584
// us), the streams' softmax in strict turns (563 us), one thread watching both
// streams' barriers (728 us), sixteen softmax warps, two threads a row (649 us).
// Warps (384 threads): 0-3 and 4-7 the streams' softmax, 8 TMA (K/V tiles in
// 64-dim boxes, 128-byte swizzle, into two rings that run ahead over the whole
// stretch; Q of bf16 calls), 9 and 10 the streams' MMAs (one lane each), 11 clears
// unseen rows of V tiles.
// TERMS is the number of bf16 terms of q and P: 1 with bf16 activations (q is
// exact, P is rounded once, 2^-8 of a weight, as the output itself is), 2 with
// fp32 ones (hi + lo, 16 mantissa bits; a third term of P has no room in the
// columns S leaves free).  Scores, maxima, sums and O are fp32.
// TMEM columns: buffer b of stream h [128 h + 64 b, +64), P there as bf16 pairs
// (hi at +0, lo at +32); O of stream h [256 + 128 h, +HD).
//
// group_merge kernels join the partials of rows whose tiles more than one
// piece attended: no atomics, always in the same order.
//
// Every mbarrier wait is bounded; one that runs out sets the device error word
// and the CTA ends without further waits on its own data.
#include "tgkv_group.cuh"
#include "tgkv_group_light.cuh"

namespace tgkv {
namespace group {

constexpr int kTmaWarp = 8, kMmaWarp = 9;
constexpr uint32_t TM_S = 0, TM_O = 256, TM_COLS = 512;
constexpr int kSub = 64;                        // half a tile

// An item as this kernel works on it.
struct PieceRows : ItemRows {
    bool wide;                                   // two row tiles
    __device__ PieceRows(const TGKvGroupShape& s, const Pieces& pc, int terms)
        : ItemRows(s, pc), wide(terms == 1 && tokens > s.tpt) {}
    // 64-position halves of tile j that hold rows
    __device__ uint32_t halves(uint32_t j) const { return rows(j) - pos(j) > kSub ? 2 : 1; }
};

template <int HD>
struct Cfg {
    static constexpr uint32_t kTile = (uint32_t)(HD / 64) * kBlock;    // one K, V or Q tile
    static constexpr int kStages = HD == 128 ? 2 : 4;                  // per ring: 128 KB in all
    static constexpr uint32_t OFF_K = 0, OFF_V = kStages * kTile, OFF_Q = 2 * kStages * kTile;
    static constexpr uint32_t OFF_BAR = OFF_Q + 2 * kTile;             // Q: two row tiles, or hi and lo
    static constexpr int B_KFULL = 0, B_KEMPTY = kStages, B_VFULL = 2 * kStages, B_VEMPTY = 3 * kStages;
    // [2 streams][2 halves], one phase per tile each:
    static constexpr int B_SFULL = 4 * kStages;      // S is in TMEM
    static constexpr int B_PFULL = B_SFULL + 4;      // its P is written, O rescaled (128 arrivals)
    static constexpr int B_PVDONE = B_PFULL + 4;     // its PV is complete
    static constexpr int B_QFULL = B_PVDONE + 4;      // a piece's Q is in shared memory
    static constexpr int B_QEMPTY = B_QFULL + 1;     // every S of a piece is complete
    static constexpr uint32_t OFF_ML = OFF_BAR + 40 * 8;               // [2 streams][128] (m, l)
    static constexpr uint32_t OFF_SLOT = OFF_ML + 2 * kRows * 8;
    static constexpr uint32_t OFF_TAB = OFF_SLOT + 16;                 // tok0, old_len
    static constexpr uint32_t OFF_STG = (OFF_TAB + (2 * TGKV_MAX_ITEMS + 1) * 4 + 127) / 128 * 128;
    static constexpr uint32_t SMEM = OFF_STG + 8 * 2048 + 1024;        // 2 KB per softmax warp; slack: alignment
    static constexpr int B_VREADY = B_QEMPTY + 1;    // a V tile's unseen rows are cleared
    static_assert(B_VREADY + kStages <= 40 && SMEM <= 232448, "shared memory per CTA");
};

// The two warps (streams 0 and 1) of a TMEM lane quarter.
__device__ __forceinline__ void pair_sync(int quarter) {
    asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
}
// The packed rows of k_new / v_new into their caches, 8 elements per thread.
template <typename T>
__global__ void __launch_bounds__(256) group_append_kernel(const __grid_constant__ TGKvGroupParams p) {
    __shared__ uint32_t tok0[TGKV_MAX_ITEMS + 1];
    copy_table(tok0, p.tok0, p.n_seq + 1, threadIdx.x, 256);
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t kv_dim = p.n_kv_heads * p.head_dim, vec = kv_dim / 8;
    const uint64_t x = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (x >= (uint64_t)tok0[p.n_seq] * vec) return;
    const uint32_t t = (uint32_t)(x / vec), e = (uint32_t)(x % vec) * 8, i = seq_of(tok0, p.n_seq, t);
    const T* src = reinterpret_cast<const T*>(blockIdx.y ? p.v_new : p.k_new) + (uint64_t)t * kv_dim + e;
    const TGKvRowCache c = p.table[i];
    uint16_t* dst = reinterpret_cast<uint16_t*>(c.base) +
                    ((uint64_t)blockIdx.y * c.max_seq + as_memory(p.old_len)[i] + (t - tok0[i])) * kv_dim + e;
    *reinterpret_cast<uint4*>(dst) = row_part(src);
    // read by the attention's TMA loads
    asm volatile("fence.proxy.async.global;" ::: "memory");
}

__device__ __forceinline__ float max32(const uint32_t (&v)[32]) {
    float a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = -INFINITY;
#pragma unroll
        for (int k = 0; k < 8; k += 2) a[i] = max3(a[i], __uint_as_float(v[8 * i + k]), __uint_as_float(v[8 * i + k + 1]));
    }
    return max3(max3(a[0], a[1], a[2]), a[3], a[3]);
}

// P = 2^(s * scale - msc) of 32 positions as bf16 words (two positions each) into
// the TMEM columns from `col` on: hi there and, with two terms, the rounding
// residuals lo 32 columns behind; the fp32 values add up in l.  A position the row
// does not see has s = -inf and gets 0.  (A part of the exponentials as a polynomial
// on the FMA units measured no faster: 490 us with none to a quarter of them, 513 us
// with three eighths, 4 prompts of 2000 tokens behind 2048; the streams' chain of
// products bounds the kernel, not the exponential unit.)
template <int TERMS>
__device__ __forceinline__ void exp32(const uint32_t (&v)[32], float scale, float msc, float2& l, uint32_t col) {
    const float2 sc = make_float2(scale, scale), nm = make_float2(-msc, -msc);
    uint32_t ph[16], pl[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) {
        const float2 d = __ffma2_rn(make_float2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), sc, nm);
        const float2 pp = make_float2(ex2_approx(d.x), ex2_approx(d.y));
        l = __fadd2_rn(l, pp);
        ph[c] = cvt_bf16x2(pp.x, pp.y);
        if (TERMS == 2) {
            const float2 r = __ffma2_rn(make_float2(lo_f(ph[c]), hi_f(ph[c])), make_float2(-1.f, -1.f), pp);
            pl[c] = cvt_bf16x2(r.x, r.y);
        }
    }
    tmem_st16(col, ph);
    if (TERMS == 2) tmem_st16(col + 32, pl);
}

// Half a query row of fp32 (64-dim halves of HD dims) as hi and lo bf16 words into
// the two Q tiles: row r of a box is 128 bytes, its 16-byte chunk c at c ^ (r % 8).
template <int HD>
__device__ __forceinline__ void store_q_terms(const float* src, bool valid, unsigned char* q, int r, int half) {
    constexpr int D = HD / 2;                    // dims of this thread
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
        if (valid) {
            x = reinterpret_cast<const float4*>(src)[2 * c];
            y = reinterpret_cast<const float4*>(src)[2 * c + 1];
        }
        const uint4 h = make_uint4(cvt_bf16x2(x.x, x.y), cvt_bf16x2(x.z, x.w), cvt_bf16x2(y.x, y.y), cvt_bf16x2(y.z, y.w));
        const uint4 l = make_uint4(cvt_bf16x2(x.x - lo_f(h.x), x.y - hi_f(h.x)), cvt_bf16x2(x.z - lo_f(h.y), x.w - hi_f(h.y)),
                                   cvt_bf16x2(y.x - lo_f(h.z), y.y - hi_f(h.z)), cvt_bf16x2(y.z - lo_f(h.w), y.w - hi_f(h.w)));
        const int d = half * D + 8 * c, chunk = ((d & 63) >> 3) ^ (r & 7);
        unsigned char* at = q + (d >> 6) * kBlock + r * 128 + chunk * 16;
        *reinterpret_cast<uint4*>(at) = h;
        *reinterpret_cast<uint4*>(at + (HD / 64) * kBlock) = l;
    }
}

template <typename T, int HD>
__device__ __forceinline__ void run(const TGKvGroupParams& p, uint32_t cta_index, unsigned char* smem_raw) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
    // With two terms (fp32 results) an accumulator takes at most 16 tiles, 256 steps of
    // 16 positions: the tensor core's fp32 sums round towards zero, and the sums of
    // longer runs would lose more bits than the two terms keep.
    constexpr uint32_t kMost = TERMS == 2 ? 32 : 0;
    using C = Cfg<HD>;
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_addr(base);
    uint64_t* bar = reinterpret_cast<uint64_t*>(base + C::OFF_BAR);
    uint32_t* tslot = reinterpret_cast<uint32_t*>(base + C::OFF_SLOT);
    volatile uint32_t* flag = tslot + 1;         // some value of V was not finite (clear_unseen)
    uint32_t* tok0 = reinterpret_cast<uint32_t*>(base + C::OFF_TAB);
    uint32_t* old_len = tok0 + p.n_seq + 1;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    copy_table(tok0, p.tok0, p.n_seq + 1, tid, kThreads);
    copy_table(old_len, p.old_len, p.n_seq, tid, kThreads);
    if (tid == 0) {
        *flag = 0;
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&bar[C::B_KFULL + i], 1);
            mbar_init(&bar[C::B_KEMPTY + i], 2);
            mbar_init(&bar[C::B_VFULL + i], 1);
            mbar_init(&bar[C::B_VEMPTY + i], 2);
            mbar_init(&bar[C::B_VREADY + i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bar[C::B_SFULL + i], 1);
            mbar_init(&bar[C::B_PFULL + i], 128);
            mbar_init(&bar[C::B_PVDONE + i], 1);
        }
        mbar_init(&bar[C::B_QFULL], TERMS == 2 ? 256 : 1);
        mbar_init(&bar[C::B_QEMPTY], 2);
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
    const uint32_t G = p.n_heads / p.n_kv_heads;
    const TGKvGroupShape sh = shape_of(p, 0, old_len, tok0);
    // Everything above overlaps the previous kernel on the stream.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    Pieces pc(sh, start_of(p, 0, cta_index), start_of(p, 0, cta_index + 1), kMost);
    if (warp >= 8) {
        if (warp == kTmaWarp && lane == 0) {
            uint32_t nk = 0, nv = 0, it = 0;     // K and V tiles and pieces issued
            bool ok = true;
            for (; ok && pc.more(); pc.next(sh, kMost)) {
                const uint32_t seq = pc.at.seq, npre = tgkv_group_prefix_tiles(&sh, seq);
                const uint32_t t0 = pc.at.at * sh.item_tokens;
                const bool wide = TERMS == 1 && tgkv_group_tokens(&sh, seq) - t0 > sh.tpt;
                const int x = (int)(pc.at.kvh * HD);
                for (uint32_t j = pc.j0; j < pc.j1; ++j) {
                    const bool own = j >= npre;
                    const uint64_t map = p.tmaps + 128ull * (own ? seq - 1 : p.n_seq);
                    const int y = (int)((own ? j - npre : j) * kPos);
                    const uint32_t s = nk % C::kStages, ph = (nk / C::kStages - 1) & 1u;
                    if (nk >= C::kStages && !(ok = mbar_wait(&bar[C::B_KEMPTY + s], ph))) break;
                    mbar_arrive_expect_tx(&bar[C::B_KFULL + s], C::kTile);
                    for (int b = 0; b < HD / 64; ++b)
                        tma_load_3d(base + C::OFF_K + s * C::kTile + b * kBlock, map, x + 64 * b, y, 0,
                                    &bar[C::B_KFULL + s]);
                    ++nk;
                    if (TERMS == 1 && j == pc.j0) {
                        // the piece's Q, once the last piece's scores are made
                        if (it > 0 && !(ok = mbar_wait(&bar[C::B_QEMPTY], (it - 1) & 1u))) break;
                        const uint32_t box = 64 * 2 * G * sh.tpt;
                        mbar_arrive_expect_tx(&bar[C::B_QFULL], box * (HD / 64) * (wide ? 2 : 1));
                        const int tok = (int)((seq ? tok0[seq - 1] : 0) + t0);
                        for (int h = 0; h < (wide ? 2 : 1); ++h)
                            for (int b = 0; b < HD / 64; ++b)
                                tma_load_3d(base + C::OFF_Q + h * C::kTile + b * kBlock,
                                            reinterpret_cast<uint64_t>(&p.qmap), 64 * b, (int)(pc.at.kvh * G),
                                            tok + h * (int)sh.tpt, &bar[C::B_QFULL]);
                        ++it;
                    }
                    if (nv >= C::kStages && !(ok = mbar_wait(&bar[C::B_VEMPTY + s], ph))) break;
                    mbar_arrive_expect_tx(&bar[C::B_VFULL + s], C::kTile);
                    for (int b = 0; b < HD / 64; ++b)
                        tma_load_3d(base + C::OFF_V + s * C::kTile + b * kBlock, map, x + 64 * b, y, 1,
                                    &bar[C::B_VFULL + s]);
                    ++nv;
                }
            }
            // every copy has landed before the CTA may end (at once in a normal run)
            for (uint32_t i = nk > C::kStages ? nk - C::kStages : 0; i < nk; ++i)
                ok = mbar_wait(&bar[C::B_KFULL + i % C::kStages], (i / C::kStages) & 1u) && ok;
            for (uint32_t i = nv > C::kStages ? nv - C::kStages : 0; i < nv; ++i)
                ok = mbar_wait(&bar[C::B_VFULL + i % C::kStages], (i / C::kStages) & 1u) && ok;
            if (TERMS == 1 && it > 0) ok = mbar_wait(&bar[C::B_QFULL], (it - 1) & 1u) && ok;
            if (!ok) atomicExch(p.err, kErrTimeout);
        } else if ((warp == kMmaWarp || warp == kMmaWarp + 1) && lane == 0) {
            // One warp per stream.  Step k of a piece belongs to stream k % 2; its K/V tile is
            // g0 + k / 2 (wide) or g0 + k (narrow).  PV of a half as soon as its P is there, then
            // the next step's S into the buffer: half by half (wide) or at once behind the second
            // half (narrow).  Both warps pass every phase of the rings and of Q, in order, so that
            // a parity always means the phase it is waited for: a tile or a Q that a stream does
            // not use, it releases when it sees it.
            const uint32_t h = (uint32_t)(warp - kMmaWarp);
            uint32_t g0 = 0, it = 0, n = 0;      // K/V tiles of earlier pieces; pieces; this stream's steps
            uint32_t ks = 0, vs = 0;             // tiles passed in each ring
            bool ok = true;
            auto pass = [&](int full, int empty, uint32_t& seen, uint32_t g) {
                for (; ok && seen < g; ++seen) {
                    ok = mbar_wait(&bar[full + seen % C::kStages], (seen / C::kStages) & 1u);
                    mbar_arrive(&bar[empty + seen % C::kStages]);
                }
            };
            for (; ok && pc.more(); pc.next(sh, kMost), ++it) {
                const PieceRows pr(sh, pc, TERMS);
                const uint32_t tiles = pc.j1 - pc.j0, steps = pr.wide ? 2 * tiles : tiles;
                ok = mbar_wait(&bar[C::B_QFULL], it & 1u);
                tc_fence_after();
                if (h >= steps) mbar_arrive(&bar[C::B_QEMPTY]);
                const uint64_t qd = umma_desc_sw128(sbase + C::OFF_Q + (pr.wide && h ? C::kTile : 0u), 16, 1024);
                // S of step k's half (both halves with half 2); half 0 or 2 comes first for a tile
                auto issue_s = [&](uint32_t k, uint32_t half) {
                    const uint32_t t = pr.wide ? k >> 1 : k, g = g0 + t, s = g % C::kStages;
                    if (half != 1) {
                        pass(C::B_KFULL, C::B_KEMPTY, ks, g);
                        ok = ok && mbar_wait(&bar[C::B_KFULL + s], (g / C::kStages) & 1u);
                    }
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t halves = pr.halves(pc.j0 + t), b = half & 1u;
                    if (b < halves) {
                        const uint32_t id = umma_idesc_bf16(kRows, half == 2 && halves == 2 ? kPos : kSub, 0, 0);
                        const uint64_t kd = umma_desc_sw128(sbase + C::OFF_K + s * C::kTile + b * (kSub * 128u), 16, 1024);
#pragma unroll
                        for (uint32_t i = 0; i < TERMS * (HD / 16); ++i) {
                            const uint32_t q = i / (HD / 16), d = i % (HD / 16);
                            const uint32_t off = (d >> 2) * kBlock + (d & 3u) * 32u;
                            umma_ss(tmem + TM_S + h * 128u + b * 64u, qd + ((q * C::kTile + off) >> 4), kd + (off >> 4), id,
                                    i != 0);
                        }
                    }
                    umma_commit(&bar[C::B_SFULL + 2 * h + b]);
                    if (half == 0) return;
                    if (half == 2) umma_commit(&bar[C::B_SFULL + 2 * h + 1]);
                    umma_commit(&bar[C::B_KEMPTY + s]);
                    ks = g + 1;
                    if (k + 2 >= steps) umma_commit(&bar[C::B_QEMPTY]);
                    if (!pr.wide && k + 1 < steps) pass(C::B_KFULL, C::B_KEMPTY, ks, g + 2);
                };
                if (ok && h < steps) issue_s(h, pr.wide ? 0 : 2);
                if (ok && pr.wide) issue_s(h, 1);
                for (uint32_t k = h; ok && k < steps; k += 2, ++n) {
                    const uint32_t t = pr.wide ? k >> 1 : k, g = g0 + t, s = g % C::kStages;
                    const uint32_t halves = pr.halves(pc.j0 + t);
                    const bool more = k + 2 < steps;
                    constexpr uint32_t id_pv = umma_idesc_bf16(kRows, HD, 0, 1);
                    pass(C::B_VFULL, C::B_VEMPTY, vs, g);
                    // P of positions 16 kk .. +15: 8 columns.  V is MN-major: 64-dim blocks 16 KB
                    // apart, 8-position groups 1 KB apart.
                    const uint64_t vd = umma_desc_sw128(sbase + C::OFF_V + s * C::kTile, kBlock, 1024);
                    for (uint32_t b = 0; ok && b < 2; ++b) {
                        ok = mbar_wait(&bar[C::B_PFULL + 2 * h + b], n & 1u) &&
                             (b || (mbar_wait(&bar[C::B_VFULL + s], (g / C::kStages) & 1u) &&
                                    mbar_wait(&bar[C::B_VREADY + s], (g / C::kStages) & 1u)));
                        if (!ok) break;
                        tc_fence_after();
                        if (b < halves)
#pragma unroll
                            for (uint32_t i = 0; i < TERMS * 4; ++i) {
                                const uint32_t q = i >> 2, kk = i & 3u;
                                umma_ts(tmem + TM_O + h * 128u, tmem + TM_S + h * 128u + b * 64u + q * 32u + kk * 8u,
                                        vd + (((4 * b + kk) * 16u * 128u) >> 4), id_pv, k > 1 || b || i != 0);
                            }
                        umma_commit(&bar[C::B_PVDONE + 2 * h + b]);
                        if (b) {
                            umma_commit(&bar[C::B_VEMPTY + s]);
                            vs = g + 1;
                        }
                        // the next S goes where this PV reads P
                        if (pr.wide || b) ok = mbar_wait(&bar[C::B_PVDONE + 2 * h + b], n & 1u);
                        if (ok && more && (pr.wide || b)) issue_s(k + 2, pr.wide ? b : 2);
                    }
                }
                g0 += tiles;
                pass(C::B_KFULL, C::B_KEMPTY, ks, g0);
                pass(C::B_VFULL, C::B_VEMPTY, vs, g0);
            }
            if (!ok) atomicExch(p.err, kErrTimeout);
        } else if (warp == kMmaWarp + 2) {
            // V rows that no query of the item sees may hold anything; P is 0 there, but 0 * Inf is
            // NaN, so they are cleared, and those that only some see are cleared of what is not
            // finite, before a PV reads the tile (a stage's next tile comes after that PV)
            uint32_t g = 0;
            bool ok = true;
            for (; ok && pc.more(); pc.next(sh, kMost)) {
                const PieceRows pr(sh, pc, TERMS);
                const uint32_t first = pc.at.seq ? old_len[pc.at.seq - 1] + pc.at.at * sh.item_tokens + 1 : 0;   // token 0 sees
                for (uint32_t j = pc.j0; ok && j < pc.j1; ++j, ++g) {
                    const uint32_t rows = pr.rows(j) - pr.pos(j), s = g % C::kStages;
                    const uint32_t lo = pr.own(j) ? (uint32_t)max((int)(first - pr.pos(j)), 0) : rows;
                    ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_VFULL + s], (g / C::kStages) & 1u));
                    if (ok && lo < kPos) {
                        clear_unseen<HD, 32>(base + C::OFF_V + s * C::kTile, lo, rows, rows > kSub ? kPos : kSub, lane, flag);
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (ok && lane == 0) mbar_arrive(&bar[C::B_VREADY + s]);
                }
            }
            if (!ok && lane == 0) atomicExch(p.err, kErrTimeout);
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, h = warp >> 2, r = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t ts = lanes + TM_S + (uint32_t)h * 128u, to = lanes + TM_O + (uint32_t)h * 128u;
        float2* ml = reinterpret_cast<float2*>(base + C::OFF_ML);
        const float scale = p.qscale;
        const uint32_t rtok = (uint32_t)r / G, sub = (uint32_t)r % G;
        const uint32_t total_rows = tok0[p.n_seq] * p.n_heads;
        uint32_t it = 0, n = 0;                  // pieces; this stream's steps
        bool ok = true;
        // Both warps of a pair meet at named barriers, so neither leaves early:
        // after a failed wait a warp only keeps the barriers' counts.
        for (; pc.more(); pc.next(sh, kMost), ++it) {
            const uint32_t seq = pc.at.seq;
            const PieceRows pr(sh, pc, TERMS);
            const bool wide = pr.wide;
            const uint32_t t0 = pc.at.at * sh.item_tokens, left = tgkv_group_tokens(&sh, seq) - t0;
            const uint32_t tb = wide && h ? sh.tpt : 0;                       // this stream's first token of the item
            const uint32_t ntok = min(sh.tpt, left - tb);
            const bool valid = rtok < ntok;
            const bool busy = (uint32_t)(quarter * 32) < ntok * G;            // the warp has rows
            const uint32_t own_first = seq ? old_len[seq - 1] + t0 + 1 : 0;      // rows the item's first token sees
            const uint32_t own_min = seq ? own_first + tb : 0;                   // the stream's first token
            const uint32_t own_mine = own_min + min(rtok, ntok - 1);             // rows this thread's token sees
            const uint64_t row = (uint64_t)((seq ? tok0[seq - 1] : 0) + t0 + tb + rtok) * p.n_heads + pc.at.kvh * G + sub;
            const uint32_t tiles = pc.j1 - pc.j0, steps = wide ? 2 * tiles : tiles;
            if constexpr (TERMS == 2) {
                if (ok && it > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_QEMPTY], (it - 1) & 1u));
                store_q_terms<HD>(reinterpret_cast<const float*>(p.q) + row * HD + h * (HD / 2), valid,
                                  base + C::OFF_Q, r, h);
                fence_proxy_async_smem();
                mbar_arrive(&bar[C::B_QFULL]);
            }

            float m = -INFINITY;                 // running maximum of the raw scores
            float2 l2 = make_float2(0.f, 0.f);
            for (uint32_t k = (uint32_t)h; k < steps; k += 2) {
                const uint32_t t = wide ? k >> 1 : k, j = pc.j0 + t;
                const uint32_t rows = pr.rows(j) - pr.pos(j);                    // of the tile, that some query sees
                const uint32_t all = (pr.own(j) ? own_min : p.prefix_len) - pr.pos(j);         // that every query sees
                const int lim = (int)((pr.own(j) ? own_mine : p.prefix_len) - pr.pos(j));      // that this thread's sees
                const bool mask = (int)all < kPos;
                const uint32_t halves = rows > kSub ? 2 : 1;
#pragma unroll 1
                for (uint32_t b = 0; b < 2; ++b) {
                    const uint32_t tsb = ts + b * 64u;
                    const int lm = lim - (int)(b * kSub);
                    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_SFULL + 2 * h + b], n & 1u));
                    if (ok && busy && b < halves) {
                        tc_fence_after();
                        uint32_t va[32], vb[32];
                        tmem_ld32(tsb, va);
                        tmem_ld32(tsb + 32, vb);
                        tmem_wait_ld(va, vb);
                        if (mask) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                if (i >= lm) va[i] = 0xff800000u;                // -inf
                                if (i >= lm - 32) vb[i] = 0xff800000u;
                            }
                        }
                        const float tm = max3(-INFINITY, max32(va), max32(vb));
                        // the running maximum moves only when exceeded by more than 2^8 (or NaN)
                        const bool grow = !((tm - m) * scale <= 8.f);
                        if (__any_sync(0xffffffffu, grow)) {
                            const float alpha = !grow ? 1.f : m == -INFINITY ? 0.f : ex2_approx((m - tm) * scale);
                            if (grow) m = tm;
                            l2.x *= alpha;
                            l2.y *= alpha;
                            if (k > 1 || b) {
                                // O holds the earlier halves: all of them, then scale it
                                ok = __all_sync(0xffffffffu,
                                                mbar_wait(&bar[C::B_PVDONE + 2 * h + (b ^ 1u)], (b ? n : n - 1) & 1u));
                                if (ok) {
                                    tc_fence_after();
#pragma unroll 1
                                    for (int c = 0; c < HD / 16; ++c) {
                                        uint32_t o[16];
                                        tmem_ld16(to + c * 16, o);
                                        tmem_wait_ld16(o);
#pragma unroll
                                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                        tmem_st16(to + c * 16, o);
                                    }
                                }
                            }
                        }
                        const float msc = m == -INFINITY ? 0.f : m * scale;
                        exp32<TERMS>(va, scale, msc, l2, tsb);
                        exp32<TERMS>(vb, scale, msc, l2, tsb + 16);
                        tmem_wait_st();
                    }
                    tc_fence_before();
                    mbar_arrive(&bar[C::B_PFULL + 2 * h + b]);
                }
                ++n;
            }

            // ---- the piece's rows: out, or a partial
            const bool mine = (uint32_t)h < steps;                               // this stream had a tile
            if (ok && mine) ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_PVDONE + 2 * h + 1], (n - 1) & 1u));
            if (ok) tc_fence_after();
            float l = l2.x + l2.y, msc = m * scale;                              // -inf if nothing was seen
            float w0 = 1.f, w1 = 0.f;                                            // weights of the streams' O
            if (!wide) {
                // both streams have the same rows: join (m, l), then each brings out half of the
                // head dims from both O
                ml[h * kRows + r] = make_float2(msc, l);
                tc_fence_before();
                pair_sync(quarter);
                tc_fence_after();
                const float2 a = ml[r], b = ml[kRows + r];
                msc = fmaxf(a.x, b.x);
                w0 = a.x == -INFINITY ? 0.f : ex2_approx(a.x - msc);
                w1 = b.x == -INFINITY ? 0.f : ex2_approx(b.x - msc);
                l = a.y * w0 + b.y * w1;
            }
            const bool whole = pc.first == 0 && pc.j1 == pc.nt && !p.share;
            const bool again = pc.j0 > pc.first;                                 // adds to the item's earlier piece here
            const uint32_t irow = (wide ? (uint32_t)h * kRows : 0u) + (uint32_t)r;
            uint64_t slot;
            if (pc.first > 0 || !p.share) slot = (uint64_t)p.line[0].cta_rows + 512u * cta_index + (pc.first > 0 ? 0u : 256u) + irow;
            else slot = (seq ? total_rows : 0u) + row;
            float keep = 0.f;                                                    // weight of the slot's earlier sum
            float2* slot_ml = reinterpret_cast<float2*>(p.part_ml) + slot;
            if (TERMS == 2 && again) {
                if (valid) {
                    const float2 old = *slot_ml;
                    const float M = fmaxf(old.x, msc), w = msc == -INFINITY ? 0.f : ex2_approx(msc - M);
                    keep = old.x == -INFINITY ? 0.f : ex2_approx(old.x - M);
                    l = l * w + old.y * keep;
                    msc = M;
                    w0 *= w;
                    w1 *= w;
                }
                pair_sync(quarter);                                              // both warps have read the slot's (m, l)
            }
            const float inv = whole ? 1.f / l : 1.f;
            w0 *= inv;
            w1 *= inv;
            keep *= inv;
            if (ok && busy) {
                // 64 bytes of each row at a time through the warp's 2 KB of shared memory, so that
                // four lanes write a row's 64 bytes: 16-byte part q of row x lies at x * 64 + (q ^
                // (x / 2 % 4)) * 16, free of bank conflicts both ways
                unsigned char* stg = base + C::OFF_STG + warp * 2048;
                const uint32_t part = (uint32_t)lane & 3u;
                uint64_t dst[4];                                                 // rows lane / 4 + 8 i
                float kp[4];
                const uint64_t mine_row = valid ? (whole ? row : slot) : ~0ull;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    dst[i] = __shfl_sync(0xffffffffu, mine_row, (lane >> 2) + 8 * i);
                    kp[i] = TERMS == 2 ? __shfl_sync(0xffffffffu, keep, (lane >> 2) + 8 * i) : 0.f;
                }
                // the earlier sums are where the earlier pieces put them: a whole item's in this
                // CTA's slots, consecutive rows for consecutive lanes
                const uint64_t first_slot = slot - (uint32_t)lane;
                auto flush = [&](const uint4 (&w)[4], unsigned char* out, uint32_t row_bytes, uint32_t off, bool add) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<uint4*>(stg + lane * 64 + ((q ^ (lane >> 1)) & 3) * 16) = w[q];
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t x = (uint32_t)(lane >> 2) + 8u * i;
                        uint4 y = *reinterpret_cast<const uint4*>(stg + x * 64 + ((part ^ (x >> 1)) & 3u) * 16);
                        if (dst[i] == ~0ull) continue;
                        if (TERMS == 2 && add) {
                            const float4 o = *reinterpret_cast<const float4*>(
                                reinterpret_cast<const unsigned char*>(p.part_o) +
                                (whole ? first_slot + x : dst[i]) * row_bytes + off + part * 16);
                            y = make_uint4(__float_as_uint(fmaf(o.x, kp[i], __uint_as_float(y.x))),
                                           __float_as_uint(fmaf(o.y, kp[i], __uint_as_float(y.y))),
                                           __float_as_uint(fmaf(o.z, kp[i], __uint_as_float(y.z))),
                                           __float_as_uint(fmaf(o.w, kp[i], __uint_as_float(y.w))));
                        }
                        *reinterpret_cast<uint4*>(out + dst[i] * row_bytes + off + part * 16) = y;
                    }
                    __syncwarp();
                };
                // 16 columns of the row's sums (columns 16 c ..), joined and scaled
                const uint32_t oa = wide ? to : lanes + TM_O;
                // (a weight that is 0 takes part too: 0 x Inf is NaN, and the row sees it)
                auto take = [&](int c, float (&o)[16]) {
                    uint32_t x[16];
                    tmem_ld16(oa + c * 16, x);
                    tmem_wait_ld16(x);
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __uint_as_float(x[i]) * w0;
                    if (!wide && steps > 1) {                                    // the other stream had a tile
                        tmem_ld16(oa + 128 + c * 16, x);
                        tmem_wait_ld16(x);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = fmaf(__uint_as_float(x[i]), w1, o[i]);
                    }
                };
                const int c0 = wide ? 0 : h * (HD / 32), c1 = wide ? HD / 16 : c0 + HD / 32;
                if (TERMS == 1 && whole) {
#pragma unroll 1
                    for (int c = c0; c < c1; c += 2) {
                        float o[16];
                        uint4 w[4];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            take(c + k, o);
#pragma unroll
                            for (int q = 0; q < 2; ++q)
                                w[2 * k + q] = make_uint4(cvt_bf16x2(o[8 * q], o[8 * q + 1]), cvt_bf16x2(o[8 * q + 2], o[8 * q + 3]),
                                                          cvt_bf16x2(o[8 * q + 4], o[8 * q + 5]), cvt_bf16x2(o[8 * q + 6], o[8 * q + 7]));
                        }
                        flush(w, reinterpret_cast<unsigned char*>(p.out), HD * 2, c * 32, false);
                    }
                } else {
#pragma unroll 1
                    for (int c = c0; c < c1; ++c) {
                        float o[16];
                        uint4 w[4];
                        take(c, o);
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            w[q] = make_uint4(__float_as_uint(o[4 * q]), __float_as_uint(o[4 * q + 1]),
                                              __float_as_uint(o[4 * q + 2]), __float_as_uint(o[4 * q + 3]));
                        flush(w, reinterpret_cast<unsigned char*>(whole ? p.out : (void*)p.part_o), HD * 4, c * 64, again);
                    }
                }
                if (valid && !whole && (wide || h == 0)) *slot_ml = make_float2(msc, l);
                if (__any_sync(0xffffffffu, *flag != 0) && valid && seq) {
                    // what the piece's V rows hold that is not finite, of those this row sees
                    const uint32_t f0 = pr.own(pc.j0) ? pr.pos(pc.j0) : 0u, f1 = pr.own(pc.j1) ? pr.pos(pc.j1) : 0u;
#pragma unroll 1
                    for (int d = c0 * 16; d < c1 * 16; ++d) {
                        const float x = cache_non_finite(p.table + (seq - 1), p.n_kv_heads * HD, pc.at.kvh * HD + d,
                                                         max(own_first, f0), min(own_mine, f1));
                        if (x == 0.f) continue;
                        if (!whole) p.part_o[slot * HD + d] += x;
                        else if constexpr (TERMS == 2) reinterpret_cast<float*>(p.out)[row * HD + d] += x;
                        else reinterpret_cast<uint16_t*>(p.out)[row * HD + d] =
                            (uint16_t)(cvt_bf16x2(lo_f(reinterpret_cast<uint16_t*>(p.out)[row * HD + d]) + x, 0.f) & 0xffffu);
                    }
                }
            }
            if (!wide) {
                // the other stream has read this one's O and (m, l), and both the slot's rows are written
                __syncwarp();
                tc_fence_before();
                pair_sync(quarter);
            }
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

// Both lines in one launch, each on its share of the SMs: what bounds line 1 is
// HBM, what bounds line 0 is not.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) group_kernel(const __grid_constant__ TGKvGroupParams p) {
    extern __shared__ unsigned char smem_raw[];
    if (blockIdx.x < p.line[0].n_cta) run<T, HD>(p, blockIdx.x, smem_raw);
    else light::run<T, HD>(p, blockIdx.x - p.line[0].n_cta, smem_raw);
}

// ------------------------------------------------------------------ merge
// A row's result from its partials (o, m, l): sum 2^(m - M) o / sum 2^(m - M) l.
// One warp per query row, HD / 32 dims per lane.  Lane i keeps partial i's place and
// (m, l), and up to 32 partials' rows are in flight at once.  What it takes is a few
// memory latencies, so the places are worked out, and the parameters read, before
// the wait for the partials.
template <int HD>
struct Acc {
    static constexpr int D = HD / 32;
    const float *part_o, *part_ml;
    float o[D], m, l;
    uint32_t n, all;                             // partials noted; in all
    uint64_t slot;                               // lane i: partial i's row
    bool ready;                                  // the partials may be read
    __device__ Acc(const TGKvGroupParams& p)
        : part_o(p.part_o), part_ml(p.part_ml), m(-INFINITY), l(0.f), n(0), all(0), slot(0), ready(false) {
        asm volatile("" : "+l"(part_o), "+l"(part_ml));
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] = 0.f;
    }
    // Notes a partial row (before the partials may be read, the first 32).
    __device__ void add(uint64_t s, int lane) {
        ++all;
        if (n == 32) {
            if (!ready) return;
            flush(lane);
        }
        if (lane == (int)n) slot = s;
        ++n;
    }
    __device__ void flush(int lane) {
        const float2 ml = lane < (int)n ? *reinterpret_cast<const float2*>(part_ml + slot * 2) : make_float2(-INFINITY, 0.f);
        float M = ml.x;
#pragma unroll
        for (int w = 16; w >= 1; w >>= 1) M = max3(M, __shfl_xor_sync(0xffffffffu, M, w), m);
        // (a part of which the row saw nothing has m = -inf and sums of 0; one whose weight
        // underflows takes part all the same, since 0 x Inf is NaN)
        const float w = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - M), a = m == -INFINITY ? 0.f : ex2_approx(m - M);
        float L = w * ml.y;
#pragma unroll
        for (int k = 16; k >= 1; k >>= 1) L += __shfl_xor_sync(0xffffffffu, L, k);
        l = l * a + L;
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] *= a;
#pragma unroll 4
        for (uint32_t i = 0; i < n; ++i) {
            const uint64_t s = __shfl_sync(0xffffffffu, slot, i);
            const float wi = __shfl_sync(0xffffffffu, w, i);
            const float* src = part_o + s * HD + lane * D;
            if constexpr (D == 4) {
                const float4 v = *reinterpret_cast<const float4*>(src);
                o[0] += wi * v.x;
                o[1] += wi * v.y;
                o[2] += wi * v.z;
                o[3] += wi * v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(src);
                o[0] += wi * v.x;
                o[1] += wi * v.y;
            }
        }
        m = M;
        n = 0;
    }
    // The sums over the partials that `note` notes; `wait` waits for them.
    template <typename Note>
    __device__ void run(Note note, int lane) {
        note();
        asm volatile("griddepcontrol.wait;" ::: "memory");
        ready = true;
        if (all > 32) {
            n = 0;
            note();
        }
        if (n) flush(lane);
    }
    template <typename T>
    __device__ void store(T* out, uint64_t row, int lane) const {
        const float inv = 1.f / l;
        T* dst = out + row * HD + lane * D;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int d = 0; d < D; d += 2) *reinterpret_cast<float2*>(dst + d) = make_float2(o[d] * inv, o[d + 1] * inv);
        } else {
#pragma unroll
            for (int d = 0; d < D; d += 2) *reinterpret_cast<uint32_t*>(dst + d) = cvt_bf16x2(o[d] * inv, o[d + 1] * inv);
        }
    }
};

// Partial rows a CTA of a line has: of the item it continues, then of the one it
// leaves unfinished.
__device__ __forceinline__ uint32_t slot_rows(int line) { return line ? TGKV_GROUP_LIGHT_ROWS : 2 * kRows; }

// A line's starts, in shared memory.
struct Starts {
    uint32_t s[(TGKV_GROUP_MAX_CTAS + 1) * 4];
    __device__ void copy(const TGKvGroupParams& p, int line) {
        copy_table(s, p.line[line].start, (p.line[line].n_cta + 1) * 4, threadIdx.x, blockDim.x);
    }
    __device__ TGKvGroupPos at(uint32_t b) const { return TGKvGroupPos{s[4 * b], s[4 * b + 1], s[4 * b + 2], s[4 * b + 3]}; }
};

// Adds the pieces of item `it` that continue it: those of the CTAs behind the one
// with its tile 0.
template <int HD>
__device__ __forceinline__ void add_continued(const TGKvGroupParams& p, int line, const Starts& st, Acc<HD>& acc,
                                              TGKvGroupPos it, uint32_t r, int lane) {
    const uint32_t n = p.line[line].n_cta;
    uint32_t lo = 0, hi = n;                     // the last CTA that starts at or before the item
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (tgkv_group_le(st.at(mid), it)) lo = mid;
        else hi = mid;
    }
    for (uint32_t b = lo + 1; b < n; ++b) {
        const TGKvGroupPos s = st.at(b);
        if (!tgkv_group_same_item(s, it)) break;
        const TGKvGroupPos e = st.at(b + 1);
        if (tgkv_group_same_item(s, e) && s.tile == e.tile) continue;            // an empty stretch
        acc.add((uint64_t)p.line[line].cta_rows + 2u * slot_rows(line) * b + r, lane);
    }
}

// The row of an item that head `sub` of its KV head's group has for token t of it.
__device__ __forceinline__ uint32_t item_row(const TGKvGroupShape& sh, uint32_t t, uint32_t G, uint32_t sub) {
    return t / sh.tpt * kRows + t % sh.tpt * G + sub;
}

// share: every query row, from its prefix part and its own part.
template <typename T, int HD>
__global__ void __launch_bounds__(256) group_merge_parts_kernel(const __grid_constant__ TGKvGroupParams p) {
    __shared__ uint32_t tok0[TGKV_MAX_ITEMS + 1];
    __shared__ Starts starts[2];
    const int lp = p.prefix_line, lo = p.own_line;
    copy_table(tok0, p.tok0, p.n_seq + 1, threadIdx.x, 256);
    starts[lp].copy(p, lp);
    if (lo != lp) starts[lo].copy(p, lo);
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5), total = tok0[p.n_seq] * p.n_heads;
    const int lane = threadIdx.x & 31;
    if (row >= total) return;
    const uint32_t G = p.n_heads / p.n_kv_heads;
    const TGKvGroupShape sp = shape_of(p, lp, nullptr, tok0), so = shape_of(p, lo, nullptr, tok0);
    const uint32_t t = row / p.n_heads, h = row % p.n_heads, kvh = h / G, sub = h % G;
    const uint32_t i = seq_of(tok0, p.n_seq, t), own = t - tok0[i];
    T* out = reinterpret_cast<T*>(p.out);
    asm volatile("" : "+l"(out));
    Acc<HD> acc(p);
    acc.run([&] {
        acc.add(row, lane);
        add_continued<HD>(p, lp, starts[lp], acc, TGKvGroupPos{0, kvh, t / sp.item_tokens, 0},
                          item_row(sp, t % sp.item_tokens, G, sub), lane);
        acc.add((uint64_t)total + row, lane);
        add_continued<HD>(p, lo, starts[lo], acc, TGKvGroupPos{i + 1, kvh, own / so.item_tokens, 0},
                          item_row(so, own % so.item_tokens, G, sub), lane);
    }, lane);
    acc.template store<T>(out, row, lane);
}

// joined: the rows of items that several CTAs worked on.  Block (b, y) merges
// query rows 16 y .. +15 of the item that CTA b leaves unfinished and began itself.
template <typename T, int HD>
__global__ void __launch_bounds__(256) group_merge_split_kernel(const __grid_constant__ TGKvGroupParams p) {
    __shared__ Starts st;
    const int line = p.own_line;
    st.copy(p, line);
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t b = blockIdx.x;
    const TGKvGroupPos s = st.at(b), e = st.at(b + 1);
    // the item that the next CTA continues, begun in this one
    if (e.seq > p.n_seq || e.tile == 0 || (tgkv_group_same_item(s, e) && s.tile > 0)) return;
    TGKvGroupPos it = e;
    it.tile = 0;
    const uint32_t G = p.n_heads / p.n_kv_heads;
    const uint32_t* tok0 = as_memory(p.tok0);
    const TGKvGroupShape sh = shape_of(p, line, nullptr, tok0);
    const uint32_t t0 = it.at * sh.item_tokens, ntok = min(sh.item_tokens, tgkv_group_tokens(&sh, it.seq) - t0);
    const uint32_t first = tok0[it.seq - 1] + t0;
    const int lane = threadIdx.x & 31;
    for (uint32_t x = blockIdx.y * 16 + (threadIdx.x >> 5); x < blockIdx.y * 16 + 16 && x < ntok * G; x += 8) {
        const uint32_t t = x / G, sub = x % G, r = item_row(sh, t, G, sub);
        Acc<HD> acc(p);
        acc.run([&] {
            acc.add((uint64_t)p.line[line].cta_rows + slot_rows(line) * (2 * b + 1) + r, lane);
            add_continued<HD>(p, line, st, acc, it, r, lane);
        }, lane);
        acc.template store<T>(reinterpret_cast<T*>(p.out), (uint64_t)(first + t) * p.n_heads + it.kvh * G + sub, lane);
    }
}

template <typename T, int HD>
int launch(const TGKvGroupParams* p, cudaStream_t st) {
    const uint32_t total = p->tok0[p->n_seq];
    static bool done[64];
    constexpr uint32_t smem = Cfg<HD>::SMEM > light::Cfg<T, HD>::SMEM ? Cfg<HD>::SMEM : light::Cfg<T, HD>::SMEM;
    cudaError_t e = allow_smem(group_kernel<T, HD>, smem, done);
    if (e != cudaSuccess) return (int)e;
    if (p->k_new && !p->append) {
        const uint64_t n = (uint64_t)total * (p->n_kv_heads * HD / 8);
        e = launch_pdl(group_append_kernel<T>, dim3((unsigned)((n + 255) / 256), 2), 256, 0, st, p);
        if (e != cudaSuccess) return (int)e;
    }
    e = launch_pdl(group_kernel<T, HD>, dim3(p->line[0].n_cta + p->line[1].n_cta), kThreads, smem, st, p);
    if (e != cudaSuccess) return (int)e;
    const TGKvGroupLine* own = &p->line[p->own_line];
    if (p->share)
        e = launch_pdl(group_merge_parts_kernel<T, HD>, dim3((total * p->n_heads + 7) / 8), 256, 0, st, p);
    else if (own->n_split)
        e = launch_pdl(group_merge_split_kernel<T, HD>, dim3(own->n_cta, p->own_line ? 1 : 16), 256, 0, st, p);
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
