// tgkv_group_light.cuh -- group attention (tgkv_group.cu) of items with few query
// rows: a decode step's tokens over their own caches, up to 16 rows of one KV
// head (10 with fp32 activations).  The part of a CTA on line 1.
//
// The products go the other way round, S^T = K Q^T and O^T += V^T P^T, with the
// rows as 16 or 32 columns: K and V tiles are the 128-row operands straight from
// the caches' layout, a softmax thread has one position and exponentiates the
// rows there are.  Bound by HBM, 512 bytes a position of 128 head dims: two
// streams take an item's alternate tiles, each with its own O^T, P^T and softmax
// warps, and join at the item's end; K and V have three 32 KB stages each.
// Decode without a prefix, 32/8 heads of 128, bf16 activations: 16 caches of
// 30000-32000 positions 292-308 us on different cards (6.6-6.9 TB/s, about the
// measured copy rate), 64 of 1000-4000 107-110 us (5.7 TB/s); fp32 activations 307
// and 113 us.  Short items are bound by their start and end, so
// what runs once an item is kept small (unrolled code costs its fetch).
// TERMS is 1 with bf16 activations; fp32 q and P enter as three bf16 terms (all 24
// bits), stacked as columns: term t of row x is column t * ROWS + x.
// Warps (384 threads): 0-3 and 4-7 the streams' softmax (thread r: position r of
// a tile; at the end head dim r), 8 TMA, 9 and 10 the streams' MMAs.
// TMEM columns: S^T of stream h [64 h, +32), O^T [128 + 64 h, +32).
// Every mbarrier wait is bounded, as in tgkv_group.cu.
#pragma once
#include "tgkv_group.cuh"

namespace tgkv {
namespace group {
namespace light {

constexpr int kTmaWarp = 8, kMmaWarp = 9;
constexpr uint32_t TM_S = 0, TM_O = 128, TM_COLS = 256;

template <typename T, int HD>
struct Cfg {
    static constexpr int TERMS = sizeof(T) == 4 ? 3 : 1;
    static constexpr int ROWS = TERMS == 3 ? 10 : TGKV_GROUP_LIGHT_ROWS;
    static constexpr int N = TERMS == 3 ? 32 : 16;                     // the products' columns
    static_assert(TERMS * ROWS <= N && ROWS <= TGKV_GROUP_LIGHT_ROWS, "columns");
    static constexpr uint32_t kTile = (uint32_t)(HD / 64) * kBlock;    // one K or V tile
    static constexpr uint32_t kSmall = N * 128;                        // N rows x 64 bf16, swizzled
    static constexpr int kStages = HD == 128 ? 3 : 6;                  // per ring: 192 KB in all
    static constexpr uint32_t OFF_K = 0, OFF_V = kStages * kTile;
    static constexpr uint32_t OFF_Q = 2 * kStages * kTile;             // HD / 64 blocks
    static constexpr uint32_t OFF_P = OFF_Q + (HD / 64) * kSmall;      // [2 streams] 2 blocks of 64 positions
    static constexpr int B_KFULL = 0, B_KEMPTY = kStages, B_VFULL = 2 * kStages, B_VEMPTY = 3 * kStages;
    // [2 streams], one phase per tile:
    static constexpr int B_SFULL = 4 * kStages;      // S^T is in TMEM, and the stream's last PV complete
    static constexpr int B_PFULL = B_SFULL + 2;      // P is written, O^T rescaled (128 arrivals)
    static constexpr int B_PVDONE = B_PFULL + 2;
    static constexpr int B_QFULL = B_PVDONE + 2;     // a piece's Q is in shared memory (256 arrivals)
    static constexpr int B_QEMPTY = B_QFULL + 1;     // every S of a piece is complete
    static constexpr int kBars = B_QEMPTY + 1;
    static constexpr uint32_t OFF_BAR = OFF_P + 4 * kSmall;
    static constexpr uint32_t OFF_RED = OFF_BAR + kBars * 8;           // [2][4 warps][16], [2][16] maxima, [2][2][16]
    static constexpr uint32_t OFF_SLOT = OFF_RED + (128 + 32 + 64) * 4;
    static constexpr uint32_t OFF_TAB = OFF_SLOT + 16;                 // tok0, old_len
    static constexpr uint32_t SMEM = OFF_TAB + (2 * TGKV_MAX_ITEMS + 1) * 4 + 1024;    // slack to align the base
    static_assert(SMEM <= 232448, "shared memory per CTA");
};

// All of a stream's softmax threads; of both streams'.
__device__ __forceinline__ void stream_sync(int h) { asm volatile("bar.sync %0, 128;" ::"r"(1 + h) : "memory"); }
__device__ __forceinline__ void streams_sync() { asm volatile("bar.sync 3, 256;" ::: "memory"); }
// stream_sync that tells whether any thread said yes.
__device__ __forceinline__ bool stream_any(int h, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred pi, po;\n\t"
        "setp.ne.u32 pi, %1, 0;\n\t"
        "bar.red.or.pred po, %2, 128, pi;\n\t"
        "selp.u32 %0, 1, 0, po;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(1 + h)
        : "memory");
    return r != 0;
}

// The columns of a product that have rows.
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&v)[32]) {
    tmem_ld32(taddr, v);
    tmem_wait_ld(v);
}
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&v)[16]) {
    tmem_ld16(taddr, v);
    tmem_wait_ld16(v);
}
__device__ __forceinline__ void tmem_st_cols(uint32_t addr, const uint32_t (&w)[32]) { tmem_st32(addr, w); }
__device__ __forceinline__ void tmem_st_cols(uint32_t addr, const uint32_t (&w)[16]) { tmem_st16(addr, w); }

// One column of this thread's TMEM lane.
__device__ __forceinline__ float tmem_ld1(uint32_t taddr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v)::"memory");
    return __uint_as_float(v);
}
// A row's sums over its terms.
template <int TERMS, int ROWS>
__device__ __forceinline__ float tmem_ld_row(uint32_t taddr) {
    if constexpr (TERMS == 1) return tmem_ld1(taddr);
    return (tmem_ld1(taddr) + tmem_ld1(taddr + ROWS)) + tmem_ld1(taddr + 2 * ROWS);
}

template <typename T, int HD>
__device__ __forceinline__ void run(const TGKvGroupParams& p, uint32_t cta_index, unsigned char* smem_raw) {
    using C = Cfg<T, HD>;
    constexpr int TERMS = C::TERMS, ROWS = C::ROWS, N = C::N;
    // fp32 sums: at most 16 tiles per accumulator (see tgkv_group.cu)
    constexpr uint32_t kMost = TERMS == 3 ? 32 : 0;
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
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(&bar[C::B_SFULL + h], 1);
            mbar_init(&bar[C::B_PFULL + h], 128);
            mbar_init(&bar[C::B_PVDONE + h], 1);
        }
        mbar_init(&bar[C::B_QFULL], 256);
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
    const TGKvGroupShape sh = shape_of(p, 1, old_len, tok0);
    // Everything above overlaps the previous kernel on the stream.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    Pieces pc(sh, start_of(p, 1, cta_index), start_of(p, 1, cta_index + 1), kMost);
    if (warp == kTmaWarp) {
        uint32_t n = 0, nv = 0;                  // K and V tiles issued
        bool ok = true;
        for (; ok && pc.more(); pc.next(sh, kMost)) {
            const uint32_t seq = pc.at.seq, npre = tgkv_group_prefix_tiles(&sh, seq);
            const int x = (int)(pc.at.kvh * HD);
            for (uint32_t j = pc.j0; ok && j < pc.j1; ++j) {
                const bool own = j >= npre;
                const uint64_t map = p.tmaps + 128ull * (own ? seq - 1 : p.n_seq);
                const uint32_t y = (own ? j - npre : j) * kPos;
                if (p.append && own) {
                    // the new rows of this KV head and tile: stored here, where alone they are
                    // loaded, 8 elements a lane
                    const uint32_t first = old_len[seq - 1], r0 = max(y, first),
                                   r1 = min(y + kPos, first + tgkv_group_tokens(&sh, seq));
                    if (r0 < r1) {
                        const uint64_t kv_dim = (uint64_t)p.n_kv_heads * HD;
                        const TGKvRowCache c = p.table[seq - 1];
                        for (uint32_t i = lane; i < (r1 - r0) * (HD / 4); i += 32) {
                            const uint32_t v = i % (HD / 4), half = v / (HD / 8), e = v % (HD / 8) * 8 + pc.at.kvh * HD;
                            const uint32_t row = r0 + i / (HD / 4);
                            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(c.base) +
                                                      (half * c.max_seq + row) * kv_dim + e) =
                                row_part(reinterpret_cast<const T*>(half ? p.v_new : p.k_new) +
                                         (uint64_t)(tok0[seq - 1] + (row - first)) * kv_dim + e);
                        }
                        asm volatile("fence.proxy.async.global;" ::: "memory");
                        __syncwarp();
                    }
                }
                const uint32_t s = n % C::kStages, ph = (n / C::kStages - 1) & 1u;
                if (lane == 0) {
                    if (n >= C::kStages) ok = mbar_wait(&bar[C::B_KEMPTY + s], ph);
                    if (ok) {
                        mbar_arrive_expect_tx(&bar[C::B_KFULL + s], C::kTile);
                        for (int b = 0; b < HD / 64; ++b)
                            tma_load_3d(base + C::OFF_K + s * C::kTile + b * kBlock, map, x + 64 * b, (int)y, 0,
                                        &bar[C::B_KFULL + s]);
                        ++n;
                        if (nv >= C::kStages) ok = mbar_wait(&bar[C::B_VEMPTY + s], ph);
                    }
                    if (ok) {
                        mbar_arrive_expect_tx(&bar[C::B_VFULL + s], C::kTile);
                        for (int b = 0; b < HD / 64; ++b)
                            tma_load_3d(base + C::OFF_V + s * C::kTile + b * kBlock, map, x + 64 * b, (int)y, 1,
                                        &bar[C::B_VFULL + s]);
                        ++nv;
                    }
                }
                ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            }
        }
        if (lane == 0) {
            // every copy has landed before the CTA may end (at once in a normal run)
            for (uint32_t i = n > C::kStages ? n - C::kStages : 0; i < n; ++i)
                ok = mbar_wait(&bar[C::B_KFULL + i % C::kStages], (i / C::kStages) & 1u) && ok;
            for (uint32_t i = nv > C::kStages ? nv - C::kStages : 0; i < nv; ++i)
                ok = mbar_wait(&bar[C::B_VFULL + i % C::kStages], (i / C::kStages) & 1u) && ok;
            if (!ok) atomicExch(p.err, kErrTimeout);
        }
        __syncwarp();
    } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
        if (lane == 0) {
            // Step k of a piece, K/V tile g0 + k, belongs to stream k % 2.  PV as soon as P is
            // there, then the next S^T (its buffer has been read by then, and a commit behind it
            // also tells that PV is complete).  Both warps pass every phase of the rings and of
            // Q, in order, so that a parity always means the phase it is waited for.
            constexpr uint32_t id_s = umma_idesc_bf16(kRows, N, 0, 0);
            constexpr uint32_t id_pv = umma_idesc_bf16(kRows, N, 1, 0);
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
            const uint64_t qd = umma_desc_sw128(sbase + C::OFF_Q, 16, 1024);
            const uint64_t pd = umma_desc_sw128(sbase + C::OFF_P + h * 2 * C::kSmall, 16, 1024);
            for (; ok && pc.more(); pc.next(sh, kMost), ++it) {
                const uint32_t steps = pc.j1 - pc.j0;
                ok = mbar_wait(&bar[C::B_QFULL], it & 1u);
                tc_fence_after();
                if (h >= steps) mbar_arrive(&bar[C::B_QEMPTY]);
                auto issue_s = [&](uint32_t k) {
                    const uint32_t g = g0 + k, s = g % C::kStages;
                    pass(C::B_KFULL, C::B_KEMPTY, ks, g);
                    ok = ok && mbar_wait(&bar[C::B_KFULL + s], (g / C::kStages) & 1u);
                    if (!ok) return;
                    tc_fence_after();
                    const uint64_t kd = umma_desc_sw128(sbase + C::OFF_K + s * C::kTile, 16, 1024);
#pragma unroll
                    for (uint32_t d = 0; d < HD / 16; ++d) {
                        const uint32_t in = (d & 3u) * 32u;
                        umma_ss(tmem + TM_S + h * 64u, kd + (((d >> 2) * kBlock + in) >> 4),
                                qd + (((d >> 2) * C::kSmall + in) >> 4), id_s, d != 0);
                    }
                    umma_commit(&bar[C::B_SFULL + h]);
                    umma_commit(&bar[C::B_KEMPTY + s]);
                    ks = g + 1;
                    if (k + 2 >= steps) umma_commit(&bar[C::B_QEMPTY]);
                    if (k + 1 < steps) pass(C::B_KFULL, C::B_KEMPTY, ks, g + 2);
                };
                if (ok && h < steps) issue_s(h);
                for (uint32_t k = h; ok && k < steps; k += 2, ++n) {
                    const uint32_t g = g0 + k, s = g % C::kStages;
                    pass(C::B_VFULL, C::B_VEMPTY, vs, g);
                    ok = ok && mbar_wait(&bar[C::B_PFULL + h], n & 1u) &&
                         mbar_wait(&bar[C::B_VFULL + s], (g / C::kStages) & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    // V^T: A, MN-major, 16 positions a step (with 64 head dims the upper 64 lanes
                    // get products of what follows in shared memory; nobody reads them)
                    const uint64_t vd = umma_desc_sw128(sbase + C::OFF_V + s * C::kTile, kBlock, 1024);
#pragma unroll
                    for (uint32_t kk = 0; kk < 8; ++kk)
                        umma_ss(tmem + TM_O + h * 64u, vd + ((kk * 16u * 128u) >> 4),
                                pd + (((kk >> 2) * C::kSmall + (kk & 3u) * 32u) >> 4), id_pv, k > 1 || kk != 0);
                    umma_commit(&bar[C::B_PVDONE + h]);
                    umma_commit(&bar[C::B_VEMPTY + s]);
                    vs = g + 1;
                    if (k + 2 < steps) issue_s(k + 2);
                }
                g0 += steps;
                pass(C::B_KFULL, C::B_KEMPTY, ks, g0);
                pass(C::B_VFULL, C::B_VEMPTY, vs, g0);
            }
            if (!ok) atomicExch(p.err, kErrTimeout);
        }
        __syncwarp();
    } else if (warp < kTmaWarp) {
        const int quarter = warp & 3, h = warp >> 2, r = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t ts = lanes + TM_S + (uint32_t)h * 64u, to = lanes + TM_O;
        const float scale = p.qscale;
        float* red_all = reinterpret_cast<float*>(base + C::OFF_RED);
        float* red = red_all + h * 64;           // [4 warps][16]
        float* maxima = red_all + 128;           // [2 streams][16]
        float* joint = red_all + 160 + h * 32;   // [2][16]: (m, l) of rows this stream brings out
        const uint32_t total_rows = tok0[p.n_seq] * p.n_heads;
        uint32_t g0 = 0, it = 0, n = 0;          // K/V tiles of earlier pieces; pieces; this stream's steps
        bool ok = true;
        // row x of an item, from its first row: its token's, one of G heads
        auto row_of = [&](uint64_t row0, uint32_t x, uint32_t tokens) -> uint64_t {
            return tokens == 1 ? row0 + x : row0 + (uint64_t)(x / G) * p.n_heads + x % G;
        };
        // q of a piece, as TERMS bf16 rows each: two dims a thread, the streams take every other
        // row.  Loaded while the piece before is worked on, stored once that one's last S^T is made.
        constexpr int kMine = (ROWS + 1) / 2;
        float2 qv[kMine];
        uint32_t q_rows = 0;
        auto load_q = [&](const Pieces& a) {
            if (!a.more()) return;
            const ItemRows ir(sh, a);
            q_rows = ir.tokens * G;
            const uint64_t row0 = (uint64_t)((a.at.seq ? tok0[a.at.seq - 1] : 0) + a.at.at * sh.item_tokens) * p.n_heads +
                                  a.at.kvh * G;
            if (r >= HD / 2) return;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const uint32_t x = 2 * i + h;
                if (x >= q_rows) break;
                const uint64_t e = row_of(row0, x, ir.tokens) * HD + 2 * r;
                if constexpr (TERMS == 3) qv[i] = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(p.q) + e);
                else qv[i].x = __uint_as_float(*reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint16_t*>(p.q) + e));
            }
        };
        auto store_q = [&](uint32_t piece) {
            if (ok && piece > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_QEMPTY], (piece - 1) & 1u));
            if (r < HD / 2) {
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const uint32_t x = 2 * i + h;
                    if (x >= q_rows) break;
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const uint32_t w = TERMS == 3 ? cvt_bf16x2(qv[i].x, qv[i].y) : __float_as_uint(qv[i].x);
                        const uint32_t c = t * ROWS + x;
                        *reinterpret_cast<uint32_t*>(base + C::OFF_Q + (r >> 5) * C::kSmall + c * 128 +
                                                     ((((uint32_t)r & 31u) >> 2) ^ (c & 7u)) * 16 + (r & 3) * 4) = w;
                        qv[i].x -= lo_f(w);
                        qv[i].y -= hi_f(w);
                    }
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&bar[C::B_QFULL]);
        };
        load_q(pc);
        if (pc.more()) store_q(0);
        while (pc.more()) {
            const ItemRows pr(sh, pc);
            const uint32_t seq = pc.at.seq, R = pr.tokens * G, t0 = pc.at.at * sh.item_tokens;
            const uint32_t own_min = seq ? old_len[seq - 1] + t0 + 1 : 0;                // rows that token 0 sees
            const uint64_t row0 = (uint64_t)((seq ? tok0[seq - 1] : 0) + t0) * p.n_heads + pc.at.kvh * G;
            const uint32_t steps = pc.j1 - pc.j0;
            const Pieces cur = pc;
            pc.next(sh, kMost);
            load_q(pc);
            float m[ROWS], l[ROWS];              // of the scaled scores, log2 domain; l: this thread's positions
#pragma unroll
            for (int x = 0; x < ROWS; ++x) { m[x] = -INFINITY; l[x] = 0.f; }
            for (uint32_t k = (uint32_t)h; k < steps; k += 2, ++n) {
                const uint32_t j = cur.j0 + k, pos = pr.pos(j), rows = pr.rows(j) - pos;
                const bool own = pr.own(j);
                const int first = (int)((own ? own_min : p.prefix_len) - pos);           // of the tile, that token 0 sees
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_SFULL + h], n & 1u));
                const uint32_t lo = (uint32_t)max(first, 0);
                if (ok && lo < kPos) {
                    // V rows that no query sees may hold anything, and those that only some see are
                    // cleared of what is not finite, before PV reads them
                    const uint32_t g = g0 + k, s = g % C::kStages;
                    ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_VFULL + s], (g / C::kStages) & 1u));
                    if (ok) clear_unseen<HD, 128>(base + C::OFF_V + s * C::kTile, lo, rows, kPos, r, flag);
                    __syncwarp();
                }
                uint32_t v[N];
                float sc[ROWS];
                bool grow = false;
                if (ok) {
                    tc_fence_after();
                    tmem_ld_cols(ts, v);
                }
                int lim = first, sub = 0;        // positions that row x's token sees
#pragma unroll
                for (int x = 0; x < ROWS; ++x) {
                    if ((uint32_t)x >= R) break;
                    float s = __uint_as_float(v[x]);
                    if constexpr (TERMS == 3) s = (s + __uint_as_float(v[ROWS + x])) + __uint_as_float(v[2 * ROWS + x]);
                    sc[x] = r < lim ? s * scale : -INFINITY;
                    grow |= !(sc[x] <= m[x] + 8.f) && sc[x] != -INFINITY;
                    if (own && ++sub == (int)G) { sub = 0; ++lim; }
                }
                // the running maxima move only when one is exceeded by more than 2^8 (or NaN)
                if (stream_any(h, grow)) {
#pragma unroll
                    for (int x = 0; x < ROWS; ++x) {
                        if ((uint32_t)x >= R) break;
                        float a = sc[x];
#pragma unroll
                        for (int o = 16; o >= 1; o >>= 1) a = max3(a, __shfl_xor_sync(0xffffffffu, a, o), a);
                        if (lane == 0) red[quarter * 16 + x] = a;
                    }
                    stream_sync(h);
                    uint32_t ov[N];
                    const bool scale_o = k > 1;  // O^T holds the stream's earlier tiles, all complete before this S^T
                    if (ok && scale_o) tmem_ld_cols(to + (uint32_t)h * 64u, ov);
#pragma unroll
                    for (int x = 0; x < ROWS; ++x) {
                        if ((uint32_t)x >= R) break;
                        const float a = max3(max3(red[x], red[16 + x], red[32 + x]), red[48 + x], m[x]);
                        const float alpha = m[x] == -INFINITY ? 0.f : ex2_approx(m[x] - a);
                        m[x] = a;
                        l[x] *= alpha;
#pragma unroll
                        for (int t = 0; t < TERMS; ++t)
                            ov[t * ROWS + x] = __float_as_uint(__uint_as_float(ov[t * ROWS + x]) * alpha);
                    }
                    if (ok && scale_o) {
                        tmem_st_cols(to + (uint32_t)h * 64u, ov);
                        tmem_wait_st();
                    }
                    stream_sync(h);              // red is free again
                }
                if (ok) {
                    const uint32_t pb = sbase + C::OFF_P + ((uint32_t)h * 2 + ((uint32_t)r >> 6)) * C::kSmall;
                    const uint32_t c = ((uint32_t)r & 63u) >> 3, e = ((uint32_t)r & 7u) * 2u;
#pragma unroll
                    for (int x = 0; x < ROWS; ++x) {
                        if ((uint32_t)x >= R) break;
                        float w = m[x] == -INFINITY ? 0.f : ex2_approx(sc[x] - m[x]);
                        l[x] += w;
#pragma unroll
                        for (int t = 0; t < TERMS; ++t) {
                            const uint32_t b = cvt_bf16x2(w, 0.f) & 0xffffu, q = t * ROWS + x;
                            asm volatile("st.shared.u16 [%0], %1;" ::"r"(pb + q * 128u + ((c ^ (q & 7u)) << 4) + e),
                                         "h"((uint16_t)b) : "memory");
                            w -= lo_f(b);
                        }
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before();
                mbar_arrive(&bar[C::B_PFULL + h]);
            }
            g0 += steps;
            ++it;
            if (pc.more()) store_q(it);          // the next piece's first scores are made meanwhile

            // ---- the rows' sums, over the stream's threads, then both streams
            if (ok && (uint32_t)h < steps) ok = __all_sync(0xffffffffu, mbar_wait(&bar[C::B_PVDONE + h], (n - 1) & 1u));
#pragma unroll
            for (int x = 0; x < ROWS; ++x) {
                if ((uint32_t)x >= R) break;
                float a = l[x];
#pragma unroll
                for (int o = 16; o >= 1; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
                if (lane == 0) {
                    red[quarter * 16 + x] = a;
                    if (quarter == 0) maxima[h * 16 + x] = m[x];
                }
            }
            tc_fence_before();
            streams_sync();
            tc_fence_after();
            const bool whole = cur.first == 0 && cur.j1 == cur.nt && !p.share;
            const bool again = TERMS == 3 && cur.j0 > cur.first;                         // adds to the item's earlier piece here
            const uint64_t cta = (uint64_t)p.line[1].cta_rows +
                                 TGKV_GROUP_LIGHT_ROWS * (2u * cta_index + (cur.first > 0 ? 0u : 1u));
            // A loop, not unrolled: code that runs once an item costs its fetch.  The streams take
            // every other row.
#pragma unroll 1
            for (uint32_t x = (uint32_t)h; ok && x < R; x += 2) {
                const float a = tmem_ld_row<TERMS, ROWS>(to + x), b = tmem_ld_row<TERMS, ROWS>(to + 64 + x);
                const float ma = maxima[x], mb = maxima[16 + x];
                float M = max3(ma, mb, ma);
                const float wa = ma == -INFINITY ? 0.f : ex2_approx(ma - M), wb = mb == -INFINITY ? 0.f : ex2_approx(mb - M);
                const float* ra = red_all + x;
                float L = wa * ((ra[0] + ra[16]) + (ra[32] + ra[48])) + wb * ((ra[64] + ra[80]) + (ra[96] + ra[112]));
                // (a stream that had no tile left O^T as it was; a weight that is 0 takes part, since
                // 0 x Inf is NaN)
                float o = a * wa;
                if (steps > 1) o += b * wb;
                if (*flag && seq && r < HD) {
                    // what the piece's V rows hold that is not finite, of those the row sees
                    const uint32_t f0 = pr.own(cur.j0) ? pr.pos(cur.j0) : 0u, f1 = pr.own(cur.j1) ? pr.pos(cur.j1) : 0u;
                    const float y = cache_non_finite(p.table + (seq - 1), p.n_kv_heads * HD, cur.at.kvh * HD + r,
                                                     max(own_min, f0), min(own_min + x / G, f1));
                    if (y != 0.f) o += y;
                }
                const uint64_t row = row_of(row0, x, pr.tokens);
                const uint64_t slot = cur.first > 0 || !p.share ? cta + x : (seq ? total_rows : 0u) + row;
                if (again) {
                    const float2 old = *reinterpret_cast<const float2*>(p.part_ml + slot * 2);
                    const float M2 = max3(M, old.x, M);
                    const float wn = M == -INFINITY ? 0.f : ex2_approx(M - M2), wo = old.x == -INFINITY ? 0.f : ex2_approx(old.x - M2);
                    if (r < HD) o = o * wn + p.part_o[slot * HD + r] * wo;
                    L = L * wn + old.y * wo;
                    M = M2;
                }
                if (r < HD) {
                    if (!whole) p.part_o[slot * HD + r] = o;
                    else if constexpr (TERMS == 3) reinterpret_cast<float*>(p.out)[row * HD + r] = o / L;
                    else reinterpret_cast<uint16_t*>(p.out)[row * HD + r] = (uint16_t)(cvt_bf16x2(o / L, 0.f) & 0xffffu);
                }
                joint[x] = M;                    // the same from every thread
                joint[16 + x] = L;
                __syncwarp();
            }
            tc_fence_before();
            streams_sync();                      // O^T, the sums and the slots' (m, l) have been read
            if (!whole && ok && (uint32_t)r < R && (r & 1) == h) {
                const uint64_t row = row_of(row0, (uint32_t)r, pr.tokens);
                const uint64_t slot = cur.first > 0 || !p.share ? cta + r : (seq ? total_rows : 0u) + row;
                *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(joint[r], joint[16 + r]);
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

}  // namespace light
}  // namespace group
}  // namespace tgkv
