// sc_attention_tile.cu — the shared-prefix attention for many rows of one KV head at once, on the
// 5th-generation tensor cores.
//
// A block takes 256 rows (two tiles of 128 (token, head) rows of one KV head) against a run of
// tokens in tiles of 128: prefix tokens, then tokens of the sequence's own cache.  Per tile pair,
//   S = Q K^T         128 x 128 x D, fp32 accumulators in tensor memory,
//   P = 2^(s - m)     one thread a row: no shuffles; written over S as 16 bits (half a step of the
//                     type off; their error as a second product, which attend_stream has, costs the
//                     softmax's instructions: prompts 470 -> 635 us, paged decode 47 -> 57),
//   O += P V          A operand from tensor memory, fp32 accumulators in tensor memory.
// Two row tiles take turns: while the tensor cores work on one, eight warps turn the other's
// scores into weights.  (With one row tile, two token tiles' scores do.)  The running maximum that scales
// O is only raised when a score passes it by 2^8 (float16: 2^7), so O is rarely rescaled; weights above
// one and their fp32 sums lose nothing.
//
// Roles: warps 0-3 and 4-7 the softmax of row tile 0 and 1, warps 8-10 the copies, warp 11 issues
// the products.  Tiles come by TMA (4-D tensor maps of prefix, caches or page pool; a page's piece
// is a box of gcd(page, 128) rows) in the 128-byte swizzle that the matrix descriptors name; what
// a map cannot say (pages of fewer than 8 rows' alignment, expanded strides) and the last values
// of a cache, whose rows behind its length must read as zero, by cp.async in the same order.
// (All tiles by cp.async from these three warps: 4.3 us a step, their address arithmetic the
// bound.)  Tensor memory: S0, S1 (128 columns each), O0, O1 (D columns each).  Every wait has a
// limit; a wait that runs out sets a status bit and the block leaves.
#include <math.h>

#include "sc_tensor.cuh"
#include "sc_tile_waits.h"

namespace sc {
namespace {

constexpr int kTThreads = 384;
constexpr int kLoadWarps = 3;
constexpr int kRowTile = 128;
constexpr int kTokTile = 128;
// log2: how far a score may pass the maximum in use, and by how much weights are lifted.  float16 ends at
// 2^16 and begins at 2^-24, so that lifted its weights count down to 2^-33 of the largest (as they are,
// 2^17 tokens 2^25 below the largest would be lost: 2^-8 of the sum); bfloat16 has room on both sides.
// 24 sequences of float16 behind 32,768: 47 us, with 2^4 and 2^11 49 (O is rescaled more often).
template <typename T>
constexpr float kRaise = std::is_same<T, __half>::value ? 7.f : 8.f;
template <typename T>
constexpr float kLiftTile = std::is_same<T, __half>::value ? 8.f : 0.f;
constexpr float kFar = 4194304.f;  // 2^22: scores of such a maximum are 1/4 off from their exact product
template <typename T>
constexpr float kUnliftTile = std::is_same<T, __half>::value ? 0x1p-8f : 1.f;  // of what goes out as a part or lse

template <int DP>
struct TileShape {
    static constexpr int kTile = 128 * DP * 2;  // bytes of 128 rows
    static constexpr int kStages = DP == 128 ? 5 : 8;
    static constexpr int kSmem = (2 + kStages) * kTile + 1024;  // + alignment
};

struct TileParams {
    AttnParams a;
    int32_t per_seq;   // rows are those of one sequence, and its own cache follows the prefix
    int32_t tiles;     // 256-row tiles of all rows together (not per_seq)
    int32_t splits;    // parts of the token axis (per_seq: of the last round's units, at most)
    int32_t sms;       // blocks of a round
    int32_t tma_p, tma_c;  // whether the maps below are in use
    int32_t box_c;         // rows of a box of the own caches
    CUtensorMap kp, vp, kc, vc;
};

// Byte offset of 16-byte chunk c (of a 128-row tile's row r).
__device__ __forceinline__ uint32_t tile_chunk(int r, int c) {
    return static_cast<uint32_t>((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// A sequence's rows in units of 256 of one KV head (per_seq).  All units take equally long, so they
// run in rounds of one unit an SM; those of the last, unfilled round are split over the SMs that
// would be idle: into `parts` parts each, whose sums join_tail adds up.  Called by whole warps.
struct Round {
    int units, full, rem, parts;  // units before the last round, in it, and parts of each there
};
__device__ __forceinline__ int units_of(const AttnParams& p, const Starts& starts, int b) {
    int tok0, n;
    starts.of(b, tok0, n);
    return (n * p.G + 2 * kRowTile - 1) / (2 * kRowTile);
}
__device__ __forceinline__ Round rounds(const TileParams& tp, const Starts& starts) {
    const AttnParams& p = tp.a;
    const int lane = threadIdx.x & 31;
    int n = 0;
    if (p.cu_q == nullptr)
        n = p.B * units_of(p, starts, 0);
    else
        for (int b0 = 0; b0 < p.B; b0 += 32)
            n += __reduce_add_sync(0xffffffffu, b0 + lane < p.B ? units_of(p, starts, b0 + lane) : 0);
    Round r;
    r.units = n * p.Hkv;
    r.full = r.units / tp.sms * tp.sms;
    r.rem = r.units - r.full;
    r.parts = r.rem ? max(1, min(tp.splits, tp.sms / r.rem)) : 1;
    return r;
}
// Unit u as sequence, head and row tile; units of a sequence lie together.
__device__ __forceinline__ void locate(const AttnParams& p, const Starts& starts, int u, int& b, int& h, int& rt) {
    const int lane = threadIdx.x & 31;
    int in = u, own = 0;
    if (p.cu_q == nullptr) {
        own = units_of(p, starts, 0);
        b = u / (own * p.Hkv);
        in = u - b * own * p.Hkv;
    } else {
        for (int b0 = 0;; b0 += 32) {
            const int n = b0 + lane < p.B ? units_of(p, starts, b0 + lane) : 0;
            int upto = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += y;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, in < upto * p.Hkv);
            if (past || b0 + 32 >= p.B) {
                const int at = past ? __ffs(past) - 1 : 31;
                in -= __shfl_sync(0xffffffffu, upto - n, at) * p.Hkv;
                own = __shfl_sync(0xffffffffu, n, at);
                b = b0 + at;
                break;
            }
            in -= __shfl_sync(0xffffffffu, upto, 31) * p.Hkv;
        }
    }
    h = own ? in / own : 0;
    rt = in - h * own;
}

// What take_out_odd kept, added to a warp's rows in tensor memory.
template <int DP>
__device__ __noinline__ void add_odd_tmem(uint32_t o_at, const int* first, int limit) {
#pragma unroll 1
    for (int c = 0; c < DP; c += 16) {
        uint32_t o[16];
        tmem_ld16(o_at + c, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            float v = __uint_as_float(o[e]);
            if (first[c + e] < limit) v += -kNegInf;
            if (first[DP + c + e] < limit) v += kNegInf;
            o[e] = __float_as_uint(v);
        }
        tmem_st16(o_at + c, o);
    }
    tmem_wait_st();
}

template <typename T, int DP>
__global__ void __launch_bounds__(kTThreads, 1) attend_tiles(const __grid_constant__ TileParams tp) {
    using Shape = TileShape<DP>;
    constexpr int TILE = Shape::kTile, NST = Shape::kStages;
    constexpr int CPR = DP / 8;
    const AttnParams& p = tp.a;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t s_bars[2 * NST + 8];
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    __shared__ int s_any_bad, s_copy;
    // Tokens of a tile whose page is there.  A tile's keys may be loaded while the softmax is still at
    // the tile three (five stages) or six (eight) before it.
    constexpr int kOks = NST == 5 ? 4 : 8;
    __shared__ unsigned char s_ok[kOks][kTokTile];
    __shared__ int s_odd[2 * DP], s_any_odd;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    int b = 0, h, rt, split = 0, splits, slot = 0;
    int tok0 = 0, n_tok, len = 0;
    let_next_start();
    if (tp.per_seq) {
        // Sequences of no rows have no block that would report what is wrong with them.
        if (blockIdx.x == 0 && warp == 10 && p.cu_q != nullptr && p.status)
            report_sequences(p.cu_q, p.B, p.N, p.nq, p.cap ? p.cache_lens : nullptr, p.cap, p.status);
        const Starts starts(p);
        const Round r = rounds(tp, starts);
        int u = blockIdx.x;
        splits = 1;
        if (u >= r.full) {
            slot = u - r.full;
            if (slot >= r.rem * r.parts) {
                wait_for_previous();
                return;
            }
            splits = r.parts;
            split = slot % splits;
            u = r.full + slot / splits;
        }
        locate(p, starts, u, b, h, rt);
        sequence_tokens(p, starts, b, tok0, n_tok);
        len = p.cap ? cache_length(p, b) : 0;
    } else {
        int u = blockIdx.x;
        splits = tp.splits;
        split = u % splits;
        u /= splits;
        rt = u % tp.tiles;
        h = u / tp.tiles;
        n_tok = used_tokens(p);
    }
    const bool direct = splits == 1 && (tp.per_seq || (p.n_pp == 1 && p.B == 0));
    const int rows = n_tok * p.G;
    const int r0 = rt * 2 * kRowTile;
    if (r0 >= rows) {
        wait_for_previous();
        return;
    }
    const int n_rows = min(2 * kRowTile, rows - r0);
    const int n_q = n_rows > kRowTile ? 2 : 1;

    // Token tiles: the prefix's, then the own cache's that the last row sees.
    const int see = len - n_tok;
    const int vis = max(0, min(len, see + static_cast<int>(fdiv(r0 + n_rows - 1, p.div_G)) + 1));
    const int whole = min(len, see + static_cast<int>(fdiv(r0, p.div_G)) + 1);  // tokens all rows see
    const int tiles_p = (p.P + kTokTile - 1) / kTokTile;
    const int tiles_all = tiles_p + (vis + kTokTile - 1) / kTokTile;
    const int per = (tiles_all + splits - 1) / splits;
    const int first = split * per;
    const int n_tiles = max(0, min(per, tiles_all - first));
    // Where row r of the unit goes as a part: per_seq, its slot of 256 rows; else its place in the call.
    auto part_at = [&](int r) -> int64_t {
        if (tp.per_seq) return static_cast<int64_t>(slot) * (2 * kRowTile) + r;
        const int j = static_cast<int>(fdiv(r0 + r, p.div_G));
        return (static_cast<int64_t>(split) * p.N + tok0 + j) * p.Hq + h * p.G + r0 + r - j * p.G;
    };

    if (n_tiles == 0) {
        if (direct) {
            for (int i = threadIdx.x; i < n_rows * (p.D / 8); i += kTThreads) {
                const int r = i / (p.D / 8), c = i - r * (p.D / 8);
                const int j = static_cast<int>(fdiv(r0 + r, p.div_G));
                T* dst = static_cast<T*>(p.out) + (tok0 + j) * p.o_t +
                         (h * p.G + r0 + r - j * p.G) * p.o_h + c * 8;
                *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
            }
        }
        for (int r = threadIdx.x; r < n_rows; r += kTThreads) {
            const int j = static_cast<int>(fdiv(r0 + r, p.div_G));
            const int64_t row = static_cast<int64_t>(tok0 + j) * p.Hq + h * p.G + r0 + r - j * p.G;
            if (!direct)
                p.part_ml[part_at(r)] = make_float2(kNegInf, 0.f);
            else if (p.lse)
                p.lse[row] = kNegInf;
        }
        wait_for_previous();
        return;
    }

    const uint32_t s_base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t s_q = s_base, s_ring = s_base + 2 * TILE;
    const uint32_t bars = smem_addr(s_bars);
    const uint32_t q_full = bars;
    auto full = [&](int s) { return bars + 8u * (1 + s); };
    auto empty = [&](int s) { return bars + 8u * (1 + NST + s); };
    auto s_full = [&](int q) { return bars + 8u * (1 + 2 * NST + q); };
    auto p_full = [&](int q) { return bars + 8u * (3 + 2 * NST + q); };
    auto o_full = [&](int q) { return bars + 8u * (5 + 2 * NST + q); };
    const uint32_t drained = bars + 8u * (7 + 2 * NST);
    volatile int* gave_up = &s_gave_up;

    if (p.D < DP) {  // columns that no copy writes
        for (int i = threadIdx.x; i < (2 + NST) * TILE / 16; i += kTThreads)
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(s_base + 16u * i), "r"(0)
                         : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }
    if (warp == 8 && lane == 0) {
        bar_init(q_full, kTThreads / 32);
        bar_init(drained, 1);
        for (int s = 0; s < NST; ++s) {
            bar_init(full(s), 1);
            bar_init(empty(s), 1);
        }
        for (int q = 0; q < 2; ++q) {
            bar_init(s_full(q), 1);
            bar_init(p_full(q), 4);
            bar_init(o_full(q), 1);
        }
        s_gave_up = 0;
        s_any_bad = 0;
        s_any_odd = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 2 * DP) s_odd[threadIdx.x] = kNoToken;
    // The first tiles of the prefix are on their way before anything else.
    const int n_loads = 2 * n_tiles;  // K0 V0 K1 V1 ...
    const int early = tp.tma_p ? min(min(n_loads, NST), 2 * max(0, tiles_p - first)) : 0;
    auto load_prefix = [&](int i) {
        const uint32_t bar = full(i % NST);
        if (lane == 0) bar_expect(bar, TILE);
        __syncwarp();
        if (lane < CPR / 8)
            tma_load(s_ring + i % NST * TILE + lane * 16384, i & 1 ? &tp.vp : &tp.kp, bar, lane * 64,
                     (first + (i >> 1)) * kTokTile, h, 0);
    };
    if (warp == 8) {
        __syncwarp();
        for (int i = 0; i < early; ++i) load_prefix(i);
    }
    if (warp == 11) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_addr(&s_tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // Chunks of eight columns: a warp-wide copy covers 4 rows x 8 chunks of one panel.
    const int sub = lane >> 3, c8 = lane & 7;
    for (int g = warp; g < n_q * 32; g += kTThreads / 32) {
        const int r = g * 4 + sub;
        const bool in = r < n_rows;
        const int row = in ? r0 + r : r0;
        const int j = static_cast<int>(fdiv(row, p.div_G));
        const T* src = static_cast<const T*>(p.q) + (tok0 + j) * p.q_t + (h * p.G + row - j * p.G) * p.q_h;
        const uint32_t dst = s_q + (r >> 7) * TILE;
#pragma unroll
        for (int pn = 0; pn < CPR / 8; ++pn) {
            const int c = pn * 8 + c8;
            if (c * 8 < p.D) cp_async16(dst + tile_chunk(r & 127, c), src + c * 8, in);
        }
    }
    cp_async_commit();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    auto copies_done = [&](uint32_t bar) {
        cp_async_wait<0>();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(bar);
    };
    copies_done(q_full);
    constexpr uint32_t kO = 256;  // first column of O0

    if (warp >= 8 && warp < 8 + kLoadWarps) {
        // ---- copies ----
        const int lw = warp - 8;
        const bool paged = p.page_table != nullptr;
        bool alive = true;
        for (int i = early; i < n_loads; ++i) {
            const int s = i % NST;
            const int tile = first + (i >> 1);
            const bool is_v = i & 1;
            const bool pre = tile < tiles_p;
            const int t0 = pre ? tile * kTokTile : (tile - tiles_p) * kTokTile;
            const uint32_t dst = s_ring + s * TILE;
            if (pre ? tp.tma_p : tp.tma_c && (!is_v || t0 + kTokTile <= whole)) {
                if (lw == 0) {
                    if (i >= NST) alive = bar_wait_warp(empty(s), ((i / NST) - 1) & 1, gave_up);
                    if (!alive) continue;
                    if (pre) {
                        load_prefix(i);
                        continue;
                    }
                    const CUtensorMap* map = is_v ? &tp.vc : &tp.kc;
                    if (!paged) {
                        if (lane == 0) bar_expect(full(s), TILE);
                        __syncwarp();
                        if (lane < CPR / 8) tma_load(dst + lane * 16384, map, full(s), lane * 64, t0, h, b);
                    } else {
                        // One lane a box; a page that is not there lies outside the map: zeros.
                        const int box = tp.box_c, n_box = kTokTile / box;
                        const int bx = lane % n_box, t = t0 + bx * box;
                        int id = static_cast<int>(p.n_pages), in = 0;
                        bool ok = true;
                        if (t < vis) {
                            const int pg = static_cast<int>(fdiv(t, p.div_page));
                            in = t - pg * p.page;
                            id = p.page_table[b * p.pt_b + pg];
                            ok = id >= 0 && id < p.n_pages;
                            if (!ok) id = static_cast<int>(p.n_pages);
                        }
                        if (!is_v) {
                            const int local = (i >> 1) % kOks;
                            for (int e = lane / n_box; e < box; e += 32 / n_box) s_ok[local][bx * box + e] = ok;
                            if (!ok) {
                                s_any_bad = 1;
                                if (p.status) atomicOr(p.status, SC_STATUS_BAD_PAGE_ID);
                            }
                            __syncwarp();
                        }
                        if (lane == 0) bar_expect(full(s), TILE);
                        __syncwarp();
                        for (int pn = lane / n_box; pn < CPR / 8; pn += 32 / n_box)
                            tma_load(dst + pn * 16384 + bx * box * 128, map, full(s), pn * 64, in, h, id);
                    }
                }
                continue;
            }
            // The first copying warp waits for the stage and tells the other two.
            if (lw == 0) {
                if (alive && i >= NST) alive = bar_wait_warp(empty(s), ((i / NST) - 1) & 1, gave_up);
                if (lane == 0) s_copy = alive;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kLoadWarps) : "memory");
            alive = *reinterpret_cast<volatile int*>(&s_copy) != 0;
            if (!alive) break;
            const T* base;
            int64_t st_t, st_b = 0;
            if (pre) {
                base = static_cast<const T*>(is_v ? p.vp : p.kp) + h * (is_v ? p.vp_h : p.kp_h);
                st_t = is_v ? p.vp_t : p.kp_t;
            } else {
                base = static_cast<const T*>(is_v ? p.vc : p.kc) + h * (is_v ? p.vc_h : p.kc_h);
                st_t = is_v ? p.vc_t : p.kc_t;
                st_b = is_v ? p.vc_b : p.kc_b;
                if (!paged) base += b * st_b;
            }
            const int t1 = pre ? p.P : vis;
            for (int g = lw; g < 32; g += kLoadWarps) {
                const int r = g * 4 + sub, t = t0 + r;
                bool in = t < t1;
                int64_t off = 0;
                if (in) {
                    if (!pre && paged) {
                        const int pg = static_cast<int>(fdiv(t, p.div_page));
                        const int id = p.page_table[b * p.pt_b + pg];
                        in = id >= 0 && id < p.n_pages;
                        if (in) off = id * st_b + (t - pg * p.page) * st_t;
                        if (!is_v && c8 == 0) {
                            s_ok[(i >> 1) % kOks][r] = in;
                            if (!in) {
                                s_any_bad = 1;
                                if (p.status) atomicOr(p.status, SC_STATUS_BAD_PAGE_ID);
                            }
                        }
                    } else {
                        off = t * st_t;
                    }
                }
#pragma unroll
                for (int pn = 0; pn < CPR / 8; ++pn) {
                    const int c = pn * 8 + c8;
                    if (c * 8 < p.D) cp_async16(dst + tile_chunk(r, c), base + off + c * 8, in);
                }
            }
            cp_async_commit();
            cp_async_wait<0>();
            if (is_v && !pre && whole < vis && t0 + kTokTile > whole) {
                // each lane what it copied itself
                for (int g = lw; g < 32; g += kLoadWarps)
                    for (int pn = 0; pn < CPR / 8; ++pn) {
                        const int r = g * 4 + sub, c = pn * 8 + c8;
                        const uint32_t at = dst + tile_chunk(r, c);
                        take_out_odd<T>(at, t0 + r, s_odd + c * 8, DP, &s_any_odd);
                    }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kLoadWarps) : "memory");
            if (lw == 0 && lane == 0) bar_arrive(full(s));
        }
    } else if (warp == 11) {
        // ---- products ----
        // The warp stays converged, so addresses and descriptors are uniform; one lane issues.
        constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
        constexpr uint32_t id_common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24);
        constexpr uint32_t id_qk = id_common | ((128u >> 3) << 17);
        constexpr uint32_t id_pv = id_common | ((static_cast<uint32_t>(DP) >> 3) << 17) | (1u << 16);
        // Descriptors of the first step; a step's address is added to the low word.
        const uint64_t q_desc = desc(s_q, 16, 1024), k_desc = desc(s_ring, 16, 1024),
                       v_desc = desc(s_ring, 16384, 1024);
        const bool leader = elect_one();
        auto qk = [&](int q, int stage, int to) {
            const uint64_t qd = q_desc + static_cast<uint32_t>(q * (TILE / 16));
            const uint64_t kd = k_desc + static_cast<uint32_t>(stage * (TILE / 16));
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                const uint32_t off = ((kk >> 2) * 16384 + (kk & 3) * 32) / 16;
                mma_ss(tmem + to * 128, qd + off, kd + off, id_qk, kk > 0);
            }
        };
        auto pv = [&](int q, int stage, int from, bool add) {
            const uint64_t vd = v_desc + static_cast<uint32_t>(stage * (TILE / 16));
#pragma unroll
            for (int kk = 0; kk < kTokTile / 16; ++kk)
                mma_ts(tmem + kO + q * DP, tmem + from * 128 + kk * 8, vd + kk * (2048 / 16), id_pv,
                       add || kk > 0);
        };
        bool alive = bar_wait_all(q_full, 0, gave_up) && bar_wait_all(full(0), 0, gave_up);
        if (alive && leader) {
            for (int q = 0; q < n_q; ++q) {
                qk(q, 0, q);
                tc_commit(s_full(q));
            }
            tc_commit(empty(0));
        }
        __syncwarp();
        // One row tile: the next tile's scores go where those of a second row tile would be, while the
        // softmax works on this one's.
        for (int i = 0; n_q == 1 && i < n_tiles && alive; ++i) {
            const int buf = i & 1, v = 2 * i + 1, k = 2 * i + 2;  // places in the order of loads
            if (i + 1 < n_tiles) {
                alive = bar_wait_all(full(k % NST), k / NST & 1, gave_up);
                // the product before this one has read the weights that lie there
                if (alive && i > 0) alive = bar_wait_all(o_full(0), (i - 1) & 1, gave_up);
                if (!alive) break;
                tc_fence_after();
                if (leader) {
                    qk(0, k % NST, buf ^ 1);
                    tc_commit(s_full(buf ^ 1));
                    tc_commit(empty(k % NST));
                }
                __syncwarp();
            }
            alive = bar_wait_both(full(v % NST), v / NST & 1, p_full(buf), i >> 1 & 1, gave_up);
            if (!alive) break;
            tc_fence_after();
            if (leader) {
                pv(0, v % NST, buf, i > 0);
                tc_commit(o_full(0));
                tc_commit(empty(v % NST));
            }
            __syncwarp();
        }
        int stage = 1 % NST, phase = 0;  // of the next tile to be read
        for (int i = 0; n_q == 2 && i < n_tiles && alive; ++i) {
            const bool more = i + 1 < n_tiles;
            const int vs = stage, vp = phase;
            if (++stage == NST) stage = 0, phase ^= 1;
            const int ks = stage, kp = phase;
            if (more && ++stage == NST) stage = 0, phase ^= 1;
            for (int q = 0; q < n_q && alive; ++q) {
                alive = q == 0 ? bar_wait_both(full(vs), vp, p_full(0), i & 1, gave_up)
                               : bar_wait_all(p_full(q), i & 1, gave_up);
                if (!alive) break;
                tc_fence_after();
                if (leader) {
                    pv(q, vs, q, i > 0);
                    tc_commit(o_full(q));
                    if (q == n_q - 1) tc_commit(empty(vs));
                }
                __syncwarp();
                if (more) {
                    // The weights that this product reads lie where the next scores go.
                    alive = q == 0 ? bar_wait_both(full(ks), kp, o_full(0), i & 1, gave_up)
                                   : bar_wait_all(o_full(q), i & 1, gave_up);
                    if (!alive) break;
                    if (leader) {
                        qk(q, ks, q);
                        tc_commit(s_full(q));
                        if (q == n_q - 1) tc_commit(empty(ks));
                    }
                    __syncwarp();
                }
            }
        }
        __syncwarp();
    } else {
        // ---- softmax: one thread a row ----
        const int q = warp >> 2;
        const int r = q * kRowTile + (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t o_at = tmem + kO + q * DP + lanes;
        const bool any = q * kRowTile + (warp & 3) * 32 < n_rows;  // a row of this warp counts
        if (q < n_q) {
            const int row = min(r0 + r, rows - 1);
            const int j = static_cast<int>(fdiv(row, p.div_G));
            const int own_limit = min(vis, see + j + 1);
            float m = kNegInf, l = 0.f;  // m: the maximum in use
            bool alive = true;
            for (int i = 0; i < n_tiles; ++i) {
                const int buf = n_q == 1 ? i & 1 : q;
                const uint32_t s_at = tmem + buf * 128 + lanes;
                alive = bar_wait_warp(s_full(buf), (n_q == 1 ? i >> 1 : i) & 1, gave_up);
                if (!alive) break;
                tc_fence_after();
                if (any) {
                    const int tile = first + i;
                    const bool pre = tile < tiles_p;
                    const int t0 = pre ? tile * kTokTile : (tile - tiles_p) * kTokTile;
                    const int seen = (pre ? p.P : own_limit) - t0;  // columns below it count
                    const bool bad = !pre && *reinterpret_cast<volatile int*>(&s_any_bad) != 0;
                    const bool masked = __any_sync(0xffffffffu, seen < kTokTile) || bad;
                    // A score above the maximum in use by kRaise raises it, and O with it.
                    auto raised = [&](float top) {
                        const bool raise = top > m + kRaise<T> || (m == kNegInf && top > m);
                        if (!__any_sync(0xffffffffu, raise)) return;
                        const float f = raise ? exp2_fast(m - top) : 1.f;
                        if (raise) m = top;
                        l *= f;
                        if (i > 0) {  // the scores are there, so phase i - 2 is over: i - 1 is the open one
                            alive = bar_wait_warp(o_full(q), (i - 1) & 1, gave_up);
                            if (!alive) return;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < DP / 32; ++c) {
                                uint32_t o[32];
                                tmem_ld32(o_at + c * 32, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tmem_st32(o_at + c * 32, o);
                            }
                        }
                    };
                    bool quick = !masked && p.scale_log2 > 0.f;
                    if (quick) {
                        // All scores in registers, one pass.
                        uint32_t x[128];
#pragma unroll
                        for (int c = 0; c < 4; ++c) tmem_ld32(s_at + c * 32, x + c * 32);
                        tmem_wait_ld();
                        float t4[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
                        for (int e = 0; e < 128; e += 2)
                            t4[(e >> 1) & 3] = max3(t4[(e >> 1) & 3], __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
                        raised(fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * p.scale_log2);
                        if (!alive) break;
                        // The fused product below is off from the maximum by its rounding, which must not count.
                        quick = !__any_sync(0xffffffffu, fabsf(m) >= kFar);
                        if (quick) {
                            const float base = m == kNegInf ? 0.f : lifted<T>(m, kLiftTile<T>);
                            const float2 mul2 = make_float2(p.scale_log2, p.scale_log2), sub2 = make_float2(-base, -base);
                            float2 sum = make_float2(0.f, 0.f), sum2 = sum;
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t w[16];
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    float2 v = make_float2(__uint_as_float(x[c * 32 + 2 * e]),
                                                           __uint_as_float(x[c * 32 + 2 * e + 1]));
                                    v = __ffma2_rn(v, mul2, sub2);
                                    v.x = exp2_fast(v.x);
                                    v.y = exp2_fast(v.y);
                                    if (e & 1)
                                        sum2 = __fadd2_rn(sum2, v);
                                    else
                                        sum = __fadd2_rn(sum, v);
                                    w[e] = pack2<T>(v.x, v.y);
                                }
                                tmem_st16(s_at + c * 16, w);
                            }
                            l += (sum.x + sum.y) + (sum2.x + sum2.y);
                        }
                    }
                    if (!quick) {
                        // A tile's end, a mask, a scale that turns the order, far scores: the few of these take short
                        // loops, which leave the others' instructions together (eight prompts of up to
                        // 512 tokens behind 8,192: 459 us, this way 452).
                        const bool turned = p.scale_log2 <= 0.f;
                        const float mul = turned ? 1.f : p.scale_log2;
                        auto scores = [&](int c, uint32_t (&x)[16]) {  // 16 columns, what is hidden -inf
                            tmem_ld16(s_at + c, x);
                            tmem_wait_ld();
                            uint32_t on = 0;
#pragma unroll
                            for (int e = 0; e < 16; ++e) on |= (c + e < seen ? 1u : 0u) << e;
                            if (bad)
                                for (int e = 0; e < 16; ++e)
                                    if (!s_ok[i % kOks][c + e]) on &= ~(1u << e);
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float v = __uint_as_float(x[e]) * (turned ? p.scale_log2 : 1.f);
                                x[e] = __float_as_uint((on >> e) & 1 ? v : kNegInf);
                            }
                        };
                        float top = kNegInf;
#pragma unroll 1
                        for (int c = 0; c < kTokTile; c += 16) {
                            uint32_t x[16];
                            scores(c, x);
#pragma unroll
                            for (int e = 0; e < 16; ++e) top = fmaxf(top, __uint_as_float(x[e]));
                        }
                        raised(top * mul);
                        if (!alive) break;
                        const float base = m == kNegInf ? 0.f : lifted<T>(m, kLiftTile<T>);
#pragma unroll 1
                        for (int c = 0; c < kTokTile; c += 16) {
                            uint32_t x[16], w[8];
                            scores(c, x);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float v0 = exp2_fast(__fsub_rn(__fmul_rn(__uint_as_float(x[2 * e]), mul), base));
                                const float v1 = exp2_fast(__fsub_rn(__fmul_rn(__uint_as_float(x[2 * e + 1]), mul), base));
                                l += v0 + v1;
                                w[e] = pack2<T>(v0, v1);
                            }
                            tmem_st8(s_at + c / 2, w);  // over columns already read
                        }
                    }
                    tmem_wait_st();
                }
                const int o_phase = phase_before_weights(n_q, i, n_tiles);
                if (o_phase >= 0) {
                    alive = bar_wait_warp(o_full(q), o_phase & 1, gave_up);
                    if (!alive) break;
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(p_full(buf));
            }
            if (alive) {  // phase n_tiles - 2 is over (phase_before_weights): this is the open one
                alive = bar_wait_warp(o_full(q), (n_tiles - 1) & 1, gave_up);
            }
            if (alive && any) {
                tc_fence_after();
                const bool mine = r < n_rows;
                const int64_t at = static_cast<int64_t>(tok0 + j) * p.Hq + h * p.G + row - j * p.G;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                if (*reinterpret_cast<volatile int*>(&s_any_odd)) add_odd_tmem<DP>(o_at, s_odd, own_limit);
                if (mine) {
                    if (!direct)
                        p.part_ml[part_at(r)] = make_float2(m, l * kUnliftTile<T>);
                    else if (p.lse)
                        p.lse[at] = l == 0.f ? kNegInf : (m + log2f(l * kUnliftTile<T>)) * 0.6931471805599453f;
                }
                // 128 bytes of each of the warp's 32 rows at a time, turned in shared memory (where the
                // warp's queries were) so that a store covers whole lines: a lane's 16 bytes in 32 rows
                // took 5 us of a block's time.
                const uint32_t stage = s_q + q * TILE + (warp & 3) * (TILE / 4);
                const int per = direct ? 64 : 32;  // columns a pass
                // Each lane knows where its row goes; a store asks the lane whose row it is.  (Eight rows'
                // places worked out by every lane: 3 us more, for fetching the instructions of it.)
                char* to = nullptr;
                if (mine)
                    to = direct ? reinterpret_cast<char*>(static_cast<T*>(p.out) + (tok0 + j) * p.o_t +
                                                          (h * p.G + row - j * p.G) * p.o_h)
                                : reinterpret_cast<char*>(p.part_o + part_at(r) * p.D);
#pragma unroll 1
                for (int c = 0; c < DP; c += per) {
                    uint32_t o[64];
                    tmem_ld32(o_at + c, o);
                    if (direct) tmem_ld32(o_at + c + 32, o + 32);
                    tmem_wait_ld();
                    if constexpr (kUnliftTile<T> != 1.f) {
                        if (!direct)
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * kUnliftTile<T>);
                    }
                    if (direct) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            o[e] = pack2<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        st_shared_v4(stage + lane * 128 + ((k ^ (lane & 7)) << 4),
                                     make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
                    __syncwarp();
                    const int col = c + c8 * (per / 8);
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int rr = it * 4 + sub;
                        const uint4 v = ld_shared_v4(stage + rr * 128 + ((c8 ^ (rr & 7)) << 4));
                        char* dst = reinterpret_cast<char*>(
                            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), rr));
                        if (dst != nullptr && col < p.D) st_v4(dst + c * (direct ? 2 : 4) + c8 * 16, v);
                    }
                    __syncwarp();
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const bool lost = s_gave_up != 0;
    if (lost) {
        // Products may still be running: let them end (again with a limit) before the memory goes.
        __syncthreads();
        if (warp == 11 && elect_one()) {
            s_gave_up = 0;
            tc_commit(drained);
            bar_wait(drained, 0, gave_up);
            let_copies_land();
            if (p.status) atomicOr(p.status, SC_STATUS_WAIT_LIMIT);
        }
        __syncthreads();
    }
    if (warp == 11)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    wait_for_previous();  // nothing is read from it, but this kernel's end stands for its end, too
}

// Rows of the last round's units: their parts joined, a warp a row, eight parts' loads in flight.
// (A part at a time waited for memory: two sequences of 40 tokens x 32 heads behind 16,384 76 us, this
// way 53; one of 24 tokens behind 8,192 59 and 29.)
constexpr int kTailRows = 8;     // rows a block at a time
constexpr int kTailBlocks = 16;  // an SM: one turn for 74 units, the most that are split
constexpr int kTailLoads = 8;
template <typename T>
__global__ void __launch_bounds__(128) join_tail(const __grid_constant__ TileParams tp) {
    const AttnParams& p = tp.a;
    const Starts starts(p);
    const Round rd = rounds(tp, starts);
    constexpr int kGroups = 2 * kRowTile / kTailRows;  // of a unit's rows
    const int lane = threadIdx.x & 31;
    wait_for_previous();
    if (rd.parts == 1) return;
    for (int g = blockIdx.x; g < rd.rem * kGroups; g += gridDim.x) {
        const int unit = g / kGroups, first = (g - unit * kGroups) * kTailRows;
        int b, h, rt, tok0, n_tok;
        locate(p, starts, rd.full + unit, b, h, rt);
        sequence_tokens(p, starts, b, tok0, n_tok);
        for (int r = first + (threadIdx.x >> 5); r < first + kTailRows; r += 4) {
            const int row = rt * 2 * kRowTile + r;
            if (row >= n_tok * p.G) break;
            const int64_t at = static_cast<int64_t>(unit) * rd.parts * (2 * kRowTile) + r;
            // a lane a part
            const float2 ml = lane < rd.parts ? p.part_ml[at + lane * (2 * kRowTile)] : make_float2(kNegInf, 0.f);
            float m = ml.x;
#pragma unroll
            for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            const float w = ml.x == kNegInf ? 0.f : exp2_fast(ml.x - m);
            float sum = ml.x == kNegInf && ml.y == 0.f ? 0.f : w * ml.y;
#pragma unroll
            for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < rd.parts; i += kTailLoads) {
                float wi[kTailLoads];
                float4 v[kTailLoads];
#pragma unroll
                for (int k = 0; k < kTailLoads; ++k) {
                    wi[k] = __shfl_sync(0xffffffffu, w, i + k);  // 0 behind the last part
                    v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (!(wi[k] == 0.f) && lane * 4 < p.D)
                        v[k] = *reinterpret_cast<const float4*>(p.part_o + (at + (i + k) * (2 * kRowTile)) * p.D + lane * 4);
                }
#pragma unroll
                for (int k = 0; k < kTailLoads; ++k)
                    a.x += wi[k] * v[k].x, a.y += wi[k] * v[k].y, a.z += wi[k] * v[k].z, a.w += wi[k] * v[k].w;
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int j = static_cast<int>(fdiv(row, p.div_G)), head = h * p.G + row - j * p.G;
            if (lane * 4 < p.D)
                st_v2(static_cast<T*>(p.out) + (tok0 + j) * p.o_t + head * p.o_h + lane * 4,
                      make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv)));
            if (p.lse && lane == 0)
                p.lse[static_cast<int64_t>(tok0 + j) * p.Hq + head] =
                    sum == 0.f ? kNegInf : (m + log2f(sum)) * 0.6931471805599453f;
        }
    }
}

template <typename T, int DP>
cudaError_t launch_tiles_dp(const TileParams& p, unsigned units, bool chained, cudaStream_t s, bool load_only) {
    auto kernel = attend_tiles<T, DP>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_shared_memory(reinterpret_cast<const void*>(kernel), TileShape<DP>::kSmem, done);
    if (e != cudaSuccess || load_only) return e;
    e = launch_chained(kernel, dim3(units), kTThreads, TileShape<DP>::kSmem, s, chained, p);
    if (e != cudaSuccess || !p.per_seq || p.splits == 1) return e;
    return launch_chained(join_tail<T>, dim3(static_cast<unsigned>(p.sms * kTailBlocks)), 128, 0, s, true, p);
}

}  // namespace

cudaError_t launch_attention_tiles(const AttnParams& a, bool half, bool per_seq, int tiles, int splits,
                                   int sms, int64_t units, bool chained, cudaStream_t s) {
    TileParams p{};
    p.a = a;
    p.per_seq = per_seq, p.tiles = tiles, p.splits = splits, p.sms = sms;
    if (a.P) {
        const int64_t n[4] = {a.D, a.P, a.Hkv, 1};
        p.tma_p = make_map(&p.kp, half, a.kp, n, {a.kp_t, a.kp_h, 0}, kTokTile, 1) &&
                  make_map(&p.vp, half, a.vp, n, {a.vp_t, a.vp_h, 0}, kTokTile, 1);
    }
    if (per_seq && a.cap) {
        const bool paged = a.page_table != nullptr;
        int box = kTokTile;
        while (paged && a.page % box) box /= 2;
        p.box_c = box;
        const int64_t n[4] = {a.D, paged ? a.page : a.cap, a.Hkv, paged ? a.n_pages : a.B};
        // a box starts at a swizzle atom: 8 rows
        p.tma_c = box >= 8 && make_map(&p.kc, half, a.kc, n, {a.kc_t, a.kc_h, a.kc_b}, box, 1) &&
                  make_map(&p.vc, half, a.vc, n, {a.vc_t, a.vc_h, a.vc_b}, box, 1);
    }
    const unsigned n = static_cast<unsigned>(units);
    if (a.D <= 64)
        return half ? launch_tiles_dp<__half, 64>(p, n, chained, s, false)
                    : launch_tiles_dp<__nv_bfloat16, 64>(p, n, chained, s, false);
    return half ? launch_tiles_dp<__half, 128>(p, n, chained, s, false)
                : launch_tiles_dp<__nv_bfloat16, 128>(p, n, chained, s, false);
}

cudaError_t preload_attention_tile_kernels() {
    TileParams p{};
    cudaError_t e = launch_tiles_dp<__half, 64>(p, 0, false, nullptr, true);
    if (e == cudaSuccess) e = launch_tiles_dp<__nv_bfloat16, 64>(p, 0, false, nullptr, true);
    if (e == cudaSuccess) e = launch_tiles_dp<__half, 128>(p, 0, false, nullptr, true);
    if (e == cudaSuccess) e = launch_tiles_dp<__nv_bfloat16, 128>(p, 0, false, nullptr, true);
    cudaFuncAttributes attr;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, join_tail<__half>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, join_tail<__nv_bfloat16>);
    return e;
}

}  // namespace sc
