// sc_attention_stream.cu — the shared-prefix attention for few rows of a KV head (a decode step's
// own caches, a short prefix): what counts is that the keys and values stream at HBM's rate.
//
// Work is counted in steps: 64 tokens of one (sequence, KV head, row tile of 16 MT rows), prefix
// first, then the sequences' own caches.  A block stays and takes one run of consecutive steps, as
// long as every other block's, so ragged lengths leave no block idle; a part is what a block sees
// of one row tile, and join_parts adds the parts up.  Warp 4 copies: TMA boxes of 64 columns in the
// 128-byte swizzle, three steps ahead across row tiles and sequences, so no part waits for its
// first keys.  Warps 0-3 take 16 of a step's tokens each, with a softmax state of their own
// (16-bit-input matrix products, fp32 sums), joined when the part ends.
// (Blocks of one part, cp.async by every warp with its address arithmetic: 750 instructions for
// 16 tokens, 4.7 TB/s at best and 33 us for 64 ragged caches of up to 512 tokens, 73 MB; this way 18,
// of which a block's set-up and first data take 5 and a part's end 1.2.)
#include <math.h>

#include "sc_tensor.cuh"

namespace sc {
namespace {

constexpr int kSThreads = 160;
constexpr int kSWarps = 4;       // of them compute
constexpr int kStep = 64;        // tokens
constexpr int kMaxChunks = 256;  // of 32 sequences

template <int DP, int MT>
struct StreamShape {
    static constexpr int kRows = MT == 0 ? 8 : 16 * MT;  // MT = 0: eight rows, see below
    static constexpr int kStageBytes = 2 * kStep * DP * 2;
    // Two blocks an SM but where registers or shared memory allow one.
    static constexpr int kBlocks = DP == 256 || (DP == 128 && MT == 2) ? 1 : 2;
    static constexpr int kStages = DP == 64 ? (MT <= 1 ? 6 : 5) : DP == 128 ? (MT <= 1 ? 3 : 6) : 2;
    static constexpr int kQueries = MT == 0 || (MT == 1 && DP < 256) ? 1 : 2;  // row tiles of queries in shared memory
    static constexpr int kQ = kRows * DP * 2;
    static constexpr int kJoin = 16 * DP * 4;
    static constexpr int kSmem = kStages * kStageBytes + kQueries * kQ + kJoin + 1024;
};

struct StreamParams {
    AttnParams a;
    int32_t least;      // steps a block, at least
    int32_t box;        // rows of a box of the own caches
    int32_t with_prefix;
    CUtensorMap kp, vp, kc, vc;
};

template <int DP>
__device__ __forceinline__ uint32_t kv_chunk(int r, int c) {
    return static_cast<uint32_t>((c >> 3) * (kStep * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
template <int ROWS>
__device__ __forceinline__ uint32_t q_chunk(int r, int c) {
    return static_cast<uint32_t>((c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <typename T, int DP, int MT>
__global__ void __launch_bounds__(kSThreads, StreamShape<DP, MT>::kBlocks) attend_stream(const __grid_constant__ StreamParams sp) {
    using Shape = StreamShape<DP, MT>;
    constexpr int MR = Shape::kRows, NST = Shape::kStages, CPR = DP / 8;
    constexpr int STAGE = Shape::kStageBytes, QB = Shape::kQueries;
    constexpr bool kEight = MT == 0;
    constexpr bool kHeld = kEight || (MT == 1 && DP < 256);  // queries in registers
    constexpr int MTN = MT == 0 ? 1 : MT;
    const AttnParams& p = sp.a;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t s_bars[2 * NST + 2 * QB];
    __shared__ int s_chunk[kMaxChunks];
    __shared__ int s_bad[NST];  // a bit a box of a step: its page is not there
    __shared__ int s_gave_up;
    __shared__ float s_m[kSWarps][MR], s_l[kSWarps][MR];
    __shared__ int s_odd[2 * DP], s_any_odd;

    let_next_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t s_ring = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t s_q = s_ring + NST * STAGE;
    float* s_join = reinterpret_cast<float*>(smem_raw + (s_q + QB * Shape::kQ - smem_addr(smem_raw)));
    const uint32_t bars = smem_addr(s_bars);
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (NST + s); };
    auto q_full = [&](int s) { return bars + 8u * (2 * NST + s); };
    auto q_empty = [&](int s) { return bars + 8u * (2 * NST + QB + s); };
    volatile int* gave_up = &s_gave_up;

    const Starts starts(p);
    // A sequence's tokens of q and length; the kernel's first block reports what is wrong with them.
    auto sequence = [&](int b, int& tok0, int& n, int& len) {
        len = p.cap;
        bool fine = starts.of(b, tok0, n);
        if (p.cache_lens != nullptr) {
            len = p.cache_lens[b];
            if (len < 0 || len > p.cap) {
                fine = false;
                len = 0;
            }
        }
        return fine;
    };
    auto tiles_of = [&](int n) { return (n * p.G + MR - 1) / MR; };
    auto steps_of = [&](int len) { return max(1, (len + kStep - 1) / kStep); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            bar_init(full(s), 1);
            bar_init(empty(s), kSWarps);
        }
        for (int s = 0; s < QB; ++s) {
            bar_init(q_full(s), 32);
            bar_init(q_empty(s), kSWarps);
        }
        s_gave_up = 0;
        s_any_odd = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    for (int i = threadIdx.x; i < 2 * DP; i += kSThreads) s_odd[i] = kNoToken;
    // Steps of 32 sequences at a time (of one KV head).
    const int chunks = p.cap ? (p.B + 31) / 32 : 0;
    for (int c = warp; c < chunks; c += kSThreads / 32) {
        const int b = c * 32 + lane;
        int steps = 0;
        if (b < p.B) {
            int tok0, n, len;
            if (!sequence(b, tok0, n, len) && blockIdx.x == 0 && p.status) atomicOr(p.status, SC_STATUS_BAD_SEQ_LEN);
            steps = tiles_of(n) * steps_of(len);
        }
        steps = __reduce_add_sync(0xffffffffu, steps);
        if (lane == 0) s_chunk[c] = steps;
    }
    __syncthreads();

    // This block's run of steps.
    const int rows_p = starts.last * p.G;
    const int steps_p = sp.with_prefix ? (p.P + kStep - 1) / kStep : 0;
    const int64_t prefix_steps = static_cast<int64_t>(p.Hkv) * ((rows_p + MR - 1) / MR) * steps_p;
    int64_t cache_steps = 0;  // of one head, then of all
    for (int c0 = 0; c0 < chunks; c0 += 32) {
        const int v = c0 + lane < chunks ? s_chunk[c0 + lane] : 0;
        cache_steps += __reduce_add_sync(0xffffffffu, v);
    }
    cache_steps *= p.Hkv;
    const int64_t all = prefix_steps + cache_steps;
    int64_t run = (all + gridDim.x - 1) / gridDim.x;
    if (run < sp.least) run = sp.least;
    const int64_t g0 = blockIdx.x * run, g1 = min(all, g0 + run);
    if (g0 >= g1) {
        wait_for_previous();
        return;
    }

    // Where a step lies.  first: the step at which its row tile begins.
    struct Place {
        bool pre;
        int b, h, rt, tiles, steps, tok0, n_tok, len;
        int j;
        int64_t first;
    };
    auto enter = [&](Place& x) {  // a sequence
        sequence(x.b, x.tok0, x.n_tok, x.len);
        x.tiles = tiles_of(x.n_tok);
        x.steps = steps_of(x.len);
    };
    auto find = [&](int64_t g) {
        Place x;
        x.pre = g < prefix_steps;
        if (x.pre) {
            x.b = 0;
            x.tok0 = 0, x.n_tok = starts.last, x.len = p.P;
            x.tiles = (rows_p + MR - 1) / MR;
            x.steps = steps_p;
            const int tile = static_cast<int>(g / steps_p);
            x.j = static_cast<int>(g - static_cast<int64_t>(tile) * steps_p);
            x.h = tile / x.tiles;
            x.rt = tile - x.h * x.tiles;
            x.first = g - x.j;
            return x;
        }
        int64_t in = g - prefix_steps;  // steps before it among the caches
        int c = 0;
        while (in >= static_cast<int64_t>(s_chunk[c]) * p.Hkv) in -= static_cast<int64_t>(s_chunk[c++]) * p.Hkv;
        // the sequence within the chunk
        const int b = c * 32 + lane;
        int own = 0;
        if (b < p.B) {
            int tok0, n, len;
            sequence(b, tok0, n, len);
            own = tiles_of(n) * steps_of(len);
        }
        int upto = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, in < static_cast<int64_t>(upto) * p.Hkv);
        const int at = __ffs(past) - 1;
        const int before = __shfl_sync(0xffffffffu, upto - own, at);
        x.b = c * 32 + at;
        enter(x);
        const int rel = static_cast<int>(in - static_cast<int64_t>(before) * p.Hkv);
        const int tile = rel / x.steps;
        x.j = rel - tile * x.steps;
        x.h = tile / x.tiles;
        x.rt = tile - x.h * x.tiles;
        x.first = g - x.j;
        return x;
    };
    auto next_tile = [&](Place& x) {  // to the first step of the next row tile
        x.first += x.steps;
        x.j = 0;
        if (++x.rt < x.tiles) return;
        x.rt = 0;
        if (++x.h < p.Hkv) return;
        x.h = 0;
        if (x.pre) {
            x.pre = false;
            x.b = -1;
        }
        do {
            if (++x.b >= p.B) return;
            enter(x);
        } while (x.tiles == 0);
    };

    Place x = find(g0);
    int stage = 0, phase = 0, qs = 0, q_phase = 0;
    bool alive = true;

    if (warp == kSWarps) {
        // ---- copies ----
        const bool paged = p.page_table != nullptr;
        const int n_box = kStep / sp.box;
        for (int64_t g = g0; g < g1 && alive;) {
            const int n = static_cast<int>(min(static_cast<int64_t>(x.steps - x.j), g1 - g));
            // the row tile's queries
            alive = bar_wait_all(q_empty(qs), q_phase ^ 1, gave_up);
            if (!alive) break;
            const uint32_t qd = s_q + qs * Shape::kQ;
            const int r0 = x.rt * MR, rows = x.n_tok * p.G;
            for (int i = lane; i < MR * CPR; i += 32) {
                const int r = i / CPR, c = i - r * CPR;
                const bool in = r0 + r < rows && c * 8 < p.D;
                const int row = in ? r0 + r : r0;
                const int jq = static_cast<int>(fdiv(row, p.div_G));
                cp_async16(qd + q_chunk<MR>(r, c),
                           static_cast<const T*>(p.q) + (x.tok0 + jq) * p.q_t +
                               (x.h * p.G + row - jq * p.G) * p.q_h + (in ? c * 8 : 0),
                           in);
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(q_full(qs)) : "memory");
            if (++qs == QB) qs = 0, q_phase ^= 1;
            for (int i = 0; i < n && alive; ++i) {
                const int t0 = (x.j + i) * kStep;
                alive = bar_wait_all(empty(stage), phase ^ 1, gave_up);
                if (!alive) break;
                const uint32_t dst = s_ring + stage * STAGE;
                if (x.pre || !paged) {
                    if (lane == 0) {
                        s_bad[stage] = 0;
                        bar_expect(full(stage), STAGE);
                    }
                    __syncwarp();
                    // a lane a panel of the keys, then of the values
                    if (lane < 2 * (DP / 64)) {
                        const bool is_v = lane >= DP / 64;
                        const CUtensorMap* map = x.pre ? (is_v ? &sp.vp : &sp.kp) : (is_v ? &sp.vc : &sp.kc);
                        tma_load(dst + lane * (kStep * 128), map, full(stage), (lane % (DP / 64)) * 64, t0, x.h,
                                 x.pre ? 0 : x.b);
                    }
                } else {
                    // A lane a box; a page that is not there lies outside the map: zeros.
                    const int bx = lane % n_box, t = t0 + bx * sp.box;
                    int id = static_cast<int>(p.n_pages), in = 0;
                    bool ok = true;
                    if (t < x.len) {
                        const int pg = static_cast<int>(fdiv(t, p.div_page));
                        in = t - pg * p.page;
                        id = p.page_table[x.b * p.pt_b + pg];
                        ok = id >= 0 && id < p.n_pages;
                        if (!ok) id = static_cast<int>(p.n_pages);
                    }
                    const uint32_t bad = __ballot_sync(0xffffffffu, !ok && lane < n_box);
                    if (lane == 0) {
                        s_bad[stage] = static_cast<int>(bad);
                        if (bad && p.status) atomicOr(p.status, SC_STATUS_BAD_PAGE_ID);
                        bar_expect(full(stage), STAGE);
                    }
                    __syncwarp();
                    for (int k = lane / n_box; k < 2 * (DP / 64); k += 32 / n_box) {
                        const bool is_v = k >= DP / 64;
                        tma_load(dst + k * (kStep * 128) + bx * sp.box * 128, is_v ? &sp.vc : &sp.kc, full(stage),
                                 (k % (DP / 64)) * 64, in, x.h, id);
                    }
                }
                if (++stage == NST) stage = 0, phase ^= 1;
            }
            g += n;
            next_tile(x);
        }
        cp_async_wait<0>();
        if (!alive) let_copies_land();
        wait_for_previous();
        return;
    }

    // ---- attention ----
    // A warp that gives up a wait still goes through the joins: the others meet it there.
    for (int64_t g = g0; g < g1;) {
        const int n = static_cast<int>(min(static_cast<int64_t>(x.steps - x.j), g1 - g));
        const int r0 = x.rt * MR, rows = x.n_tok * p.G, n_rows = min(MR, rows - r0);
        if (alive) alive = bar_wait_warp(q_full(qs), q_phase, gave_up);
        const uint32_t q_at = s_q + qs * Shape::kQ, q_done = q_empty(qs);
        if (++qs == QB) qs = 0, q_phase ^= 1;

        // The queries of 16 rows stay in registers.
        // (Eight rows: two registers of a product's second operand for each 16 columns.)
        uint32_t qf[kEight ? DP / 32 : kHeld ? DP / 16 : 1][4];
        if constexpr (kEight) {
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk += 2)
                ldmatrix4(qf[kk / 2], q_at + q_chunk<MR>(lane & 7, kk * 2 + (lane >> 3)));
            __syncwarp();
            if (lane == 0) bar_arrive(q_done);
        } else if constexpr (kHeld) {
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk)
                ldmatrix4(qf[kk], q_at + q_chunk<MR>(lane & 15, kk * 2 + (lane >> 4)));
            __syncwarp();
            if (lane == 0) bar_arrive(q_done);
        }

        // 16 MT rows: o[mt][k] is 16 rows x 8 columns, row lane / 4 (+ 8).  Eight rows: the products are
        // turned over, o[0][k] is 16 columns x 8 rows, rows 2 (lane % 4) and + 1, and half of the
        // 16-row products' work and registers is gone.
        constexpr int OK = kEight ? DP / 16 : DP / 8;
        float o[MTN][OK][4];
        float m[MTN][2], l[MTN][2];
        int lim[MTN][2];  // tokens below it are seen
        const int see = x.len - x.n_tok;
#pragma unroll
        for (int mt = 0; mt < MTN; ++mt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[mt][e] = kNegInf;
                l[mt][e] = 0.f;
                const int r = kEight ? (lane & 3) * 2 + e : mt * 16 + e * 8 + (lane >> 2);
                const int jq = static_cast<int>(fdiv(min(r0 + r, rows - 1), p.div_G));
                lim[mt][e] = x.pre ? x.len : min(x.len, see + jq + 1);
            }
#pragma unroll
            for (int k = 0; k < OK; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][k][e] = 0.f;
        }
        // Steps that end below it are seen whole by every row.
        const int whole = x.pre ? x.len : min(x.len, see + static_cast<int>(fdiv(r0, p.div_G)) + 1);

        for (int i = 0; i < n; ++i) {
            if (alive) alive = bar_wait_warp(full(stage), phase, gave_up);
            const int tt = (x.j + i) * kStep + warp * 16;  // this warp's tokens
            const uint32_t kt = s_ring + stage * STAGE, vt = kt + kStep * DP * 2;
            const int bad = s_bad[stage];
            const bool mask = tt + 16 > whole || bad != 0;
            if (alive && tt < x.len) {
                if (tt + 16 > x.len) {  // what lies behind the length must not reach the product
                    for (int i2 = lane; i2 < 16 * CPR; i2 += 32) {
                        const int r = i2 / CPR, c = i2 - r * CPR;
                        if (tt + r >= x.len)
                            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(
                                             vt + kv_chunk<DP>(warp * 16 + r, c)),
                                         "r"(0)
                                         : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if (whole < x.len && tt + 16 > whole) {  // some rows do not see some of the tokens
                    for (int i2 = lane; i2 < 16 * CPR; i2 += 32) {
                        const int r = i2 / CPR, c = i2 - r * CPR;
                        take_out_odd<T>(vt + kv_chunk<DP>(warp * 16 + r, c), tt + r, s_odd + c * 8, DP, &s_any_odd);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if constexpr (kEight) {
                    // S^T = K Q^T in two chains
                    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                    for (int kk = 0; kk < DP / 16; ++kk) {
                        uint32_t a[4];
                        ldmatrix4(a, kt + kv_chunk<DP>(warp * 16 + (lane & 15), kk * 2 + (lane >> 4)));
                        mma16816<T>(s[kk & 1], a, qf[kk / 2][(kk & 1) * 2], qf[kk / 2][(kk & 1) * 2 + 1]);
                    }
                    float mx[2] = {m[0][0], m[0][1]};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = __fmul_rn(s[0][e] + s[1][e], p.scale_log2);  // as the maximum has it, not fused below
                        if (mask) {
                            const int t = tt + (lane >> 2) + (e >> 1) * 8;
                            bool seen = t < lim[0][e & 1];
                            if (bad) seen = seen && !((bad >> ((t & (kStep - 1)) / sp.box)) & 1);
                            if (!seen) v = kNegInf;
                        }
                        s[0][e] = v;
                        mx[e & 1] = fmaxf(mx[e & 1], v);
                    }
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], d));
                        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], d));
                    }
                    if (__any_sync(0xffffffffu, mx[0] > m[0][0] || mx[1] > m[0][1])) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float f = mx[e] == kNegInf ? 1.f : exp2_fast(m[0][e] - mx[e]);
                            m[0][e] = mx[e];
                            l[0][e] *= f;
#pragma unroll
                            for (int k = 0; k < OK; ++k) {
                                o[0][k][e] *= f;
                                o[0][k][e + 2] *= f;
                            }
                        }
                    }
                    const float base[2] = {mx[0] == kNegInf ? 0.f : lifted<T>(mx[0], kLift<T>),
                                           mx[1] == kNegInf ? 0.f : lifted<T>(mx[1], kLift<T>)};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[0][e] = exp2_fast(s[0][e] - base[e & 1]);
                        l[0][e & 1] += s[0][e];
                    }
                    // O^T += V^T P^T: the weights' two pieces, turned within the warp
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t w, r;
                        two_pieces<T>(s[0][2 * e], s[0][2 * e + 1], w, r);
                        hi[e] = turn8x8(w);
                        lo[e] = turn8x8(r);
                    }
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        uint32_t a[4];
                        ldmatrix4_t(a, vt + kv_chunk<DP>(warp * 16 + (lane & 7) + ((lane >> 4) << 3),
                                                         k * 2 + ((lane >> 3) & 1)));
                        mma16816<T>(o[0][k], a, hi[0], hi[1]);
                        mma16816<T>(o[0][k], a, lo[0], lo[1]);
                    }
                } else {
                    float s[MT][2][4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[mt][k][e] = 0.f;
#pragma unroll
                    for (int kk = 0; kk < DP / 16; ++kk) {
                        uint32_t kb[4];
                        ldmatrix4(kb, kt + kv_chunk<DP>(warp * 16 + (lane & 7) + ((lane >> 4) << 3),
                                                        kk * 2 + ((lane >> 3) & 1)));
                        if constexpr (kHeld) {
                            mma16816<T>(s[0][0], qf[kk], kb[0], kb[1]);
                            mma16816<T>(s[0][1], qf[kk], kb[2], kb[3]);
                        } else {
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                uint32_t a[4];
                                ldmatrix4(a, q_at + q_chunk<MR>(mt * 16 + (lane & 15), kk * 2 + (lane >> 4)));
                                mma16816<T>(s[mt][0], a, kb[0], kb[1]);
                                mma16816<T>(s[mt][1], a, kb[2], kb[3]);
                            }
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        float mx[2] = {m[mt][0], m[mt][1]};
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float v = __fmul_rn(s[mt][k][e], p.scale_log2);
                                if (mask) {
                                    const int t = tt + k * 8 + (lane & 3) * 2 + (e & 1);
                                    bool seen = t < lim[mt][e >> 1];
                                    if (bad) seen = seen && !((bad >> ((t & (kStep - 1)) / sp.box)) & 1);
                                    if (!seen) v = kNegInf;
                                }
                                s[mt][k][e] = v;
                                mx[e >> 1] = fmaxf(mx[e >> 1], v);
                            }
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
                            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
                        }
                        if (__any_sync(0xffffffffu, mx[0] > m[mt][0] || mx[1] > m[mt][1])) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float f = mx[e] == kNegInf ? 1.f : exp2_fast(m[mt][e] - mx[e]);
                                m[mt][e] = mx[e];
                                l[mt][e] *= f;
#pragma unroll
                                for (int k = 0; k < DP / 8; ++k) {
                                    o[mt][k][2 * e] *= f;
                                    o[mt][k][2 * e + 1] *= f;
                                }
                            }
                        }
                        const float base[2] = {mx[0] == kNegInf ? 0.f : lifted<T>(mx[0], kLift<T>),
                                               mx[1] == kNegInf ? 0.f : lifted<T>(mx[1], kLift<T>)};
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float w = exp2_fast(s[mt][k][e] - base[e >> 1]);
                                s[mt][k][e] = w;
                                l[mt][e >> 1] += w;
                            }
                    }
                    // o += P V, the weights in two pieces: the copies, not the products, bound this.
                    uint32_t hi[MT][4], lo[MT][4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            two_pieces<T>(s[mt][e >> 1][2 * (e & 1)], s[mt][e >> 1][2 * (e & 1) + 1], hi[mt][e],
                                          lo[mt][e]);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        uint32_t vb[4];
                        ldmatrix4_t(vb, vt + kv_chunk<DP>(warp * 16 + (lane & 7) + (((lane >> 3) & 1) << 3),
                                                          k * 2 + (lane >> 4)));
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma16816<T>(o[mt][2 * k], hi[mt], vb[0], vb[1]);
                            mma16816<T>(o[mt][2 * k + 1], hi[mt], vb[2], vb[3]);
                            mma16816<T>(o[mt][2 * k], lo[mt], vb[0], vb[1]);
                            mma16816<T>(o[mt][2 * k + 1], lo[mt], vb[2], vb[3]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) bar_arrive(empty(stage));
            if (++stage == NST) stage = 0, phase ^= 1;
        }
        if constexpr (!kHeld) {
            __syncwarp();
            if (lane == 0) bar_arrive(q_done);
        }

        // Join the four warps' states.
#pragma unroll
        for (int mt = 0; mt < MTN; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = kEight ? 4 : 1; d < (kEight ? 32 : 4); d <<= 1)
                    l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], d);
                const int r = kEight ? lane * 2 + e : mt * 16 + e * 8 + (lane >> 2);
                if (kEight ? lane < 4 : (lane & 3) == 0) {
                    s_m[warp][r] = m[mt][e];
                    s_l[warp][r] = l[mt][e];
                }
            }
        auto meet = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
        meet();
        const int64_t unit_part = g / run - x.first / run;  // which of its parts this is
        const int part = static_cast<int>(unit_part) + (x.pre ? 0 : p.n_pp);
        const int parts_end = x.pre ? p.n_pp : p.n_pp + p.n_cp;
        const int64_t all_rows = static_cast<int64_t>(p.N) * p.Hq;
        const bool last = x.j + n == x.steps;
        // Eight rows at a time, as a tree: warps 2 and 3 leave theirs, 0 and 1 add them, 1 leaves its sum,
        // 0 adds that and writes.  (Four warps in turn through one buffer: 6,300 clocks a part.)
        if constexpr (kEight) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = (lane & 3) * 2 + e;
                float top = s_m[0][r];
#pragma unroll
                for (int w = 1; w < kSWarps; ++w) top = fmaxf(top, s_m[w][r]);
                const float f = m[0][e] == kNegInf ? 0.f : exp2_fast(m[0][e] - top) * kOnePiece<T>;
#pragma unroll
                for (int k = 0; k < OK; ++k) {
                    o[0][k][e] *= f;
                    o[0][k][e + 2] *= f;
                }
            }
            float4* slot = reinterpret_cast<float4*>(s_join) + (warp & 1) * (2 * DP) + lane;
            auto leave = [&] {
#pragma unroll
                for (int k = 0; k < OK; ++k) slot[k * 32] = make_float4(o[0][k][0], o[0][k][1], o[0][k][2], o[0][k][3]);
            };
            auto take = [&](const float4* from) {
#pragma unroll
                for (int k = 0; k < OK; ++k) {
                    const float4 v = from[k * 32];
                    o[0][k][0] += v.x, o[0][k][1] += v.y, o[0][k][2] += v.z, o[0][k][3] += v.w;
                }
            };
            if (warp >= 2) leave();
            meet();
            if (warp < 2) take(slot);
            if (warp == 1) leave();
            meet();
            if (warp == 0) {
                take(slot + 2 * DP);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = (lane & 3) * 2 + e;
                    if (r >= n_rows) continue;
                    const int row = r0 + r, jq = static_cast<int>(fdiv(row, p.div_G));
                    float* dst = p.part_o + (part * all_rows + static_cast<int64_t>(x.tok0 + jq) * p.Hq + x.h * p.G +
                                             row - jq * p.G) * p.D + (lane >> 2);
#pragma unroll
                    for (int k = 0; k < OK; ++k) {
                        if (k * 16 < p.D) dst[k * 16] = o[0][k][e];
                        if (k * 16 + 8 < p.D) dst[k * 16 + 8] = o[0][k][e + 2];
                    }
                }
            }
            meet();
        } else {
#pragma unroll
        for (int half = 0; half < 2 * MT; ++half) {
            if (half * 8 >= n_rows) break;
            const int mt = half >> 1, e = half & 1, r = half * 8 + (lane >> 2);
            float top = s_m[0][r];
#pragma unroll
            for (int w = 1; w < kSWarps; ++w) top = fmaxf(top, s_m[w][r]);
            const float f = m[mt][e] == kNegInf ? 0.f : exp2_fast(m[mt][e] - top) * kOnePiece<T>;
#pragma unroll
            for (int k = 0; k < DP / 8; ++k) {
                o[mt][k][2 * e] *= f;
                o[mt][k][2 * e + 1] *= f;
            }
            // a lane's 8-byte values side by side with its neighbours': no bank conflicts
            float2* slot = reinterpret_cast<float2*>(s_join) + (warp & 1) * (4 * DP) + lane;
            auto leave = [&] {
#pragma unroll
                for (int k = 0; k < DP / 8; ++k) slot[k * 32] = make_float2(o[mt][k][2 * e], o[mt][k][2 * e + 1]);
            };
            auto take = [&](const float2* from) {
#pragma unroll
                for (int k = 0; k < DP / 8; ++k) {
                    const float2 v = from[k * 32];
                    o[mt][k][2 * e] += v.x;
                    o[mt][k][2 * e + 1] += v.y;
                }
            };
            if (warp >= 2) leave();
            meet();
            if (warp < 2) take(slot);
            if (warp == 1) leave();
            meet();
            if (warp == 0) {
                take(slot + 4 * DP);
                if (r < n_rows) {
                    const int row = r0 + r, jq = static_cast<int>(fdiv(row, p.div_G));
                    const int64_t at =
                        part * all_rows + static_cast<int64_t>(x.tok0 + jq) * p.Hq + x.h * p.G + row - jq * p.G;
                    float* dst = p.part_o + at * p.D + (lane & 3) * 2;
#pragma unroll
                    for (int k = 0; k < DP / 8; ++k)
                        if (k * 8 < p.D)
                            *reinterpret_cast<float2*>(dst + k * 8) = make_float2(o[mt][k][2 * e], o[mt][k][2 * e + 1]);
                }
            }
            meet();
        }
        }
        const bool odd = *reinterpret_cast<volatile int*>(&s_any_odd) != 0;
        for (int r = threadIdx.x; r < n_rows; r += 32 * kSWarps) {
            float top = s_m[0][r], sum = 0.f;
#pragma unroll
            for (int w = 1; w < kSWarps; ++w) top = fmaxf(top, s_m[w][r]);
#pragma unroll
            for (int w = 0; w < kSWarps; ++w)
                sum += s_l[w][r] * (s_m[w][r] == kNegInf ? 0.f : exp2_fast(s_m[w][r] - top));
            const int jq = static_cast<int>(fdiv(r0 + r, p.div_G));
            const int64_t row = static_cast<int64_t>(x.tok0 + jq) * p.Hq + x.h * p.G + r0 + r - jq * p.G;
            p.part_ml[part * all_rows + row] = make_float2(top, sum * kUnlift<T>);
            if (odd) add_odd(p.part_o + (part * all_rows + row) * p.D, p.D, s_odd, DP, min(x.len, see + jq + 1));
            if (last)  // parts that this row tile does not have
                for (int k = part + 1; k < parts_end; ++k) p.part_ml[k * all_rows + row] = make_float2(kNegInf, 0.f);
        }
        meet();
        if (odd) {
            for (int i = threadIdx.x; i < 2 * DP; i += 32 * kSWarps) s_odd[i] = kNoToken;
            if (threadIdx.x == 0) s_any_odd = 0;
            meet();
        }
        g += n;
        next_tile(x);
    }
    if (!alive && lane == 0 && p.status) atomicOr(p.status, SC_STATUS_WAIT_LIMIT);
    wait_for_previous();  // nothing is read from it, but this kernel's end stands for its end, too
}

template <typename T, int DP, int MT>
cudaError_t launch_stream(const StreamParams& p, unsigned blocks, bool chained, cudaStream_t s, bool load_only) {
    using Shape = StreamShape<DP, MT>;
    auto kernel = attend_stream<T, DP, MT>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_shared_memory(reinterpret_cast<const void*>(kernel), Shape::kSmem, done);
    if (e != cudaSuccess || load_only) return e;
    return launch_chained(kernel, dim3(blocks), kSThreads, Shape::kSmem, s, chained, p);
}

template <typename T>
cudaError_t launch_stream_dp(const StreamParams& p, int dp, int mt, unsigned blocks, bool chained, cudaStream_t s,
                             bool load_only) {
    if (mt == 0)
        return dp == 64    ? launch_stream<T, 64, 0>(p, blocks, chained, s, load_only)
               : dp == 128 ? launch_stream<T, 128, 0>(p, blocks, chained, s, load_only)
                           : launch_stream<T, 256, 0>(p, blocks, chained, s, load_only);
    if (dp == 64)
        return mt == 1 ? launch_stream<T, 64, 1>(p, blocks, chained, s, load_only) : launch_stream<T, 64, 2>(p, blocks, chained, s, load_only);
    if (dp == 128)
        return mt == 1 ? launch_stream<T, 128, 1>(p, blocks, chained, s, load_only)
                       : launch_stream<T, 128, 2>(p, blocks, chained, s, load_only);
    return launch_stream<T, 256, 1>(p, blocks, chained, s, load_only);
}

}  // namespace

bool make_stream_maps(const AttnParams& a, bool half, bool with_prefix, StreamMaps* m) {
    static_assert(sizeof(m->map[0]) == sizeof(CUtensorMap), "room for a map");
    auto* map = reinterpret_cast<CUtensorMap*>(m->map);
    if (with_prefix) {
        const int64_t n[4] = {a.D, a.P, a.Hkv, 1};
        if (!make_map(&map[0], half, a.kp, n, {a.kp_t, a.kp_h, 0}, kStep, 1) ||
            !make_map(&map[1], half, a.vp, n, {a.vp_t, a.vp_h, 0}, kStep, 1))
            return false;
    }
    m->box = kStep;
    if (a.cap) {
        const bool paged = a.page_table != nullptr;
        while (paged && a.page % m->box) m->box /= 2;
        const int64_t n[4] = {a.D, paged ? a.page : a.cap, a.Hkv, paged ? a.n_pages : a.B};
        // a box starts at a swizzle atom: 8 rows
        if (m->box < 8 || (a.B + 31) / 32 > kMaxChunks ||
            !make_map(&map[2], half, a.kc, n, {a.kc_t, a.kc_h, a.kc_b}, m->box, 1) ||
            !make_map(&map[3], half, a.vc, n, {a.vc_t, a.vc_h, a.vc_b}, m->box, 1))
            return false;
    }
    return true;
}

cudaError_t launch_attention_stream(const AttnParams& a, const StreamMaps& m, bool half, bool with_prefix, int dp,
                                    int mt, int least, int blocks, bool chained, cudaStream_t s) {
    StreamParams p{};
    p.a = a;
    p.least = least;
    p.box = m.box;
    p.with_prefix = with_prefix;
    const auto* map = reinterpret_cast<const CUtensorMap*>(m.map);
    p.kp = map[0], p.vp = map[1], p.kc = map[2], p.vc = map[3];
    return half ? launch_stream_dp<__half>(p, dp, mt, static_cast<unsigned>(blocks), chained, s, false)
                : launch_stream_dp<__nv_bfloat16>(p, dp, mt, static_cast<unsigned>(blocks), chained, s, false);
}

cudaError_t preload_attention_stream_kernels() {
    StreamParams p{};
    const int shapes[8][2] = {{64, 0}, {64, 1}, {64, 2}, {128, 0}, {128, 1}, {128, 2}, {256, 0}, {256, 1}};
    cudaError_t e = cudaSuccess;
    for (const auto& x : shapes) {
        if (e == cudaSuccess) e = launch_stream_dp<__half>(p, x[0], x[1], 0, false, nullptr, true);
        if (e == cudaSuccess) e = launch_stream_dp<__nv_bfloat16>(p, x[0], x[1], 0, false, nullptr, true);
    }
    return e;
}

}  // namespace sc
