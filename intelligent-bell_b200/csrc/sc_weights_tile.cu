// sc_weights_tile.cu — the attention weights per cached token on the 5th-generation tensor cores.
//
// S = K Q^T with 128 tokens as the rows of a product and NR query rows as its columns: a token is
// a lane of tensor memory, so one thread adds up a token's weights over all queries, in their
// order, without a shuffle.  A unit is 256 tokens (two tiles) of a (sequence, KV head); its keys
// are loaded once and its queries pass by in chunks of NR rows.  Blocks stay and take every
// grid-th unit, so the next unit's keys are on their way while this one's are weighed.
//
// NR = 16 (a decode step's few rows; HBM bounds it: the keys are read once) or 128 (many rows;
// the exponentials bound it: 16 a clock and SM against 4,096 multiplications).
//
// Roles: warps 0-3 and 4-7 the weights of tile 0 and 1, warp 8 the copies (TMA), warp 9 the
// products, warps 10 and 11 the scores of tokens that are not in use.  Each tile has two score
// buffers in tensor memory.
//
// Measured, 32 query heads on 8 KV heads of 128: one query of each of 16 sequences of up to 8,192
// tokens 29 us (22 at a copy's rate); 64 queries on 32,768 tokens 37, the exponentials alone 15.
#include <limits.h>
#include <math.h>

#include "sc_tensor.cuh"
#include "sc_weights.cuh"

namespace sc {
namespace {

constexpr int kThreadsW = 384;
constexpr int kTile = 128;           // tokens
constexpr int kPiece = 1024;         // scores copied by a warp at a time
constexpr int kMaxSequences = 1024;  // their lengths are held in shared memory

template <int DP, int NR>
struct WeighShape {
    static constexpr int kK = kTile * DP * 2;
    static constexpr int kQ = NR * DP * 2;
    static constexpr int kStagesQ = NR == 16 ? 4 : 2 * (128 / DP);
    static constexpr int kStagesK = (NR == 16 ? 6 : 4) * (128 / DP);
    static constexpr int kSmem = kK * kStagesK + kQ * kStagesQ + 1024;
    static constexpr int kColumns = 4 * NR;  // of tensor memory
};

struct WeighParams {
    WeightParams w;
    int32_t chunk_tokens;  // tokens of q a chunk
    FastDiv div_chunk;
    int32_t pieces;        // of a score row, for the copy
    CUtensorMap k, q;
};

template <typename T, int DP, int NR>
__global__ void __launch_bounds__(kThreadsW, 1) weigh_tiles(const __grid_constant__ WeighParams wp) {
    using Shape = WeighShape<DP, NR>;
    constexpr int KST = Shape::kStagesK, QST = Shape::kStagesQ;
    const WeightParams& p = wp.w;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t s_bars[2 * KST + 2 * QST + 9];
    __shared__ __align__(16) float s_neg_lse[QST][NR];
    __shared__ __align__(16) int s_lim[QST][NR];
    __shared__ int s_all_seen[QST];  // tokens below it are seen by the whole chunk
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    __shared__ int s_len[kMaxSequences];
    __shared__ int s_first[kMaxSequences + 1];  // units (of one head) before each sequence

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t s_k = (smem_addr(smem_raw) + 1023u) & ~1023u, s_q = s_k + KST * Shape::kK;
    const uint32_t bars = smem_addr(s_bars);
    auto k_full = [&](int s) { return bars + 8u * s; };
    auto k_empty = [&](int s) { return bars + 8u * (KST + s); };
    auto q_full = [&](int s) { return bars + 8u * (2 * KST + s); };
    auto q_empty = [&](int s) { return bars + 8u * (2 * KST + QST + s); };
    auto s_full = [&](int t, int b) { return bars + 8u * (2 * KST + 2 * QST + t * 2 + b); };
    auto s_empty = [&](int t, int b) { return bars + 8u * (2 * KST + 2 * QST + 4 + t * 2 + b); };
    const uint32_t drained = bars + 8u * (2 * KST + 2 * QST + 8);
    volatile int* gave_up = &s_gave_up;

    auto length_of = [&](int b) {
        if (p.cache_lens == nullptr) return p.S;
        const int len = p.cache_lens[b];
        return len < 0 || len > p.S ? 0 : len;
    };
    const Starts starts(p.cu_q, p.B, p.N, p.nq);
    auto tokens_of = [&](int b, int& tok0, int& n) { return starts.of(b, tok0, n); };

    if (warp == 8) {
        // Units of 256 tokens in use, per sequence.
        int sum = 0;
        for (int b0 = 0; b0 < p.B; b0 += 32) {
            const int b = b0 + lane;
            int n = 0;
            if (b < p.B) {
                const int len = length_of(b);
                s_len[b] = len;
                n = (len + 2 * kTile - 1) / (2 * kTile);
                if (blockIdx.x == 0 && p.cache_lens != nullptr &&
                    (p.cache_lens[b] < 0 || p.cache_lens[b] > p.S))
                    atomicOr(p.status, SC_STATUS_BAD_SEQ_LEN);
                if (int tok0, n_tok; blockIdx.x == 0 && !tokens_of(b, tok0, n_tok))
                    atomicOr(p.status, SC_STATUS_BAD_SEQ_LEN);
            }
            int v = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v += y;
            }
            if (b < p.B) s_first[b] = sum + v - n;
            sum += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) {
            s_first[p.B] = sum;
            for (int s = 0; s < KST; ++s) {
                bar_init(k_full(s), 1);
                bar_init(k_empty(s), 1);
            }
            for (int s = 0; s < QST; ++s) {
                bar_init(q_full(s), 1);
                bar_init(q_empty(s), 1 + 8);  // the products and the weights' warps
            }
            for (int i = 0; i < 4; ++i) {
                bar_init(s_full(i >> 1, i & 1), 1);
                bar_init(s_empty(i >> 1, i & 1), 4);
            }
            bar_init(drained, 1);
            s_gave_up = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    } else if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_addr(&s_tmem)),
                     "n"(Shape::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        // Query rows that no copy writes must be numbers.
        for (int i = threadIdx.x; i < QST * Shape::kQ / 16; i += 256)
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(s_q + 16u * i), "r"(0) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    // Units in the order of sequences, their heads, their tokens; a block takes a run of them.
    const int n_units = s_first[p.B] * p.Hkv;
    const int run = (n_units + gridDim.x - 1) / gridDim.x;
    const int u0 = min(n_units, static_cast<int>(blockIdx.x) * run), u1 = min(n_units, u0 + run);

    struct Unit {
        int b, h, t0, len, tok0, n_tok, n_t, c0, c1;
    };
    auto settle = [&](Unit& x) {  // what follows from sequence and first token
        x.n_t = x.t0 + kTile < x.len ? 2 : 1;
        x.c1 = static_cast<int>(fdiv(x.n_tok + wp.chunk_tokens - 1, wp.div_chunk));
        // queries before the first that sees token t0 see nothing of the unit
        const int j = p.causal ? x.t0 - (x.len - x.n_tok) : 0;
        x.c0 = j > 0 ? static_cast<int>(fdiv(j, wp.div_chunk)) : 0;
    };
    auto first_unit = [&] {
        Unit x{};
        if (u0 >= u1) return x;
        int lo = 0, hi = p.B;  // the last sequence whose first unit is not behind u0
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_first[mid] * p.Hkv <= u0)
                lo = mid;
            else
                hi = mid;
        }
        x.b = lo;
        x.len = s_len[lo];
        const int per_head = s_first[lo + 1] - s_first[lo], in = u0 - s_first[lo] * p.Hkv;
        x.h = in / per_head;
        x.t0 = (in - x.h * per_head) * 2 * kTile;
        tokens_of(lo, x.tok0, x.n_tok);
        settle(x);
        return x;
    };
    auto next_unit = [&](Unit& x) {
        x.t0 += 2 * kTile;
        if (x.t0 >= x.len) {
            x.t0 = 0;
            if (++x.h == p.Hkv) {
                x.h = 0;
                do ++x.b;
                while (x.b < p.B && s_len[x.b] == 0);
                if (x.b >= p.B) return;
                x.len = s_len[x.b];
                tokens_of(x.b, x.tok0, x.n_tok);
            }
        }
        settle(x);
    };

    if (warp == 8) {
        // ---- copies ----
        int kc = 0, qc = 0;
        bool alive = true;
        Unit x = first_unit();
        for (int u = u0; u < u1 && alive; ++u, next_unit(x)) {
            if (x.c0 >= x.c1) continue;
            // A chunk's lse, asked for before the copies are waited for.
            constexpr int PL = (NR + 31) / 32;
            float lse[PL];
            auto ask = [&](int c) {
#pragma unroll
                for (int i = 0; i < PL; ++i) {
                    const int r = i * 32 + lane;
                    const int j = static_cast<int>(fdiv(r, p.div_G)), g = r - j * p.G;
                    const int jj = c * wp.chunk_tokens + j;
                    lse[i] = r < NR && j < wp.chunk_tokens && jj < x.n_tok
                                 ? p.lse[(x.tok0 + jj) * p.lse_t + (x.h * p.G + g) * p.lse_h]
                                 : kNegInf;
                }
            };
            ask(x.c0);
            for (int t = 0; t < x.n_t && alive; ++t, ++kc) {
                const int s = kc % KST;
                alive = bar_wait_warp(k_empty(s), (kc / KST & 1) ^ 1, gave_up);
                if (!alive) break;
                if (lane == 0) bar_expect(k_full(s), Shape::kK);
                __syncwarp();
                if (lane < DP / 64)
                    tma_load(s_k + s * Shape::kK + lane * (kTile * 128), &wp.k, k_full(s), lane * 64,
                             x.t0 + t * kTile, x.h, x.b);
            }
            for (int c = x.c0; c < x.c1 && alive; ++c, ++qc) {
                const int s = qc % QST;
                alive = bar_wait_warp(q_empty(s), (qc / QST & 1) ^ 1, gave_up);
                if (!alive) break;
                const int j0 = c * wp.chunk_tokens;
                int least = INT_MAX;
#pragma unroll
                for (int i = 0; i < PL; ++i) {
                    const int r = i * 32 + lane;
                    if (r < NR) {
                        // no row, another sequence's, or one that saw nothing: it gives nothing
                        const bool is = lse[i] != kNegInf;
                        const int j = static_cast<int>(fdiv(r, p.div_G));
                        const int lim = !is ? INT_MIN : p.causal ? x.len - x.n_tok + j0 + j + 1 : INT_MAX;
                        s_neg_lse[s][r] = is ? -lse[i] * 1.4426950408889634f : 0.f;
                        s_lim[s][r] = lim;
                        least = min(least, lim);
                    }
                }
                if (c + 1 < x.c1) ask(c + 1);
                least = __reduce_min_sync(0xffffffffu, least);
                if (lane == 0) {
                    s_all_seen[s] = least;
                    bar_expect(q_full(s), wp.chunk_tokens * p.G * DP * 2);
                }
                __syncwarp();
                if (lane < DP / 64)
                    tma_load(s_q + s * Shape::kQ + lane * (NR * 128), &wp.q, q_full(s), lane * 64, 0,
                             x.tok0 + j0, x.h);
            }
        }
    } else if (warp == 9) {
        // ---- products ----
        // The warp stays converged, so addresses and descriptors are uniform; one lane issues.
        // (One lane in a branch of its own: 40.4 instead of 36.7 us for 16 x up to 8,192 tokens.)
        constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
        constexpr uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) |
                                   ((static_cast<uint32_t>(NR) >> 3) << 17) | ((128u >> 4) << 24);
        const uint64_t k_desc = desc(s_k, 16, 1024), q_desc = desc(s_q, 16, 1024);
        const bool leader = elect_one();
        int ks = 0, kp = 0, qs = 0, qp = 0, it0 = 0, it1 = 0;  // stages and phases; products a tile
        bool alive = true;
        Unit x = first_unit();
        for (int u = u0; u < u1 && alive; ++u, next_unit(x)) {
            if (x.c0 >= x.c1) continue;
            const int ks0 = ks;
            for (int c = x.c0; c < x.c1 && alive; ++c) {
                alive = bar_wait_all(q_full(qs), qp, gave_up);
                for (int t = 0; t < x.n_t && alive; ++t) {
                    const int it = t ? it1 : it0, buf = it & 1;
                    int s = ks0 + t;
                    s = s >= KST ? s - KST : s;
                    if (c == x.c0) {
                        alive = bar_wait_all(k_full(s), kp, gave_up);
                        if (++ks == KST) ks = 0, kp ^= 1;
                    }
                    if (alive) alive = bar_wait_all(s_empty(t, buf), (it >> 1 & 1) ^ 1, gave_up);
                    if (!alive) break;
                    tc_fence_after();
                    const uint64_t kd = k_desc + static_cast<uint32_t>(s * (Shape::kK / 16));
                    const uint64_t qd = q_desc + static_cast<uint32_t>(qs * (Shape::kQ / 16));
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < DP / 16; ++kk)
                            mma_ss(tmem + (t * 2 + buf) * NR,
                                   kd + ((kk >> 2) * (kTile * 128) + (kk & 3) * 32) / 16,
                                   qd + ((kk >> 2) * (NR * 128) + (kk & 3) * 32) / 16, idesc, kk > 0);
                        tc_commit(s_full(t, buf));
                        if (t == x.n_t - 1) tc_commit(q_empty(qs));
                        if (c == x.c1 - 1) tc_commit(k_empty(s));
                    }
                    __syncwarp();
                    if (t)
                        ++it1;
                    else
                        ++it0;
                }
                if (++qs == QST) qs = 0, qp ^= 1;
            }
        }
        __syncwarp();
    } else if (warp >= 10) {
        // ---- tokens not in use keep their score ----
        if (p.out != p.scores) {
            const int rows = p.B * p.Hkv;
            for (int piece = blockIdx.x * 2 + warp - 10; piece < rows * wp.pieces; piece += gridDim.x * 2) {
                const int row = piece / wp.pieces, b = row / p.Hkv, h = row - b * p.Hkv;
                const int i0 = (piece - row * wp.pieces) * kPiece, i1 = min(i0 + kPiece, p.S);
                const float* in = p.scores + b * p.s_b + h * p.s_h;
                float* out = p.out + b * p.o_b + h * p.o_h;
                const int lo = max(i0, s_len[b]);
                for (int i = lo + lane; i < i1; i += 32 * 16) {
                    float v[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (i + k * 32 < i1) v[k] = in[i + k * 32];
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (i + k * 32 < i1) out[i + k * 32] = v[k];
                }
            }
        }
    } else {
        // ---- weights: one thread a token ----
        const int t = warp >> 2;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const float2 mul2 = make_float2(p.scale_log2, p.scale_log2);
        int qc = 0, it = 0;
        bool alive = true;
        const int mine = t * kTile + (warp & 3) * 32 + lane;
        auto score_of = [&](const Unit& x) {
            return x.t0 + mine < x.len ? p.scores[x.b * p.s_b + x.h * p.s_h + x.t0 + mine] : 0.f;
        };
        Unit x = first_unit();
        float before = u0 < u1 ? score_of(x) : 0.f;
        for (int u = u0; u < u1 && alive; ++u) {
            const int tok = x.t0 + mine;
            const int last = x.t0 + t * kTile + (warp & 3) * 32 + 31;
            // the next unit's scores are on their way during this one
            Unit next = x;
            float next_before = 0.f;
            if (u + 1 < u1) {
                next_unit(next);
                next_before = score_of(next);
            }
            float2 acc = make_float2(0.f, 0.f), acc2 = acc;
            for (int c = x.c0; c < x.c1; ++c, ++qc) {
                const int qs = qc % QST;
                // the queries' lse and limits (with one tile the other warps keep in step, too)
                alive = bar_wait_warp(q_full(qs), qc / QST & 1, gave_up);
                if (!alive) break;
                if (t < x.n_t) {
                    const int buf = it & 1;
                    alive = bar_wait_warp(s_full(t, buf), it >> 1 & 1, gave_up);
                    if (!alive) break;
                    tc_fence_after();
                    const bool masked = last >= s_all_seen[qs];
                    const uint32_t at = tmem + (t * 2 + buf) * NR + lanes;
                    auto weigh = [&](const uint32_t* s, int c0, int n) {
#pragma unroll
                        for (int e = 0; e < n; e += 4) {
                            const float4 nl = *reinterpret_cast<const float4*>(&s_neg_lse[qs][c0 + e]);
                            float2 v0 = make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                            float2 v1 = make_float2(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
                            v0 = __ffma2_rn(v0, mul2, make_float2(nl.x, nl.y));
                            v1 = __ffma2_rn(v1, mul2, make_float2(nl.z, nl.w));
                            v0.x = exp2_fast(v0.x), v0.y = exp2_fast(v0.y);
                            v1.x = exp2_fast(v1.x), v1.y = exp2_fast(v1.y);
                            if (masked) {
                                const int4 lim = *reinterpret_cast<const int4*>(&s_lim[qs][c0 + e]);
                                v0.x = tok < lim.x ? v0.x : 0.f, v0.y = tok < lim.y ? v0.y : 0.f;
                                v1.x = tok < lim.z ? v1.x : 0.f, v1.y = tok < lim.w ? v1.y : 0.f;
                            }
                            acc = __fadd2_rn(acc, v0);
                            acc2 = __fadd2_rn(acc2, v1);
                        }
                    };
                    if constexpr (NR == 16) {
                        uint32_t s[16];
                        tmem_ld16(at, s);
                        tmem_wait_ld();
                        weigh(s, 0, 16);
                    } else {
#pragma unroll 1
                        for (int c0 = 0; c0 < NR; c0 += 64) {
                            uint32_t s[64];
                            tmem_ld32(at + c0, s);
                            tmem_ld32(at + c0 + 32, s + 32);
                            tmem_wait_ld();
                            weigh(s, c0, 64);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(s_empty(t, buf));
                    ++it;
                }
                __syncwarp();
                if (lane == 0) bar_arrive(q_empty(qs));
            }
            if (alive && tok < x.len)
                p.out[x.b * p.o_b + x.h * p.o_h + tok] = before + ((acc.x + acc.y) + (acc2.x + acc2.y));
            x = next;
            before = next_before;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const bool lost = s_gave_up != 0;
    if (lost) {
        // Products may still be running: let them end (again with a limit) before the memory goes.
        __syncthreads();
        if (warp == 9 && elect_one()) {
            s_gave_up = 0;
            tc_commit(drained);
            bar_wait(drained, 0, gave_up);
            let_copies_land();
            atomicOr(p.status, SC_STATUS_WAIT_LIMIT);
        }
        __syncthreads();
    }
    if (warp == 9)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "n"(Shape::kColumns)
                     : "memory");
}

template <typename T, int DP, int NR>
cudaError_t launch_weigh(const WeighParams& p, cudaStream_t s, bool load_only) {
    using Shape = WeighShape<DP, NR>;
    auto kernel = weigh_tiles<T, DP, NR>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_shared_memory(reinterpret_cast<const void*>(kernel), Shape::kSmem, done);
    if (e != cudaSuccess || load_only) return e;
    const int64_t most = size_product(p.w.B, p.w.Hkv, (p.w.S + 2 * kTile - 1) / (2 * kTile));
    const int sms = sm_count();
    kernel<<<static_cast<unsigned>(most < sms ? most : sms), kThreadsW, Shape::kSmem, s>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_weigh_type(const WeighParams& p, int nr, cudaStream_t s) {
    if (p.w.D <= 64) return nr == 16 ? launch_weigh<T, 64, 16>(p, s, false) : launch_weigh<T, 64, 128>(p, s, false);
    return nr == 16 ? launch_weigh<T, 128, 16>(p, s, false) : launch_weigh<T, 128, 128>(p, s, false);
}

template <typename T>
cudaError_t preload_weigh_type() {
    WeighParams p{};
    cudaError_t e = launch_weigh<T, 64, 16>(p, nullptr, true);
    if (e == cudaSuccess) e = launch_weigh<T, 64, 128>(p, nullptr, true);
    if (e == cudaSuccess) e = launch_weigh<T, 128, 16>(p, nullptr, true);
    if (e == cudaSuccess) e = launch_weigh<T, 128, 128>(p, nullptr, true);
    return e;
}

}  // namespace

cudaError_t launch_weight_tiles(const WeightParams& w, bool half, cudaStream_t s, bool* taken) {
    *taken = false;
    if (w.D > 128 || w.G > 128 || w.B > kMaxSequences || w.nq == 0 ||
        size_product(w.B, w.Hkv, (w.S + 2 * kTile - 1) / (2 * kTile)) >= (int64_t(1) << 31))
        return cudaSuccess;
    WeighParams p{};
    p.w = w;
    const int nr = size_product(w.nq, w.G) <= 16 ? 16 : 128;
    p.chunk_tokens = nr / w.G < w.nq ? nr / w.G : w.nq;
    p.pieces = (w.S + kPiece - 1) / kPiece;
    p.div_chunk = make_fastdiv(static_cast<uint32_t>(p.chunk_tokens));
    const int64_t nk[4] = {w.D, w.S, w.Hkv, w.B}, nqs[4] = {w.D, w.G, w.N, w.Hkv};
    if (!make_map(&p.k, half, w.k, nk, {w.k_t, w.k_h, w.k_b}, kTile, 1) ||
        !make_map(&p.q, half, w.q, nqs, {w.q_h, w.q_t, w.q_h * w.G}, w.G, p.chunk_tokens))
        return cudaSuccess;
    *taken = true;
    return half ? launch_weigh_type<__half>(p, nr, s) : launch_weigh_type<__nv_bfloat16>(p, nr, s);
}

cudaError_t preload_weight_tile_kernels() {
    cudaError_t e = preload_weigh_type<__half>();
    if (e == cudaSuccess) e = preload_weigh_type<__nv_bfloat16>();
    return e;
}

}  // namespace sc
