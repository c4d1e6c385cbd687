// sc_attention.cu — attention of a batch that shares a long prefix.
//
// Mathematics.  A query row (token j of sequence b, head h) sees the P prefix tokens and the
// tokens t <= len_b - n_b + j of its own cache:
//   o = sum_t e^{s_t - m} v_t / sum_t e^{s_t - m},  s_t = scale q . k_t,  m = max_t s_t.
// The sums are split over token ranges ("parts"); a part keeps (m, l, o) not normalised and
// parts join by rescaling to the common maximum.  All rows of all sequences read the prefix
// together: rows of one KV head are packed (token, head of the group) over the whole batch, so a
// prefix token is loaded once for 16 or 32 rows instead of once per sequence.
//
// Three kernels write parts, by the rows that one KV head has in common (plan_split):
//   attend_tiles (sc_attention_tile.cu)    64 rows and more over the prefix, 32 to 96 and more of
//                                          one sequence over prefix and own cache: tensor memory;
//   attend_stream (sc_attention_stream.cu) fewer: HBM bounds it;
//   attend_rows (here)                     what tensor maps cannot say: pages that no box of 8 rows
//                                          divides, expanded strides, more than 8,192 sequences.
// 64 sequences of one token, 32 query heads of 128 on 8 KV heads, 8,192 shared tokens, own caches
// of up to 512: 45 us, of which reading everything once takes 16.
//
// attend_rows: 16 * MT rows of one KV head against one part.  The four warps take turns at tiles
// of TK tokens; each keeps its own ring of tiles in shared memory (cp.async, 16 bytes a lane),
// its own softmax state and its own 16-bit-input, fp32-accumulating matrix products, and the
// four states are joined at the end of the part.  Rows of a tile are stored with their 16-byte
// chunks permuted by the row number, so ldmatrix reads without bank conflicts.
// join_parts adds the parts up.
#include <math.h>

#include "sc_attention.cuh"

namespace sc {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kSms = 148;          // blocks of attend_tiles at a time
constexpr int kPartTokens = 64;    // parts are multiples of this many tokens
constexpr int kMaxPagesPerPart = 2048;

// Byte offset of 16-byte chunk c of row r in a tile of DP-element rows.
template <int DP>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return static_cast<uint32_t>(r) * (DP * 2) + static_cast<uint32_t>((c ^ (r & 7)) * 16);
}

template <int DP, int MT, int TK, int NST>
struct RowsShape {
    static constexpr int kRing = kWarps * NST * 2 * TK * DP * 2;  // bytes of the warps' rings
    static constexpr int kSmem = 16 * MT * DP * 2 + kRing;
};

template <typename T, int DP, int MT, int TK, int NST>
__global__ void __launch_bounds__(kThreads) attend_rows(const __grid_constant__ AttnParams p) {
    constexpr int MR = 16 * MT;
    constexpr int CPR = DP / 8;            // chunks a row
    constexpr int RPI = 32 / CPR;          // rows a warp-wide copy covers
    constexpr int KT = TK * DP * 2;        // bytes of a K (or V) tile
    static_assert(kWarps * MR * DP * 4 <= RowsShape<DP, MT, TK, NST>::kRing, "join buffer");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int32_t s_page[kMaxPagesPerPart];
    __shared__ float s_m[kWarps][MR], s_l[kWarps][MR];
    __shared__ int s_bad;
    __shared__ int s_odd[2 * DP], s_any_odd;

    let_next_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* s_q = smem;
    unsigned char* s_ring = smem + MR * DP * 2;

    // Which rows and tokens: own caches first (they are the longer wait), then the prefix.
    int u = blockIdx.x;
    const int n_cache_units = p.n_cp * p.tiles_c * p.Hkv * p.B;
    const bool is_prefix = u >= n_cache_units;
    int b = 0, part;
    if (is_prefix) u -= n_cache_units;
    const int tiles = is_prefix ? p.tiles_p : p.tiles_c;
    const int rt = u % tiles;
    u /= tiles;
    const int h = u % p.Hkv;
    u /= p.Hkv;
    int tok0, n_tok;
    if (is_prefix) {
        part = u;
        tok0 = 0;
        n_tok = used_tokens(p);
    } else {
        part = u % p.n_cp;
        b = u / p.n_cp;
        sequence_tokens(p, Starts(p), b, tok0, n_tok);
    }
    const int rows = n_tok * p.G;
    const int r0 = rt * MR;
    if (r0 >= rows) return;
    const int n_rows = min(MR, rows - r0);

    int t0, t1, see = 0;  // see: own cache tokens the first token of the sequence sees, minus one
    if (is_prefix) {
        t0 = part * p.chunk_p;
        t1 = min(p.P, t0 + p.chunk_p);
    } else {
        const int len = cache_length(p, b);
        const int blocks = (len + kPartTokens - 1) / kPartTokens;
        const int chunk = (blocks + p.n_cp - 1) / p.n_cp * kPartTokens;
        see = len - n_tok;
        const int j_last = static_cast<int>(fdiv(r0 + n_rows - 1, p.div_G));
        t0 = part * chunk;
        t1 = min(min(len, t0 + chunk), see + j_last + 1);
        part += p.n_pp;
    }
    const int64_t part_row = static_cast<int64_t>(part) * p.N * p.Hq;
    if (t0 >= t1) {
        for (int r = threadIdx.x; r < n_rows; r += kThreads) {
            const int j = static_cast<int>(fdiv(r0 + r, p.div_G));
            const int g = r0 + r - j * p.G;
            p.part_ml[part_row + static_cast<int64_t>(tok0 + j) * p.Hq + h * p.G + g] =
                make_float2(kNegInf, 0.f);
        }
        return;
    }

    if (p.D < DP) {  // columns that no copy writes
        for (int i = threadIdx.x; i < RowsShape<DP, MT, TK, NST>::kRing / 16; i += kThreads)
            reinterpret_cast<uint4*>(s_ring)[i] = make_uint4(0, 0, 0, 0);
    }
    const bool paged = !is_prefix && p.page_table != nullptr;
    int first_page = 0;
    if (threadIdx.x == 0) s_bad = s_any_odd = 0;
    for (int i = threadIdx.x; i < 2 * DP; i += kThreads) s_odd[i] = kNoToken;
    if (paged || p.D < DP) __syncthreads();
    if (paged) {
        first_page = static_cast<int>(fdiv(t0, p.div_page));
        const int last = static_cast<int>(fdiv(t1 - 1, p.div_page));
        for (int i = threadIdx.x; i <= last - first_page; i += kThreads) {
            int id = p.page_table[b * p.pt_b + first_page + i];
            if (id < 0 || id >= p.n_pages) {
                id = -1;
                s_bad = 1;
                if (p.status) atomicOr(p.status, SC_STATUS_BAD_PAGE_ID);
            }
            s_page[i] = id;
        }
        __syncthreads();
    }
    const T* kbase;
    const T* vbase;
    int64_t k_t, v_t, k_b = 0, v_b = 0;
    if (is_prefix) {
        kbase = static_cast<const T*>(p.kp) + h * p.kp_h;
        vbase = static_cast<const T*>(p.vp) + h * p.vp_h;
        k_t = p.kp_t, v_t = p.vp_t;
    } else {
        kbase = static_cast<const T*>(p.kc) + h * p.kc_h;
        vbase = static_cast<const T*>(p.vc) + h * p.vc_h;
        k_t = p.kc_t, v_t = p.vc_t, k_b = p.kc_b, v_b = p.vc_b;
        if (!paged) kbase += b * k_b, vbase += b * v_b;
    }

    const uint32_t ring = smem_addr(s_ring) + warp * NST * 2 * KT;
    const int n_tiles = (t1 - t0 + TK - 1) / TK;
    const int my_tiles = n_tiles > warp ? (n_tiles - warp + kWarps - 1) / kWarps : 0;

    auto issue = [&](int i) {
        if (i < my_tiles) {
            const uint32_t dst = ring + (i % NST) * 2 * KT;
            const int tt = t0 + (warp + i * kWarps) * TK;
            const int c = lane % CPR;
            if (c * 8 < p.D) {
#pragma unroll
                for (int it = 0; it < TK / RPI; ++it) {
                    const int r = it * RPI + lane / CPR;
                    const int t = tt + r;
                    bool valid = t < t1;
                    int64_t ko = 0, vo = 0;
                    if (valid) {
                        if (paged) {
                            const int pg = static_cast<int>(fdiv(t, p.div_page));
                            const int id = s_page[pg - first_page];
                            const int in = t - pg * p.page;
                            valid = id >= 0;
                            if (valid) {
                                ko = id * k_b + in * k_t;
                                vo = id * v_b + in * v_t;
                            }
                        } else {
                            ko = t * k_t;
                            vo = t * v_t;
                        }
                    }
                    cp_async16(dst + chunk_at<DP>(r, c), kbase + ko + c * 8, valid);
                    cp_async16(dst + KT + chunk_at<DP>(r, c), vbase + vo + c * 8, valid);
                }
            }
        }
        cp_async_commit();
    };

    for (int i = 0; i < NST - 1; ++i) issue(i);
    // Queries of the tile, zeros behind the last row and behind D.
    for (int i = threadIdx.x; i < MR * CPR; i += kThreads) {
        const int r = i / CPR, c = i - r * CPR;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < n_rows && c * 8 < p.D) {
            const int j = static_cast<int>(fdiv(r0 + r, p.div_G));
            const int g = r0 + r - j * p.G;
            v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (tok0 + j) * p.q_t +
                                                (h * p.G + g) * p.q_h + c * 8);
        }
        *reinterpret_cast<uint4*>(s_q + chunk_at<DP>(r, c)) = v;
    }
    __syncthreads();
    const bool bad = s_bad != 0;

    float o[MT][DP / 8][4];
    float m[MT][2], l[MT][2];
    int lim[MT][2];  // tokens below it are seen
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            m[mt][e] = kNegInf;
            l[mt][e] = 0.f;
            const int r = mt * 16 + e * 8 + (lane >> 2);
            const int j = static_cast<int>(fdiv(min(r0 + r, rows - 1), p.div_G));
            lim[mt][e] = is_prefix ? t1 : min(t1, see + j + 1);
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
    }
    // Tiles that end below it are seen whole by every row.
    const int seen_whole = is_prefix ? t1 : min(t1, see + static_cast<int>(fdiv(r0, p.div_G)) + 1);
    const int whole = bad ? -1 : seen_whole;

    const uint32_t q_addr = smem_addr(s_q);
    for (int i = 0; i < my_tiles; ++i) {
        cp_async_wait<NST - 2>();
        __syncwarp();
        issue(i + NST - 1);
        const uint32_t kt = ring + (i % NST) * 2 * KT, vt = kt + KT;
        const int tt = t0 + (warp + i * kWarps) * TK;

        float s[MT][TK / 8][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < TK / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[mt][n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
            uint32_t a[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                ldmatrix4(a[mt], q_addr + chunk_at<DP>(mt * 16 + (lane & 15), kk * 2 + (lane >> 4)));
#pragma unroll
            for (int n = 0; n < TK / 16; ++n) {
                uint32_t kb[4];
                ldmatrix4(kb, kt + chunk_at<DP>(n * 16 + (lane & 7) + ((lane >> 4) << 3),
                                                kk * 2 + ((lane >> 3) & 1)));
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    mma16816<T>(s[mt][2 * n], a[mt], kb[0], kb[1]);
                    mma16816<T>(s[mt][2 * n + 1], a[mt], kb[2], kb[3]);
                }
            }
        }
        const bool mask = tt + TK > whole;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float mx[2] = {m[mt][0], m[mt][1]};
#pragma unroll
            for (int n = 0; n < TK / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = __fmul_rn(s[mt][n][e], p.scale_log2);  // as the maximum has it, not fused below
                    if (mask) {
                        const int t = tt + n * 8 + (lane & 3) * 2 + (e & 1);
                        bool seen = t < lim[mt][e >> 1];
                        if (bad && seen)
                            seen = s_page[static_cast<int>(fdiv(t, p.div_page)) - first_page] >= 0;
                        if (!seen) x = kNegInf;
                    }
                    s[mt][n][e] = x;
                    mx[e >> 1] = fmaxf(mx[e >> 1], x);
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
                    for (int n = 0; n < DP / 8; ++n) {
                        o[mt][n][2 * e] *= f;
                        o[mt][n][2 * e + 1] *= f;
                    }
                }
            }
            const float base[2] = {mx[0] == kNegInf ? 0.f : lifted<T>(mx[0], kLift<T>),
                                   mx[1] == kNegInf ? 0.f : lifted<T>(mx[1], kLift<T>)};
#pragma unroll
            for (int n = 0; n < TK / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float w = exp2_fast(s[mt][n][e] - base[e >> 1]);
                    s[mt][n][e] = w;
                    l[mt][e >> 1] += w;
                }
        }
        if (!is_prefix && tt + TK > seen_whole && seen_whole < t1) {  // some rows do not see some of the tokens
            for (int c = lane; c < TK * CPR; c += 32)
                take_out_odd<T>(vt + chunk_at<DP>(c / CPR, c % CPR), tt + c / CPR, s_odd + c % CPR * 8, DP, &s_any_odd);
            __syncwarp();
        }
        // o += P V, the weights in two pieces: this kernel waits for memory and the products are free.
#pragma unroll
        for (int kk = 0; kk < TK / 16; ++kk) {
            uint32_t hi[MT][4], lo[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    two_pieces<T>(s[mt][2 * kk + (e >> 1)][2 * (e & 1)], s[mt][2 * kk + (e >> 1)][2 * (e & 1) + 1],
                                  hi[mt][e], lo[mt][e]);
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                uint32_t vb[4];
                ldmatrix4_t(vb, vt + chunk_at<DP>(kk * 16 + (lane & 7) + (((lane >> 3) & 1) << 3),
                                                  n * 2 + (lane >> 4)));
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    mma16816<T>(o[mt][2 * n], hi[mt], vb[0], vb[1]);
                    mma16816<T>(o[mt][2 * n + 1], hi[mt], vb[2], vb[3]);
                    mma16816<T>(o[mt][2 * n], lo[mt], vb[0], vb[1]);
                    mma16816<T>(o[mt][2 * n + 1], lo[mt], vb[2], vb[3]);
                }
            }
        }
    }

    // Join the four warps' states.
    cp_async_wait<0>();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 1);
            l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 2);
            if ((lane & 3) == 0) {
                s_m[warp][mt * 16 + e * 8 + (lane >> 2)] = m[mt][e];
                s_l[warp][mt * 16 + e * 8 + (lane >> 2)] = l[mt][e];
            }
        }
    __syncthreads();
    float* s_o = reinterpret_cast<float*>(s_ring);  // [warp][MR][DP]
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = mt * 16 + e * 8 + (lane >> 2);
            float all = s_m[0][r];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) all = fmaxf(all, s_m[w][r]);
            const float f = m[mt][e] == kNegInf ? 0.f : exp2_fast(m[mt][e] - all) * kOnePiece<T>;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
                *reinterpret_cast<float2*>(s_o + (warp * MR + r) * DP + n * 8 + (lane & 3) * 2) =
                    make_float2(o[mt][n][2 * e] * f, o[mt][n][2 * e + 1] * f);
        }
    __syncthreads();
    const int cpr = p.D / 4;
    for (int i = threadIdx.x; i < n_rows * cpr; i += kThreads) {
        const int r = i / cpr, c = (i - r * cpr) * 4;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(s_o + (w * MR + r) * DP + c);
            acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
        }
        const int j = static_cast<int>(fdiv(r0 + r, p.div_G));
        const int64_t at = part_row + static_cast<int64_t>(tok0 + j) * p.Hq + h * p.G + r0 + r - j * p.G;
        *reinterpret_cast<float4*>(p.part_o + at * p.D + c) = acc;
    }
    const bool odd = s_any_odd != 0;
    if (odd) __syncthreads();
    for (int r = threadIdx.x; r < n_rows; r += kThreads) {
        float all = s_m[0][r], sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) all = fmaxf(all, s_m[w][r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
            sum += s_l[w][r] * (s_m[w][r] == kNegInf ? 0.f : exp2_fast(s_m[w][r] - all));
        const int j = static_cast<int>(fdiv(r0 + r, p.div_G));
        const int64_t at = part_row + static_cast<int64_t>(tok0 + j) * p.Hq + h * p.G + r0 + r - j * p.G;
        p.part_ml[at] = make_float2(all, sum * kUnlift<T>);
        if (odd) add_odd(p.part_o + at * p.D, p.D, s_odd, DP, min(t1, see + j + 1));
    }
}

// o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i over a row's parts.  W warps a row, each a run of
// the parts in order, joined in order through shared memory: one warp waits for memory part after
// part (672 rows of 37 parts: 11 us), four have four times as much on its way.
template <typename T, int W>
__global__ void __launch_bounds__(kThreads) join_parts(const __grid_constant__ AttnParams p) {
    __shared__ float4 s_o[kWarps][64];
    __shared__ float s_sum[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = W == 1 ? static_cast<int64_t>(blockIdx.x) * kWarps + warp : blockIdx.x;
    const int64_t all_rows = static_cast<int64_t>(p.N) * p.Hq;
    // Rows of no sequence stay as they are: nobody has written their own caches' parts.
    bool counts = row < all_rows;
    if (p.cu_q != nullptr) {
        counts = counts && in_sequence(p.cu_q, p.B, p.N, p.nq, static_cast<int>(static_cast<uint32_t>(row) / p.Hq));
        if (p.cap == 0 && blockIdx.x == 0 && warp == 0 && p.status)  // no kernel before looked at the sequences
            report_sequences(p.cu_q, p.B, p.N, p.nq, nullptr, 0, p.status);
    }
    wait_for_previous();
    if (!counts) return;
    const int parts = p.n_pp + p.n_cp;
    const int each = (parts + W - 1) / W, i0 = W == 1 ? 0 : warp * each, i1 = min(parts, i0 + each);
    float m = kNegInf;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, p.part_ml[i * all_rows + row].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    float sum = 0.f;
    const int d0 = lane * 4, d1 = 128 + lane * 4;
    const int64_t step = all_rows * p.D;
    for (int g = i0; g < i1; g += 32) {
        // A lane a part: its weight; 0 where the part saw nothing (its o was not written).
        float w = 0.f;
        if (g + lane < i1) {
            const float2 ml = p.part_ml[(g + lane) * all_rows + row];
            w = ml.x == kNegInf ? 0.f : exp2_fast(ml.x - m);
            sum += ml.x == kNegInf && ml.y == 0.f ? 0.f : w * ml.y;
        }
        const int n = min(32, i1 - g);
        const float* src = p.part_o + (g * all_rows + row) * p.D;
        for (int i = 0; i < n; i += 4, src += 4 * step) {
            float wi[4];
            float4 v[4], u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // four parts' loads in flight
                wi[j] = __shfl_sync(0xffffffffu, w, i + j);
                v[j] = u[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (!(wi[j] == 0.f)) {
                    if (d0 < p.D) v[j] = *reinterpret_cast<const float4*>(src + j * step + d0);
                    if (d1 < p.D) u[j] = *reinterpret_cast<const float4*>(src + j * step + d1);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a.x += wi[j] * v[j].x, a.y += wi[j] * v[j].y, a.z += wi[j] * v[j].z, a.w += wi[j] * v[j].w;
                b.x += wi[j] * u[j].x, b.y += wi[j] * u[j].y, b.z += wi[j] * u[j].z, b.w += wi[j] * u[j].w;
            }
        }
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if constexpr (W > 1) {
        s_o[warp][lane] = a;
        s_o[warp][32 + lane] = b;
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        if (warp) return;
        for (int w = 1; w < W; ++w) {
            const float4 v = s_o[w][lane], u = s_o[w][32 + lane];
            a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
            b.x += u.x, b.y += u.y, b.z += u.z, b.w += u.w;
            sum += s_sum[w];
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zero
    const int64_t tok = row / p.Hq, head = row - tok * p.Hq;
    T* dst = static_cast<T*>(p.out) + tok * p.o_t + head * p.o_h;
    if (d0 < p.D)
        st_v2(dst + d0, make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv)));
    if (d1 < p.D)
        st_v2(dst + d1, make_uint2(pack2<T>(b.x * inv, b.y * inv), pack2<T>(b.z * inv, b.w * inv)));
    if (p.lse && lane == 0)
        p.lse[row] = sum == 0.f ? kNegInf : (m + log2f(sum)) * 0.6931471805599453f;
}

// Four warps a row where rows are fewer than 8 an SM and parts enough to share: 672 rows of 37 parts
// 11 -> 5 us, but 2,048 rows of 12 parts 5 -> 8.
template <typename T>
cudaError_t launch_join(const AttnParams& p, int64_t rows, bool chained, cudaStream_t s) {
    if (rows >= kSms * 8 || p.n_pp + p.n_cp < 4)
        return launch_chained(join_parts<T, 1>, dim3(static_cast<unsigned>((rows + kWarps - 1) / kWarps)), kThreads,
                              0, s, chained, p);
    return launch_chained(join_parts<T, kWarps>, dim3(static_cast<unsigned>(rows)), kThreads, 0, s, chained, p);
}

struct Variant {
    int dp, mt;
};

Variant pick_variant(int32_t D, int64_t rows) {
    const int dp = D <= 64 ? 64 : D <= 128 ? 128 : 256;
    return {dp, dp < 256 && rows > 16 ? 2 : 1};
}

template <typename T, int DP, int MT>
cudaError_t launch_rows(const AttnParams& p, int64_t units, cudaStream_t s, bool load_only) {
    constexpr int TK = 16, NST = DP == 64 ? 4 : 3;
    constexpr int bytes = RowsShape<DP, MT, TK, NST>::kSmem;
    auto kernel = attend_rows<T, DP, MT, TK, NST>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_shared_memory(reinterpret_cast<const void*>(kernel), bytes, done);
    if (e != cudaSuccess || load_only) return e;
    kernel<<<static_cast<unsigned>(units), kThreads, bytes, s>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_rows_dp(const AttnParams& p, Variant v, int64_t units, cudaStream_t s) {
    if (v.dp == 64)
        return v.mt == 1 ? launch_rows<T, 64, 1>(p, units, s, false)
                         : launch_rows<T, 64, 2>(p, units, s, false);
    if (v.dp == 128)
        return v.mt == 1 ? launch_rows<T, 128, 1>(p, units, s, false)
                         : launch_rows<T, 128, 2>(p, units, s, false);
    return launch_rows<T, 256, 1>(p, units, s, false);
}

template <typename T>
cudaError_t preload_attention_type() {
    AttnParams p{};
    cudaError_t e = launch_rows<T, 64, 1>(p, 0, nullptr, true);
    if (e == cudaSuccess) e = launch_rows<T, 64, 2>(p, 0, nullptr, true);
    if (e == cudaSuccess) e = launch_rows<T, 128, 1>(p, 0, nullptr, true);
    if (e == cudaSuccess) e = launch_rows<T, 128, 2>(p, 0, nullptr, true);
    if (e == cudaSuccess) e = launch_rows<T, 256, 1>(p, 0, nullptr, true);
    cudaFuncAttributes attr;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, join_parts<T, 1>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, join_parts<T, kWarps>);
    return e;
}

// How the rows and tokens are split over kernels and parts.
struct Split {
    Variant v;
    bool tile_p;   // the prefix by attend_tiles
    bool fused;    // prefix and own caches together by attend_tiles, a sequence's rows at a time
    bool direct;   // no parts of the whole call: the output is written at once
    int32_t tiles_p, tiles_c;  // row tiles (of the kernel that takes them)
    int32_t chunk_p, n_pp, n_cp;
    int64_t units_tile, units_rows;
    int32_t sms_left;  // SMs beside attend_tiles; 0: all, one kernel after the other
    int32_t stream_mt;
    int32_t least, blocks, s_pp, s_cp;  // attend_stream: steps and blocks, and its parts
};

constexpr int kTileRows = 256, kTileTokens = 128, kStepTokens = 64;
constexpr int kMinTileRows = 64;   // fewer rows: the copies bound both kernels
constexpr int kTailParts = 16;     // of a unit in the last round, at most
constexpr int kMaxFused = 1024;    // sequences: every block counts their units
constexpr int kMinFusedRows = 32;  // of a sequence and KV head: fewer leave a row tile nearly empty
constexpr int kAllFusedRows = 96;  // from here on packing the batch's rows never won

// Parts of the token axis for attend_tiles: the number that ends soonest, in units of one step
// (256 rows x 128 tokens, about 2 us), counting whole rounds of 148 blocks, a block's start and
// end (4 steps), and the parts' way through memory.
int32_t plan_parts(double blocks, int64_t steps, double rows, int32_t D) {
    int32_t best = 1;
    double best_cost = 0.;
    for (int32_t n = 1; n <= 64 && (n == 1 || n * 2 <= steps); ++n) {
        const double waves = ceil(blocks * n / kSms);
        double cost = waves * (static_cast<double>((steps + n - 1) / n) + 4.0) * 2.0;
        if (n > 1) cost += 2.0 + n * rows * D * 8.0 / 5e6;
        if (n == 1 || cost < best_cost) best = n, best_cost = cost;
    }
    return best;
}

// Whether attend_tiles takes each sequence's rows over prefix and own cache (a row tile each, mostly
// empty with few rows), or the batch's rows packed over the prefix and attend_stream the caches (whose
// parts go through memory): whichever is estimated to end first, in us.  Measured (fused, packed), 8 KV
// heads of 128: 16 sequences of 64 rows behind 4,096 with 500 own 62, 103; 4 behind 8,192 with 300 39, 62;
// 32 of 40 rows behind 1,000 with 1,000 69, 165; 64 of 32 rows behind 4,096 with 500 212, 141; 16 of 40
// rows of 64 behind 4,099 with 700 64, 51.
bool fuse(int64_t rows_p, int64_t rows_c, int32_t B, int32_t Hkv, int32_t D, int32_t P, int32_t cap) {
    if (rows_c < kMinFusedRows || rows_c >= kAllFusedRows) return rows_c >= kAllFusedRows;
    const double units = static_cast<double>(B) * Hkv;
    const double steps_p = (P + kTileTokens - 1) / kTileTokens, steps_c = (cap + kTileTokens - 1) / kTileTokens;
    const double fused = 12.0 + units * (steps_p + steps_c) * 1.5 / kSms;
    const double prefix = static_cast<double>((rows_p + kTileRows - 1) / kTileRows) * Hkv * steps_p * 2.3;
    const double caches = units * ((rows_c + 31) / 32) * ((cap + kStepTokens - 1) / kStepTokens) * 2.6;
    const double packed = 24.0 + (prefix + caches / (D <= 64 ? 2 : 1)) / kSms;
    return fused < packed;
}

int32_t plan_split(int32_t N, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t nq, int32_t P,
                   int32_t cap, int32_t page, Split* out) {
    const int64_t G = Hq / Hkv;
    const int64_t rows_p = N * G, rows_c = cap ? nq * G : 0;
    Split s{};
    s.fused = D <= 128 && cap && B <= kMaxFused && fuse(rows_p, rows_c, B, Hkv, D, P, cap);
    s.tile_p = !s.fused && D <= 128 && P && rows_p >= kMinTileRows;
    const double rows = static_cast<double>(N) * Hq;
    if (s.fused) {
        s.tiles_c = static_cast<int32_t>((rows_c + kTileRows - 1) / kTileRows);
        const int64_t steps = (P + kTileTokens - 1) / kTileTokens + (cap + kTileTokens - 1) / kTileTokens;
        const int64_t most = rows_p / kTileRows + B, all = size_product(B, s.tiles_c);  // ragged: fewer than all
        s.n_pp = steps < 2 ? 1 : steps / 2 < kTailParts ? static_cast<int32_t>(steps / 2) : kTailParts;
        s.direct = true;
        s.units_tile = size_product(most < all ? most : all, Hkv) + (s.n_pp > 1 ? kSms - 1 : 0);
    } else {
        if (s.tile_p) {
            s.tiles_p = static_cast<int32_t>((rows_p + kTileRows - 1) / kTileRows);
            const double blocks = static_cast<double>(s.tiles_p) * Hkv;
            const int64_t tile_steps = (P + kTileTokens - 1) / kTileTokens;
            s.n_pp = plan_parts(blocks, tile_steps, rows, D);
            if (cap) {
                // attend_tiles on some SMs beside attend_stream on the others: both have some 10 us of
                // start and end, which this way pass at the same time.  A stream block takes 1 us a step.
                const double stream_steps = 0.75 * ((cap + kStepTokens - 1) / kStepTokens) * Hkv *
                                            static_cast<double>(B) * ((rows_c + 31) / 32);
                double best = -1.;
                for (int32_t n = 1; n <= 64 && n <= tile_steps && blocks * n <= kSms - 16; ++n) {
                    const int left = kSms - static_cast<int>(blocks * n);
                    const double tile_us = 10.0 + static_cast<double>((tile_steps + n - 1) / n) * (D <= 64 ? 1.5 : 2.0);
                    const double stream_us = 8.0 + stream_steps / (2.0 * left);
                    const double cost = (tile_us > stream_us ? tile_us : stream_us) + n * rows * D * 8.0 / 5e6;
                    if (best < 0. || cost < best) best = cost, s.n_pp = n, s.sms_left = left;
                }
            }
            s.direct = s.n_pp == 1 && !B;  // with sequences, join_parts knows whose rows count
            s.units_tile = size_product(s.n_pp, s.tiles_p, Hkv);
        }
        const int64_t rows_most = !P || s.tile_p ? rows_c : rows_p > rows_c ? rows_p : rows_c;
        s.v = pick_variant(D, rows_most);
        const int64_t mr = 16 * s.v.mt;
        s.stream_mt = rows_most <= 8 ? 0 : s.v.mt;
        const int32_t P_rows = s.tile_p ? 0 : P;
        if (!s.tile_p) s.tiles_p = static_cast<int32_t>((rows_p + mr - 1) / mr);
        s.tiles_c = static_cast<int32_t>((rows_c + mr - 1) / mr);

        // attend_stream: as many blocks as stay, each with a run of steps; a run is 1 to 4 steps
        // at least, and long enough that a row tile has 64 parts at most.
        const int64_t steps_p = (P_rows + kStepTokens - 1) / kStepTokens;
        const int64_t steps_c = cap ? (cap + kStepTokens - 1) / kStepTokens : 0;
        // (32 sequences' steps are counted in 32 bits)
        if (size_product(size_product(B < 32 ? B : 32, Hkv), s.tiles_c * 2 * s.v.mt, steps_c) >= (int64_t(1) << 31))
            return set_error(SC_ERR_INVALID_ARGUMENT, "too many rows and tokens in one call; split it");
        const double steps = static_cast<double>(steps_p) * Hkv * s.tiles_p +
                             static_cast<double>(steps_c) * Hkv * B * s.tiles_c;
        const int resident = (s.sms_left ? s.sms_left : kSms) * (s.v.dp == 256 || (s.v.dp == 128 && s.v.mt == 2) ? 1 : 2);
        s.blocks = steps < 1 ? 0 : static_cast<int32_t>(steps < resident ? steps : resident);
        const int64_t longest_steps = steps_p > steps_c ? steps_p : steps_c;
        const double each = steps / resident;
        int64_t least = each < 1 ? 1 : each > 4 ? 4 : static_cast<int64_t>(each);
        if (least < (longest_steps + 62) / 63) least = (longest_steps + 62) / 63;
        s.least = static_cast<int32_t>(least);
        auto parts = [&](int64_t n) { return n ? static_cast<int32_t>((n + least - 1) / least + (n > 1)) : 0; };
        s.s_pp = s.tile_p ? s.n_pp : parts(steps_p);
        s.s_cp = parts(steps_c);

        // attend_rows: two blocks fit an SM; two rounds of equal parts.
        const double work = static_cast<double>(P_rows) * Hkv * s.tiles_p +
                            static_cast<double>(cap) * Hkv * B * s.tiles_c;
        double chunk = ceil(work / (kSms * 2 * 2) / kPartTokens) * kPartTokens;
        const double longest = P_rows > cap ? P_rows : cap;
        const double most_parts = 64;
        if (chunk < longest / most_parts) chunk = ceil(longest / most_parts / kPartTokens) * kPartTokens;
        if (chunk < kPartTokens) chunk = kPartTokens;
        s.chunk_p = static_cast<int32_t>(chunk > 0x40000000 ? 0x40000000 : chunk);
        if (!s.tile_p) s.n_pp = P ? (P - 1) / s.chunk_p + 1 : 0;
        s.n_cp = cap ? (cap - 1) / s.chunk_p + 1 : 0;
        // A part's page ids are held in shared memory.
        if (cap && page < cap) {
            const int64_t room = static_cast<int64_t>(kMaxPagesPerPart - 1) * page / kPartTokens * kPartTokens;
            const int64_t blocks = (static_cast<int64_t>(cap) + kPartTokens - 1) / kPartTokens;
            const int64_t need = (blocks * kPartTokens + room - 1) / room;
            if (need > s.n_cp) s.n_cp = static_cast<int32_t>(need);
        }
        s.units_rows = (s.tile_p ? 0 : size_product(s.n_pp, s.tiles_p, Hkv)) +
                       size_product(size_product(s.n_cp, s.tiles_c, Hkv), B);
    }
    if (s.units_rows >= (int64_t(1) << 31) || s.units_tile >= (int64_t(1) << 31))
        return set_error(SC_ERR_INVALID_ARGUMENT, "too many blocks in one call; split it");
    *out = s;
    return SC_OK;
}

int32_t check_sizes(int64_t N, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int64_t nq, int64_t P,
                    int64_t cap) {
    if (N < 0 || B < 0 || Hq < 0 || Hkv < 0 || nq < 0 || P < 0 || cap < 0)
        return set_error(SC_ERR_INVALID_ARGUMENT, "negative size");
    if (Hkv == 0 ? Hq != 0 : Hq % Hkv != 0)
        return set_error(SC_ERR_INVALID_ARGUMENT, "%d query heads are no multiple of %d KV heads", Hq, Hkv);
    if (D <= 0 || D % 8 != 0 || D > 256)
        return set_error(SC_ERR_UNSUPPORTED, "head_dim %d: a multiple of 8, at most 256", D);
    if (size_product(N, Hq) >= (int64_t(1) << 31) || P >= (int64_t(1) << 30) || cap >= (int64_t(1) << 30) ||
        B >= (1 << 24) || size_product(nq, Hq) >= (int64_t(1) << 31))
        return set_error(SC_ERR_INVALID_ARGUMENT, "too many rows or tokens in one call; split it");
    return SC_OK;
}

int64_t workspace_floats(const Split& s, int64_t N, int32_t Hq, int32_t D) {
    const int64_t rows = static_cast<int64_t>(s.n_pp) + s.n_cp, stream = static_cast<int64_t>(s.s_pp) + s.s_cp;
    if (s.fused) return s.n_pp > 1 ? static_cast<int64_t>(kSms) * kTileRows * (D + 2) : 0;
    return s.direct ? 0 : size_product(rows > stream ? rows : stream, N * Hq, D + 2);
}

}  // namespace

cudaError_t preload_attention_kernels() {
    cudaError_t e = preload_attention_type<__half>();
    if (e == cudaSuccess) e = preload_attention_type<__nv_bfloat16>();
    if (e == cudaSuccess) e = preload_attention_tile_kernels();
    if (e == cudaSuccess) e = preload_attention_stream_kernels();
    return e;
}

}  // namespace sc

using namespace sc;

extern "C" int32_t sc_shared_prefix_attention_workspace(int64_t n_tokens, int32_t batch,
                                                        int32_t q_heads, int32_t kv_heads,
                                                        int32_t head_dim, int64_t max_q_len,
                                                        int64_t prefix_len, int64_t cache_len,
                                                        int32_t page_size, int64_t* bytes) {
    if (!bytes) return set_error(SC_ERR_INVALID_ARGUMENT, "null pointer argument");
    *bytes = 0;
    const int64_t cap = batch ? cache_len : 0;
    int32_t rc = check_sizes(n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, prefix_len, cap);
    if (rc != SC_OK) return rc;
    if (cap && page_size <= 0) return set_error(SC_ERR_INVALID_ARGUMENT, "page_size %d", page_size);
    if (n_tokens == 0 || q_heads == 0) return ok();
    Split s;
    rc = plan_split(static_cast<int32_t>(n_tokens), batch, q_heads, kv_heads, head_dim,
                    static_cast<int32_t>(max_q_len), static_cast<int32_t>(prefix_len),
                    static_cast<int32_t>(cap), page_size, &s);
    if (rc != SC_OK) return rc;
    *bytes = size_product(workspace_floats(s, n_tokens, q_heads, head_dim), 4);
    return ok();
}

extern "C" int32_t sc_shared_prefix_attention(
    int64_t n_tokens, int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
    int32_t dtype, const void* q, const int64_t* q_strides, int64_t prefix_len, const void* k_prefix,
    const int64_t* kp_strides, const void* v_prefix, const int64_t* vp_strides, int64_t cache_len,
    const void* k_cache, const int64_t* kc_strides, const void* v_cache, const int64_t* vc_strides,
    const int32_t* cache_lens, const int32_t* page_table, int64_t page_table_stride, int32_t page_size,
    int64_t n_pages, const int32_t* cu_q_lens, int64_t max_q_len, double scale, void* out,
    const int64_t* out_strides, float* lse, void* workspace, int64_t workspace_bytes, int32_t* status,
    void* stream) {
    const int64_t cap = batch ? cache_len : 0;
    int32_t rc = check_sizes(n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, prefix_len, cap);
    if (rc != SC_OK) return rc;
    if (dtype != SC_DTYPE_F16 && dtype != SC_DTYPE_BF16)
        return set_error(SC_ERR_INVALID_DTYPE, "dtype code %d: float16 or bfloat16", dtype);
    if (!isfinite(static_cast<float>(scale * 1.4426950408889634)))
        return set_error(SC_ERR_INVALID_ARGUMENT, "scale must be finite in float32, got %g", scale);
    if (n_tokens == 0 || q_heads == 0) return ok();
    if (!cu_q_lens && batch && n_tokens != max_q_len * batch)
        return set_error(SC_ERR_INVALID_ARGUMENT, "%lld tokens are not %d sequences of %lld",
                         (long long)n_tokens, batch, (long long)max_q_len);
    if (cap && page_size <= 0) return set_error(SC_ERR_INVALID_ARGUMENT, "page_size %d", page_size);
    if (!q || !q_strides || !out || !out_strides || (prefix_len && (!k_prefix || !v_prefix ||
        !kp_strides || !vp_strides)) || (cap && (!k_cache || !v_cache || !kc_strides || !vc_strides)) ||
        (cu_q_lens && batch == 0))
        return set_error(SC_ERR_INVALID_ARGUMENT, "null pointer argument");
    auto aligned = [&](const void* ptr, const int64_t* st, int n) {
        bool ok = reinterpret_cast<uintptr_t>(ptr) % 16 == 0;
        for (int i = 0; i < n; ++i) ok = ok && st[i] % 8 == 0;
        return ok;
    };
    if (!aligned(q, q_strides, 2) || !aligned(out, out_strides, 2) ||
        (prefix_len && (!aligned(k_prefix, kp_strides, 2) || !aligned(v_prefix, vp_strides, 2))) ||
        (cap && (!aligned(k_cache, kc_strides, 3) || !aligned(v_cache, vc_strides, 3))))
        return set_error(SC_ERR_INVALID_ARGUMENT, "rows must start at multiples of 16 bytes");

    Split s;
    rc = plan_split(static_cast<int32_t>(n_tokens), batch, q_heads, kv_heads, head_dim,
                    static_cast<int32_t>(max_q_len), static_cast<int32_t>(prefix_len),
                    static_cast<int32_t>(cap), page_size, &s);
    if (rc != SC_OK) return rc;
    const int64_t need = size_product(workspace_floats(s, n_tokens, q_heads, head_dim), 4);
    if (workspace_bytes < need || (need && !workspace) || reinterpret_cast<uintptr_t>(workspace) % 16)
        return set_error(SC_ERR_INVALID_ARGUMENT, "workspace of %lld bytes (16-byte aligned) needed, got %lld",
                         (long long)need, (long long)workspace_bytes);

    AttnParams p{};
    p.q = q, p.q_t = q_strides[0], p.q_h = q_strides[1];
    p.kp = k_prefix, p.vp = v_prefix;
    if (prefix_len)
        p.kp_t = kp_strides[0], p.kp_h = kp_strides[1], p.vp_t = vp_strides[0], p.vp_h = vp_strides[1];
    p.kc = k_cache, p.vc = v_cache;
    if (cap) {
        p.kc_b = kc_strides[0], p.kc_t = kc_strides[1], p.kc_h = kc_strides[2];
        p.vc_b = vc_strides[0], p.vc_t = vc_strides[1], p.vc_h = vc_strides[2];
    }
    p.page_table = cap ? page_table : nullptr, p.pt_b = page_table_stride, p.n_pages = n_pages;
    p.cache_lens = cache_lens, p.cu_q = cu_q_lens;
    p.N = static_cast<int32_t>(n_tokens), p.B = batch, p.Hq = q_heads, p.Hkv = kv_heads;
    p.G = q_heads / kv_heads, p.D = head_dim, p.nq = static_cast<int32_t>(max_q_len);
    p.P = static_cast<int32_t>(prefix_len), p.cap = static_cast<int32_t>(cap);
    p.page = page_size > 0 ? page_size : 1;
    p.div_G = make_fastdiv(static_cast<uint32_t>(p.G));
    p.div_page = make_fastdiv(static_cast<uint32_t>(p.page));
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    p.chunk_p = s.chunk_p, p.tiles_p = s.tiles_p, p.tiles_c = s.tiles_c;
    const int64_t rows = n_tokens * q_heads;
    p.part_o = static_cast<float*>(workspace);
    auto set_parts = [&](int32_t n_pp, int32_t n_cp) {
        p.n_pp = n_pp, p.n_cp = n_cp;
        const int64_t part_rows = s.fused ? static_cast<int64_t>(kSms) * kTileRows : (n_pp + n_cp) * rows;
        p.part_ml = reinterpret_cast<float2*>(p.part_o + part_rows * head_dim);
    };
    const bool half = dtype == SC_DTYPE_F16, with_prefix = !s.tile_p && prefix_len > 0;
    // Few rows: the streaming kernel, or attend_rows where tensor maps cannot say the layout (pages
    // that no box of 8 rows divides, expanded strides).
    StreamMaps maps{};
    const bool streams = s.units_rows && s.blocks > 0 && make_stream_maps(p, half, with_prefix, &maps);
    set_parts(streams ? s.s_pp : s.n_pp, streams ? s.s_cp : s.n_cp);
    p.out = out, p.o_t = out_strides[0], p.o_h = out_strides[1];
    p.lse = lse, p.status = status;

    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (s.units_tile) {
        e = launch_attention_tiles(p, half, s.fused, s.fused ? s.tiles_c : s.tiles_p, s.n_pp, kSms,
                                   s.units_tile, false, st);
        if (e != cudaSuccess) return cuda_error(e, "attention tiles launch");
    }
    if (s.units_rows) {
        if (streams)
            e = launch_attention_stream(p, maps, half, with_prefix, s.v.dp, s.stream_mt, s.least, s.blocks,
                                        s.units_tile > 0, st);
        else
            e = half ? launch_rows_dp<__half>(p, s.v, s.units_rows, st)
                     : launch_rows_dp<__nv_bfloat16>(p, s.v, s.units_rows, st);
        if (e != cudaSuccess) return cuda_error(e, "attention launch");
    }
    if (s.direct) return ok();
    const bool after = s.units_tile > 0 || s.units_rows > 0;
    e = half ? launch_join<__half>(p, rows, after, st) : launch_join<__nv_bfloat16>(p, rows, after, st);
    if (e != cudaSuccess) return cuda_error(e, "attention join launch");
    return ok();
}
