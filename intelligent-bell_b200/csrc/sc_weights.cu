// sc_weights.cu — attention weights added up per cached token, the measure an eviction goes by.
//
// Mathematics.  For KV head h and token t of sequence b,
//   out[b, h, t] = scores[b, h, t] + sum over the sequence's rows (query j, head g of the group
//                  of h) that see t of e^{scale q_{j,g} . k_t - lse_{j,g}},
// the weights that the attention gave, from its log-sum-exp, without a second softmax pass.
//
// add_weights: tokens are the rows of the matrix product and queries its columns, so a token's
// sum stays in the registers of four lanes and is joined by two shuffles: no atomics, one order
// of addition.  A warp loads 32 tokens (its own cp.async ring), keeps them as fragments, and
// walks over the queries in shared memory.  With few queries it waits for the keys (HBM); with
// many, for the exponentials.  weigh_tiles (sc_weights_tile.cu) is faster wherever its tensor maps
// can say the layout (16 sequences of up to 8,192 tokens 29 us against 60, 64 queries on 32,768
// tokens 37 against 158); this kernel takes head_dim above 128, more than 128 heads a group, more
// than 1,024 sequences and expanded strides.
#include <limits.h>
#include <math.h>

#include "sc_weights.cuh"

namespace sc {
namespace {

constexpr int kWWarps = 4;
constexpr int kWThreads = 32 * kWWarps;
constexpr int kWTile = 32;                     // tokens a warp's tile
constexpr int kWBlock = kWTile * kWWarps;      // tokens a block's step

template <int DP>
__device__ __forceinline__ uint32_t w_chunk_at(int r, int c) {
    return static_cast<uint32_t>(r) * (DP * 2) + static_cast<uint32_t>((c ^ (r & 7)) * 16);
}

template <typename T, int DP, int NST>
__global__ void __launch_bounds__(kWThreads) add_weights(const __grid_constant__ WeightParams p) {
    constexpr int CPR = DP / 8, RPI = 32 / CPR, KT = kWTile * DP * 2;
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* s_ring = smem;
    unsigned char* s_q = smem + kWWarps * NST * KT;
    float* s_lse = reinterpret_cast<float*>(s_q + p.row_room * DP * 2);
    int* s_lim = reinterpret_cast<int*>(s_lse + p.row_room);

    int u = blockIdx.x;
    const int part = u % p.parts;
    u /= p.parts;
    const int h = u % p.Hkv, b = u / p.Hkv;

    int tok0, n_tok;
    if (!Starts(p.cu_q, p.B, p.N, p.nq).of(b, tok0, n_tok) && threadIdx.x == 0)
        atomicOr(p.status, SC_STATUS_BAD_SEQ_LEN);
    int len = p.S;
    if (p.cache_lens != nullptr) {
        len = p.cache_lens[b];
        if (len < 0 || len > p.S) {
            if (threadIdx.x == 0) atomicOr(p.status, SC_STATUS_BAD_SEQ_LEN);
            len = 0;
        }
    }
    const int rows = n_tok * p.G;
    const int t0 = part * p.chunk, t_end = min(p.S, t0 + p.chunk);
    const int t1 = rows > 0 ? min(t_end, len) : t0;  // tokens that get something
    const float* in = p.scores + b * p.s_b + h * p.s_h;
    float* out = p.out + b * p.o_b + h * p.o_h;
    if (in != out)
        for (int t = max(t0, t1) + threadIdx.x; t < t_end; t += kWThreads) out[t] = in[t];
    if (t0 >= t1) return;

    const T* kbase = static_cast<const T*>(p.k) + b * p.k_b + h * p.k_h;
    const uint32_t ring = smem_addr(s_ring) + warp * NST * KT;
    const int steps = (t1 - t0 + kWBlock - 1) / kWBlock;
    auto issue = [&](int i) {
        const int tt = t0 + i * kWBlock + warp * kWTile;
        const int c = lane % CPR;
        if (i < steps && c * 8 < p.D) {
            const uint32_t dst = ring + (i % NST) * KT;
#pragma unroll
            for (int it = 0; it < kWTile / RPI; ++it) {
                const int r = it * RPI + lane / CPR;
                const bool valid = tt + r < t1;
                cp_async16(dst + w_chunk_at<DP>(r, c),
                           kbase + (valid ? (tt + r) * p.k_t : 0) + c * 8, valid);
            }
        }
        cp_async_commit();
    };
    if (p.D < DP) {  // columns that no copy writes
        for (int i = threadIdx.x; i < kWWarps * NST * KT / 16; i += kWThreads)
            reinterpret_cast<uint4*>(s_ring)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    for (int i = 0; i < NST - 1; ++i) issue(i);

    auto load_rows = [&](int r0, int n) {  // n <= row_room rows from r0, padded to 8
        const int padded = (n + 7) & ~7;
        for (int i = threadIdx.x; i < padded * CPR; i += kWThreads) {
            const int r = i / CPR, c = i - r * CPR;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < n && c * 8 < p.D) {
                const int j = static_cast<int>(fdiv(r0 + r, p.div_G));
                const int g = r0 + r - j * p.G;
                v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (tok0 + j) * p.q_t +
                                                    (h * p.G + g) * p.q_h + c * 8);
            }
            *reinterpret_cast<uint4*>(s_q + w_chunk_at<DP>(r, c)) = v;
        }
        for (int r = threadIdx.x; r < padded; r += kWThreads) {
            float x = 0.f;
            int lim = INT_MIN;
            if (r < n) {
                const int j = static_cast<int>(fdiv(r0 + r, p.div_G));
                const int g = r0 + r - j * p.G;
                x = p.lse[(tok0 + j) * p.lse_t + (h * p.G + g) * p.lse_h] * 1.4426950408889634f;
                // a row that saw nothing gives nothing
                if (x != kNegInf) lim = p.causal ? len - n_tok + j + 1 : INT_MAX;
            }
            s_lse[r] = x;
            s_lim[r] = lim;
        }
    };
    const int chunks = (rows + p.row_room - 1) / p.row_room;
    if (chunks == 1) load_rows(0, rows);
    __syncthreads();

    const uint32_t q_addr = smem_addr(s_q);
    for (int i = 0; i < steps; ++i) {
        cp_async_wait<NST - 2>();
        __syncwarp();
        issue(i + NST - 1);
        const uint32_t kt = ring + (i % NST) * KT;
        const int tt = t0 + i * kWBlock + warp * kWTile;
        uint32_t a[2][DP / 16][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk)
                ldmatrix4(a[mt][kk], kt + w_chunk_at<DP>(mt * 16 + (lane & 15), kk * 2 + (lane >> 4)));
        float acc[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
        for (int ch = 0; ch < chunks; ++ch) {
            const int r0 = ch * p.row_room, n = min(p.row_room, rows - r0);
            if (chunks > 1) {
                __syncthreads();
                load_rows(r0, n);
                __syncthreads();
            }
            if (tt >= t1) continue;
            for (int r = 0; r < n; r += 8) {
                float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk += 2) {
                    uint32_t qb[4];
                    ldmatrix4(qb, q_addr + w_chunk_at<DP>(r + (lane & 7), kk * 2 + (lane >> 3)));
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        mma16816<T>(s[mt], a[mt][kk], qb[0], qb[1]);
                        mma16816<T>(s[mt], a[mt][kk + 1], qb[2], qb[3]);
                    }
                }
                const int r1 = r + (lane & 3) * 2;
                const float2 ls = *reinterpret_cast<const float2*>(s_lse + r1);
                const int2 lim = *reinterpret_cast<const int2*>(s_lim + r1);
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int t = tt + mt * 16 + e * 8 + (lane >> 2);
                        const float w0 = exp2_fast(fmaf(s[mt][2 * e], p.scale_log2, -ls.x));
                        const float w1 = exp2_fast(fmaf(s[mt][2 * e + 1], p.scale_log2, -ls.y));
                        acc[mt][e] += t < lim.x ? w0 : 0.f;
                        acc[mt][e] += t < lim.y ? w1 : 0.f;
                    }
            }
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = acc[mt][e];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                const int t = tt + mt * 16 + e * 8 + (lane >> 2);
                if ((lane & 3) == 0 && t < t1) out[t] = in[t] + x;
            }
    }
    cp_async_wait<0>();
}

template <typename T, int DP, int NST>
cudaError_t launch_weights(const WeightParams& p, int64_t blocks, cudaStream_t s, bool load_only) {
    auto kernel = add_weights<T, DP, NST>;
    constexpr int kMost = kWWarps * NST * kWTile * DP * 2 + (DP == 256 ? 128 : 256) * (DP * 2 + 8);
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_shared_memory(reinterpret_cast<const void*>(kernel), kMost, done);
    if (e != cudaSuccess || load_only) return e;
    const int bytes = kWWarps * NST * kWTile * DP * 2 + p.row_room * (DP * 2 + 8);
    kernel<<<static_cast<unsigned>(blocks), kWThreads, bytes, s>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_weights_dp(const WeightParams& p, int64_t blocks, cudaStream_t s) {
    if (p.D <= 64) return launch_weights<T, 64, 4>(p, blocks, s, false);
    if (p.D <= 128) return launch_weights<T, 128, 3>(p, blocks, s, false);
    return launch_weights<T, 256, 2>(p, blocks, s, false);
}

template <typename T>
cudaError_t preload_weights_type() {
    WeightParams p{};
    cudaError_t e = launch_weights<T, 64, 4>(p, 0, nullptr, true);
    if (e == cudaSuccess) e = launch_weights<T, 128, 3>(p, 0, nullptr, true);
    if (e == cudaSuccess) e = launch_weights<T, 256, 2>(p, 0, nullptr, true);
    return e;
}

}  // namespace

cudaError_t preload_weights_kernels() {
    cudaError_t e = preload_weights_type<__half>();
    if (e == cudaSuccess) e = preload_weights_type<__nv_bfloat16>();
    if (e == cudaSuccess) e = preload_weight_tile_kernels();
    return e;
}

}  // namespace sc

using namespace sc;

extern "C" int32_t sc_accumulate_attention_weights(
    int64_t n_tokens, int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
    int32_t dtype, const void* q, const int64_t* q_strides, int64_t cache_len, const void* k_cache,
    const int64_t* kc_strides, const int32_t* cache_lens, const int32_t* cu_q_lens,
    int64_t max_q_len, int32_t causal, double scale, const float* lse, const int64_t* lse_strides,
    const float* scores, const int64_t* scores_strides, float* out, const int64_t* out_strides,
    int32_t* status, void* stream) {
    if (n_tokens < 0 || batch < 0 || q_heads < 0 || kv_heads < 0 || cache_len < 0 || max_q_len < 0)
        return set_error(SC_ERR_INVALID_ARGUMENT, "negative size");
    if (kv_heads == 0 ? q_heads != 0 : q_heads % kv_heads != 0)
        return set_error(SC_ERR_INVALID_ARGUMENT, "%d query heads are no multiple of %d KV heads",
                         q_heads, kv_heads);
    if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > 256)
        return set_error(SC_ERR_UNSUPPORTED, "head_dim %d: a multiple of 8, at most 256", head_dim);
    if (dtype != SC_DTYPE_F16 && dtype != SC_DTYPE_BF16)
        return set_error(SC_ERR_INVALID_DTYPE, "dtype code %d: float16 or bfloat16", dtype);
    if (!isfinite(static_cast<float>(scale * 1.4426950408889634)))
        return set_error(SC_ERR_INVALID_ARGUMENT, "scale must be finite in float32, got %g", scale);
    if (size_product(n_tokens, q_heads) >= (int64_t(1) << 31) || cache_len >= (int64_t(1) << 30) ||
        size_product(max_q_len, q_heads) >= (int64_t(1) << 31))
        return set_error(SC_ERR_INVALID_ARGUMENT, "too many rows or tokens in one call; split it");
    if (!cu_q_lens && n_tokens != size_product(max_q_len, batch))
        return set_error(SC_ERR_INVALID_ARGUMENT, "%lld tokens are not %d sequences of %lld",
                         (long long)n_tokens, batch, (long long)max_q_len);
    if (batch == 0 || kv_heads == 0 || cache_len == 0) return ok();
    const bool rows = n_tokens > 0 && q_heads > 0;
    if (!scores || !out || !scores_strides || !out_strides || !status ||
        (rows && (!q || !q_strides || !k_cache || !kc_strides || !lse || !lse_strides)))
        return set_error(SC_ERR_INVALID_ARGUMENT, "null pointer argument");
    if (rows && (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(k_cache) % 16 ||
                 q_strides[0] % 8 || q_strides[1] % 8 || kc_strides[0] % 8 || kc_strides[1] % 8 ||
                 kc_strides[2] % 8))
        return set_error(SC_ERR_INVALID_ARGUMENT, "rows must start at multiples of 16 bytes");

    WeightParams p{};
    p.q = q, p.k = k_cache, p.lse = lse, p.scores = scores, p.out = out;
    if (rows) {
        p.q_t = q_strides[0], p.q_h = q_strides[1];
        p.k_b = kc_strides[0], p.k_t = kc_strides[1], p.k_h = kc_strides[2];
        p.lse_t = lse_strides[0], p.lse_h = lse_strides[1];
    }
    p.s_b = scores_strides[0], p.s_h = scores_strides[1];
    p.o_b = out_strides[0], p.o_h = out_strides[1];
    p.cache_lens = cache_lens, p.cu_q = cu_q_lens;
    p.N = static_cast<int32_t>(n_tokens), p.B = batch, p.Hq = q_heads, p.Hkv = kv_heads;
    p.G = rows ? q_heads / kv_heads : 1;
    p.D = head_dim, p.nq = rows ? static_cast<int32_t>(max_q_len) : 0;
    if (!rows) p.cu_q = nullptr;
    p.S = static_cast<int32_t>(cache_len), p.causal = causal != 0;
    p.div_G = make_fastdiv(static_cast<uint32_t>(p.G));
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    p.status = status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    bool taken = false;
    cudaError_t e = launch_weight_tiles(p, dtype == SC_DTYPE_F16, s, &taken);
    if (e != cudaSuccess) return cuda_error(e, "attention weights launch");
    if (taken) return ok();
    const int64_t most = size_product(p.nq, p.G);
    const int room = head_dim > 128 ? 128 : 256;
    p.row_room = most >= room ? room : most < 16 ? 16 : static_cast<int32_t>((most + 15) / 16 * 16);
    // Two blocks an SM; two rounds of them.
    const double total = static_cast<double>(batch) * kv_heads * cache_len;
    double chunk = ceil(total / (148.0 * 2 * 4) / kWBlock) * kWBlock;
    if (chunk > cache_len) chunk = ceil(static_cast<double>(cache_len) / kWBlock) * kWBlock;
    p.chunk = static_cast<int32_t>(chunk);
    p.parts = static_cast<int32_t>((cache_len + p.chunk - 1) / p.chunk);
    const int64_t blocks = size_product(p.parts, batch, kv_heads);
    if (blocks >= (int64_t(1) << 31))
        return set_error(SC_ERR_INVALID_ARGUMENT, "%lld blocks in one call; split it", (long long)blocks);
    e = dtype == SC_DTYPE_F16 ? launch_weights_dp<__half>(p, blocks, s)
                              : launch_weights_dp<__nv_bfloat16>(p, blocks, s);
    if (e != cudaSuccess) return cuda_error(e, "attention weights launch");
    return ok();
}
