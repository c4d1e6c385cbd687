// sc_evict.cu — a cache cut to its budget by accumulated attention weight.
//
// Definition.  Of a (sequence, KV head)'s len tokens, min(len, budget) stay: the first
// keep_first and the last keep_recent, and of the others those of the highest score, equal
// scores by the lower index (NaN counts as minus infinity).  The kept keys, values and scores
// move together to the front, in their order.
//
// select_tokens: one block, or a cluster of up to 16, holds the scores of a (b, h) as ordered
// 32-bit keys in registers (read from HBM once, every load in flight at once) and finds the last
// kept key by three radix passes (11, 11 and 10 bits, from the top) over histograms in shared
// memory, added up in the first block's through distributed shared memory.  A token's place is then
// the number of kept tokens before it: (those above the key or forced) + min(equal ones before
// it, equal ones wanted), so one count per warp and one scan are enough and no order depends on
// timing.  (Keys in shared memory, 512 threads, clusters of 8: 20 us for 128 rows of 8,192 and 50
// for 8 rows of 131,072.)
//
// move_rows / move_rows_in_place: the kept rows, 16 bytes a lane.  In place, row i comes from
// row idx[i] >= i, so a block that owns a column slice of a (b, h) moves it front to back: a
// step's loads come before its stores, and stores reach only rows that later steps do not read.
// HBM bounds both: every kept row is read and written once.
//
// Measured: 128 rows of up to 8,192 tokens to 2,048, selection 11 us and move 49, as long as a plain
// copy of the kept rows; 8 rows of 131,072 to 16,384, 20.5 and 26.  In place the latter's move takes 345:
// 72 blocks of 128 threads, each 128 rounds that wait for one another.
#include <cooperative_groups.h>

#include "sc_common.cuh"

namespace cg = cooperative_groups;

namespace sc {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 16;
constexpr int kMaxKeys = 32;  // a thread
constexpr int kMaxTokens = 393216;  // as documented; the registers of 16 blocks would hold 524,288 keys

struct SelectParams {
    const float* scores;
    int64_t s_b, s_h;
    const int32_t* cache_lens;
    int32_t* new_lens;
    int32_t* indices;  // [B, H, budget]
    int32_t B, H, S, budget, first, recent;
    int32_t* status;
};

// fp32 scores as unsigned keys of the same order; -0 becomes +0 and NaN minus infinity.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    if (x != x) return 0x007fffffu;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int evict_length(const int32_t* lens, int b, int S, int32_t* status) {
    if (lens == nullptr) return S;
    const int len = lens[b];
    if (len < 0 || len > S) {
        if (threadIdx.x == 0) atomicOr(status, SC_STATUS_BAD_SEQ_LEN);
        return 0;
    }
    return len;
}

__device__ __forceinline__ int warp_scan(int x, int lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    return x;
}

// The sum of x over the warps before this one (x: one value a warp) and over all.  Called by
// every thread; s_warp is free again after the next block-wide barrier.
__device__ __forceinline__ int warps_before(int x, int& total, int* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) s_warp[warp] = x;
    __syncthreads();
    const int v = warp_scan(s_warp[lane], lane);
    total = __shfl_sync(0xffffffffu, v, 31);
    return __shfl_sync(0xffffffffu, v, warp) - x;
}

// KPT keys a thread: warp w of rank r holds tokens [(r * 32 + w) * 32 KPT, + 32 KPT), key j of lane l
// being token 32 j + l of them.
template <int KPT>
__global__ void __launch_bounds__(kSelThreads) select_tokens(const __grid_constant__ SelectParams p) {
    __shared__ uint32_t s_hist[kBins];
    __shared__ uint32_t s_all[2][kBins];  // the first block's: the cluster's histograms, in turn
    __shared__ int s_warp[3][kSelWarps];
    __shared__ int2 s_pick[2];   // digit, equal ones still wanted; in turn
    __shared__ int s_counts[2];  // this block's kept-for-sure and equal tokens
    let_next_start();
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank());
    const int ranks = static_cast<int>(cluster.num_blocks());
    auto sync_all = [&] {
        if (ranks > 1)
            cluster.sync();
        else
            __syncthreads();
    };
    const int row = blockIdx.x / ranks;
    const int b = row / p.H, h = row - b * p.H;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

    const int len = evict_length(p.cache_lens, b, p.S, p.status);
    const int n_new = min(len, p.budget);
    int32_t* idx = p.indices + static_cast<int64_t>(row) * p.budget;
    for (int i = n_new + rank * kSelThreads + threadIdx.x; i < p.budget; i += ranks * kSelThreads)
        idx[i] = -1;
    if (h == 0 && rank == 0 && threadIdx.x == 0) p.new_lens[b] = n_new;
    if (len <= p.budget) {  // everything stays
        for (int i = rank * kSelThreads + threadIdx.x; i < len; i += ranks * kSelThreads) idx[i] = i;
        return;  // the whole cluster takes this way
    }

    // Free tokens are [lo, hi); budget >= first + recent, so some of them go.
    const int lo = min(p.first, len), hi = max(lo, len - p.recent);
    const int t0 = (rank * kSelWarps + warp) * 32 * KPT + lane;
    const float* scores = p.scores + b * p.s_b + h * p.s_h;
    float raw[KPT];
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        const int t = t0 + 32 * j;
        raw[j] = t >= lo && t < hi ? __ldg(scores + t) : 0.f;
    }
    if (ranks > 1) {
        if (rank == 0)
            for (int i = threadIdx.x; i < kBins; i += kSelThreads) s_all[0][i] = 0;
        cluster.sync();
    }
    uint32_t keys[KPT];
#pragma unroll
    for (int j = 0; j < KPT; ++j) keys[j] = order_key(raw[j]);

    int want = n_new - lo - (len - hi);  // free tokens that stay
    uint32_t key = 0;                    // the last kept key's bits found so far
    int shift = 32;
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10;
        const uint32_t above = shift == 32 ? 0u : key >> shift;
        const int top = shift;
        shift -= bits;
        const uint32_t digits = (1u << bits) - 1u;
        for (int i = threadIdx.x; i < kBins; i += kSelThreads) s_hist[i] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
            const int t = t0 + 32 * j;
            if (t >= lo && t < hi && (top == 32 || (keys[j] >> top) == above))
                atomicAdd(&s_hist[(keys[j] >> shift) & digits], 1u);
        }
        if (ranks > 1) {
            __syncthreads();
            uint32_t* all = cluster.map_shared_rank(s_all[pass & 1], 0);
            for (int i = threadIdx.x; i < kBins; i += kSelThreads) {
                if (s_hist[i]) atomicAdd(&all[i], s_hist[i]);
                if (rank == 0) s_all[(pass + 1) & 1][i] = 0;  // last read a pass ago
            }
        }
        sync_all();
        if (rank == 0) {
            // Bins in descending order, two a thread.
            static_assert(kBins == 2 * kSelThreads, "two bins a thread");
            const uint32_t* all = ranks > 1 ? s_all[pass & 1] : s_hist;
            const int bin = kBins - 1 - 2 * threadIdx.x;
            const int n0 = static_cast<int>(all[bin]), n1 = static_cast<int>(all[bin - 1]);
            const int upto = warp_scan(n0 + n1, lane);
            int total;
            const int before =
                warps_before(__shfl_sync(0xffffffffu, upto, 31), total, s_warp[0]) + upto - n0 - n1;
            if (want > 0 && before < want && before + n0 + n1 >= want) {
                const bool second = before + n0 < want;
                const int2 pick = make_int2(second ? bin - 1 : bin, want - before - (second ? n0 : 0));
                for (int r = 0; r < ranks; ++r) *cluster.map_shared_rank(&s_pick[pass & 1], r) = pick;
            }
        }
        sync_all();
        if (want > 0) {
            const int2 pick = s_pick[pass & 1];
            key |= static_cast<uint32_t>(pick.x) << shift;
            want = pick.y;
        }
    }
    // Free tokens above `key` stay, and the first `want` equal to it (want = 0: none do).
    const int wanted = want;
    const bool none = n_new - lo - (len - hi) <= 0;

    auto kind = [&](int j) -> int {  // 0 goes, 1 stays, 2 equal
        const int t = t0 + 32 * j;
        if (t >= len) return 0;
        if (t < lo || t >= hi) return 1;
        if (none) return 0;
        return keys[j] > key ? 1 : keys[j] == key ? 2 : 0;
    };
    int stay = 0, equal = 0;
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        const int k = kind(j);
        stay += __popc(__ballot_sync(0xffffffffu, k == 1));
        equal += __popc(__ballot_sync(0xffffffffu, k == 2));
    }
    int total_stay, total_equal;
    int g = warps_before(stay, total_stay, s_warp[1]), e = warps_before(equal, total_equal, s_warp[2]);
    if (ranks > 1) {
        if (threadIdx.x == 0) {
            s_counts[0] = total_stay;
            s_counts[1] = total_equal;
        }
        cluster.sync();
        int cg_ = 0, ce = 0;  // a lane a rank before this one
        if (lane < rank) {
            const int* c = cluster.map_shared_rank(s_counts, lane);
            cg_ = c[0], ce = c[1];
        }
        g += __reduce_add_sync(0xffffffffu, cg_);
        e += __reduce_add_sync(0xffffffffu, ce);
    }
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        const int k = kind(j);
        const uint32_t bs = __ballot_sync(0xffffffffu, k == 1), be = __ballot_sync(0xffffffffu, k == 2);
        const uint32_t below = (1u << lane) - 1u;
        const int gb = g + __popc(bs & below), eb = e + __popc(be & below);
        if (k == 1 || (k == 2 && eb < wanted)) idx[gb + min(eb, wanted)] = t0 + 32 * j;
        g += __popc(bs);
        e += __popc(be);
    }
    if (ranks > 1) cluster.sync();  // no block leaves while another reads its shared memory
}

// ---------------------------------------------------------------------------------------
constexpr int kMoveThreads = 128;
constexpr int kMoveUnroll = 4;

struct MoveTensor {
    const void* src;
    void* dst;
    int64_t s_b, s_t, s_h;  // bytes
    int64_t d_b, d_t, d_h;
};
struct MoveParams {
    MoveTensor x[3];  // keys, values, scores
    const int32_t* indices;
    int32_t H, budget;
    int32_t row16;    // 16-byte pieces of a key row (scores: one 4-byte piece)
    FastDiv div_row16;
    int32_t slice16;  // in place: pieces of a slice
    int32_t slices;   // in place: slices of a key row
};

__global__ void __launch_bounds__(kMoveThreads) move_rows(const __grid_constant__ MoveParams p) {
    wait_for_previous();
    const MoveTensor& x = p.x[blockIdx.z];
    const int row = blockIdx.y, b = row / p.H, h = row - b * p.H;
    const int32_t* idx = p.indices + static_cast<int64_t>(row) * p.budget;
    const char* src = static_cast<const char*>(x.src) + b * x.s_b + h * x.s_h;
    char* dst = static_cast<char*>(x.dst) + b * x.d_b + h * x.d_h;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kMoveThreads * kMoveUnroll + threadIdx.x;
    if (blockIdx.z == 2) {
#pragma unroll
        for (int j = 0; j < kMoveUnroll; ++j) {
            const int64_t i = first + j * kMoveThreads;
            if (i < p.budget) {
                const int t = idx[i];
                if (t >= 0)
                    *reinterpret_cast<float*>(dst + i * x.d_t) =
                        *reinterpret_cast<const float*>(src + t * x.s_t);
            }
        }
        return;
    }
    const int64_t all = static_cast<int64_t>(p.budget) * p.row16;
    int from[kMoveUnroll], to[kMoveUnroll], c[kMoveUnroll];
#pragma unroll
    for (int j = 0; j < kMoveUnroll; ++j) {
        const int64_t w = first + j * kMoveThreads;
        from[j] = -1;
        if (w < all) {
            to[j] = static_cast<int>(fdiv(static_cast<uint32_t>(w), p.div_row16));
            c[j] = static_cast<int>(w) - to[j] * p.row16;
            from[j] = idx[to[j]];
        }
    }
    uint4 v[kMoveUnroll];
#pragma unroll
    for (int j = 0; j < kMoveUnroll; ++j)
        if (from[j] >= 0) v[j] = ld_stream_v4(src + from[j] * x.s_t + c[j] * 16);
#pragma unroll
    for (int j = 0; j < kMoveUnroll; ++j)
        if (from[j] >= 0) st_v4(dst + to[j] * x.d_t + c[j] * 16, v[j]);
}

// blockIdx.x: a slice of the keys, of the values, or the scores.  W: 16-byte pieces or floats.
template <typename W>
__device__ __forceinline__ void move_slice(const char* src, char* dst, int64_t s_t, int64_t d_t,
                                           const int32_t* idx, int budget, int pieces) {
    const int rows = kMoveThreads / pieces;  // rows a round of the block
    const int r = threadIdx.x / pieces, c = threadIdx.x - r * pieces;
    const bool in = r < rows;
    const int step = rows * kMoveUnroll;
    W cur[kMoveUnroll], next[kMoveUnroll];
    auto load = [&](int i0, W(&v)[kMoveUnroll]) {
#pragma unroll
        for (int j = 0; j < kMoveUnroll; ++j) {
            const int i = i0 + j * rows + r;
            const int t = in && i < budget ? idx[i] : -1;
            if (t >= 0) v[j] = *reinterpret_cast<const W*>(src + t * s_t + c * static_cast<int>(sizeof(W)));
        }
    };
    load(0, cur);
    for (int i0 = 0; i0 < budget; i0 += step) {
        load(i0 + step, next);
        __syncthreads();  // every load of rows [i0, i0 + step) is before the stores there
#pragma unroll
        for (int j = 0; j < kMoveUnroll; ++j) {
            const int i = i0 + j * rows + r;
            const int t = in && i < budget ? idx[i] : -1;
            if (t >= 0) *reinterpret_cast<W*>(dst + i * d_t + c * static_cast<int>(sizeof(W))) = cur[j];
            cur[j] = next[j];
        }
    }
}

__global__ void __launch_bounds__(kMoveThreads) move_rows_in_place(const __grid_constant__ MoveParams p) {
    wait_for_previous();
    const int row = blockIdx.y, b = row / p.H, h = row - b * p.H;
    const int32_t* idx = p.indices + static_cast<int64_t>(row) * p.budget;
    const int which = blockIdx.x < 2 * p.slices ? blockIdx.x / p.slices : 2;
    const MoveTensor& x = p.x[which];
    const char* src = static_cast<const char*>(x.src) + b * x.s_b + h * x.s_h;
    char* dst = static_cast<char*>(x.dst) + b * x.d_b + h * x.d_h;
    if (which == 2) {
        move_slice<float>(src, dst, x.s_t, x.d_t, idx, p.budget, 1);
    } else {
        const int c0 = (blockIdx.x - which * p.slices) * p.slice16;
        const int n = min(p.slice16, p.row16 - c0);
        move_slice<uint4>(src + c0 * 16, dst + c0 * 16, x.s_t, x.d_t, idx, p.budget, n);
    }
}

template <int KPT>
cudaError_t launch_select(const SelectParams& p, int ranks, cudaStream_t s, bool load_only) {
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_clusters(reinterpret_cast<const void*>(select_tokens<KPT>), done);
    if (e != cudaSuccess || load_only) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(p.B * p.H * ranks));
    cfg.blockDim = dim3(kSelThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(ranks);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, select_tokens<KPT>, p);
}

}  // namespace

cudaError_t preload_evict_kernels() {
    SelectParams p{};
    cudaError_t e = launch_select<8>(p, 1, nullptr, true);
    if (e == cudaSuccess) e = launch_select<16>(p, 1, nullptr, true);
    if (e == cudaSuccess) e = launch_select<kMaxKeys>(p, 1, nullptr, true);
    cudaFuncAttributes attr;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, move_rows);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, move_rows_in_place);
    return e;
}

}  // namespace sc

using namespace sc;

extern "C" int32_t sc_evict_tokens(int32_t batch, int32_t n_heads, int64_t cache_len,
                                   int32_t head_dim, int32_t elem_size, int64_t budget,
                                   int64_t keep_first, int64_t keep_recent, const void* k_cache,
                                   const int64_t* kc_strides, const void* v_cache,
                                   const int64_t* vc_strides, const float* scores,
                                   const int64_t* scores_strides, const int32_t* cache_lens,
                                   int32_t in_place, void* k_out, const int64_t* ko_strides,
                                   void* v_out, const int64_t* vo_strides, float* scores_out,
                                   const int64_t* so_strides, int32_t* indices, int32_t* new_lens,
                                   int32_t* status, void* stream) {
    if (batch < 0 || n_heads < 0 || cache_len < 0 || head_dim < 0 || budget < 0 || keep_first < 0 ||
        keep_recent < 0)
        return set_error(SC_ERR_INVALID_ARGUMENT, "negative size");
    if (elem_size != 1 && elem_size != 2 && elem_size != 4)
        return set_error(SC_ERR_INVALID_DTYPE, "elements of %d bytes: 1, 2 or 4", elem_size);
    if (head_dim > kMaxHeadDim)
        return set_error(SC_ERR_UNSUPPORTED, "head_dim %d exceeds %d", head_dim, kMaxHeadDim);
    const int32_t row_bytes = head_dim * elem_size;
    if (keep_first > budget || keep_recent > budget - keep_first)
        return set_error(SC_ERR_INVALID_ARGUMENT,
                         "keep_first %lld and keep_recent %lld exceed the budget of %lld tokens",
                         (long long)keep_first, (long long)keep_recent, (long long)budget);
    if (row_bytes % 16 != 0)
        return set_error(SC_ERR_UNSUPPORTED, "rows of %d bytes: a multiple of 16", row_bytes);
    if (cache_len > kMaxTokens)
        return set_error(SC_ERR_UNSUPPORTED, "caches of %lld tokens: at most %d", (long long)cache_len,
                         kMaxTokens);
    if (budget >= (int64_t(1) << 24) || size_product(budget, row_bytes / 16) >= (int64_t(1) << 31) ||
        size_product(batch, n_heads) > 65535)
        return set_error(SC_ERR_INVALID_ARGUMENT, "too many rows in one call; split it");
    if (batch == 0) return ok();
    if (!new_lens || !status) return set_error(SC_ERR_INVALID_ARGUMENT, "null pointer argument");
    const int64_t rows = static_cast<int64_t>(batch) * n_heads;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        const cudaError_t e = cudaMemsetAsync(new_lens, 0, sizeof(int32_t) * batch, st);
        return e == cudaSuccess ? ok() : cuda_error(e, "clearing the lengths");
    }
    if (!kc_strides || !vc_strides || !scores_strides || !ko_strides || !vo_strides || !so_strides ||
        (cache_len && (!scores || (row_bytes && (!k_cache || !v_cache)))) ||
        (budget && (!indices || !scores_out || (row_bytes && (!k_out || !v_out)))))
        return set_error(SC_ERR_INVALID_ARGUMENT, "null pointer argument");
    auto aligned = [&](const void* ptr, const int64_t* s) {
        const int64_t n = 16 / elem_size;
        return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && s[0] % n == 0 && s[1] % n == 0 &&
               s[2] % n == 0;
    };
    if (!aligned(k_cache, kc_strides) || !aligned(v_cache, vc_strides) || !aligned(k_out, ko_strides) ||
        !aligned(v_out, vo_strides))
        return set_error(SC_ERR_INVALID_ARGUMENT, "rows must start at multiples of 16 bytes");

    SelectParams sp{};
    sp.scores = scores, sp.s_b = scores_strides[0], sp.s_h = scores_strides[1];
    sp.cache_lens = cache_lens, sp.new_lens = new_lens, sp.indices = indices;
    sp.B = batch, sp.H = n_heads, sp.S = static_cast<int32_t>(cache_len);
    sp.budget = static_cast<int32_t>(budget);
    sp.first = static_cast<int32_t>(keep_first), sp.recent = static_cast<int32_t>(keep_recent);
    sp.status = status;
    // A cluster where there are fewer rows than SMs, down to 16 keys a thread (8 rows of 131,072 to
    // 16,384, move included: 47.2 us; 8 keys and twice the blocks 61.0, 32 keys 57.4), or where one
    // block cannot hold a row's keys.
    int ranks = 1;
    auto per_thread = [&] { return (cache_len + ranks * kSelThreads - 1) / (ranks * kSelThreads); };
    while (ranks < kMaxCluster && (per_thread() > kMaxKeys || (rows * ranks * 2 <= 148 && per_thread() > 16)))
        ranks *= 2;
    cudaError_t e = per_thread() <= 8    ? launch_select<8>(sp, ranks, st, false)
                    : per_thread() <= 16 ? launch_select<16>(sp, ranks, st, false)
                                         : launch_select<kMaxKeys>(sp, ranks, st, false);
    if (e != cudaSuccess) return cuda_error(e, "eviction select launch");
    if (budget == 0) return ok();

    MoveParams mp{};
    auto fill = [](MoveTensor& t, const void* src, const int64_t* ss, void* dst, const int64_t* ds,
                   int64_t size) {
        t.src = src, t.dst = dst;
        t.s_b = ss[0] * size, t.s_t = ss[1] * size, t.s_h = ss[2] * size;
        t.d_b = ds[0] * size, t.d_t = ds[1] * size, t.d_h = ds[2] * size;
    };
    const int64_t ss[3] = {scores_strides[0], 1, scores_strides[1]};
    const int64_t so[3] = {so_strides[0], 1, so_strides[1]};
    fill(mp.x[0], k_cache, kc_strides, k_out, ko_strides, elem_size);
    fill(mp.x[1], v_cache, vc_strides, v_out, vo_strides, elem_size);
    fill(mp.x[2], scores, ss, scores_out, so, 4);
    mp.indices = indices, mp.H = n_heads, mp.budget = sp.budget;
    mp.row16 = row_bytes / 16;
    mp.div_row16 = make_fastdiv(static_cast<uint32_t>(mp.row16 ? mp.row16 : 1));
    if (in_place) {
        mp.slice16 = 4;  // 64 bytes: the DRAM access granularity
        mp.slices = (mp.row16 + mp.slice16 - 1) / mp.slice16;
        e = launch_chained(move_rows_in_place, dim3(2 * mp.slices + 1, static_cast<unsigned>(rows)), kMoveThreads, 0,
                           st, true, mp);
    } else {
        const int64_t pieces = budget * (mp.row16 ? mp.row16 : 1);
        const int64_t per = kMoveThreads * kMoveUnroll;
        e = launch_chained(move_rows, dim3(static_cast<unsigned>((pieces + per - 1) / per), static_cast<unsigned>(rows), 3),
                           kMoveThreads, 0, st, true, mp);
    }
    if (e != cudaSuccess) return cuda_error(e, "eviction move launch");
    return ok();
}
