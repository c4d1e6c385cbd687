// sc_evict.cu — a cache cut to its budget by accumulated attention weight.
//
// Definition.  Of a (sequence, KV head)'s len tokens, min(len, budget) stay: the first
// keep_first and the last keep_recent, and of the others those of the highest score, equal
// scores by the lower index (NaN counts as minus infinity).  The kept keys, values and scores
// move together to the front, in their order.
//
// select_tokens: one block, or a cluster of up to 8, holds the scores of a (b, h) as ordered
// 32-bit keys in shared memory (read from HBM once) and finds the last kept key by three radix
// passes (11, 11 and 10 bits, from the top) over histograms in shared memory, summed over the
// cluster through distributed shared memory.  A token's place is then the number of kept tokens
// before it: (those above the key or forced) + min(equal ones before it, equal ones wanted), so
// one count per warp and one scan are enough and no order depends on timing.
//
// move_rows / move_rows_in_place: the kept rows, 16 bytes a lane.  In place, row i comes from
// row idx[i] >= i, so a block that owns a column slice of a (b, h) moves it front to back: a
// step's loads come before its stores, and stores reach only rows that later steps do not read.
// HBM bounds both: every kept row is read and written once.
#include <cooperative_groups.h>

#include "sc_common.cuh"

namespace cg = cooperative_groups;

namespace sc {
namespace {

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kMaxSegment = 49152;  // keys a block: 192 KiB of shared memory

struct SelectParams {
    const float* scores;
    int64_t s_b, s_h;
    const int32_t* cache_lens;
    int32_t* new_lens;
    int32_t* indices;  // [B, H, budget]
    int32_t B, H, S, budget, first, recent;
    int32_t segment;   // keys a block of the cluster
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

// Sum over the block of x, and the sum before this thread (exclusive).  Called by every thread.
__device__ __forceinline__ int block_scan(int x, int& total, int* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int v = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += y;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = v;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
        const int y = s_warp[w];
        if (w < warp) before += y;
        all += y;
    }
    total = all;
    return before + v - x;
}

__global__ void __launch_bounds__(kSelThreads) select_tokens(const __grid_constant__ SelectParams p) {
    extern __shared__ __align__(16) uint32_t s_keys[];
    __shared__ uint32_t s_hist[kBins];
    __shared__ int s_warp[kSelWarps];
    __shared__ int s_pick[2];    // digit, equal ones still wanted
    __shared__ int s_counts[2];  // this block's kept-for-sure and equal tokens
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank());
    const int ranks = static_cast<int>(cluster.num_blocks());
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
    const int base = rank * p.segment;
    const int f0 = max(base, lo) - base, f1 = min(base + p.segment, hi) - base;  // free, local
    const float* scores = p.scores + b * p.s_b + h * p.s_h + base;
    for (int i = f0 + threadIdx.x; i < f1; i += kSelThreads) s_keys[i] = order_key(scores[i]);

    int want = n_new - lo - (len - hi);  // free tokens that stay
    uint32_t key = 0;                    // the last kept key's bits found so far
    int shift = 32;
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10;
        const uint32_t above = shift == 32 ? 0u : key >> shift;
        const int top = shift;
        shift -= bits;
        const uint32_t digits = (1u << bits) - 1u;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kSelThreads) s_hist[i] = 0;
        __syncthreads();
        for (int i = f0 + threadIdx.x; i < f1; i += kSelThreads) {
            const uint32_t x = s_keys[i];
            if (top == 32 || (x >> top) == above) atomicAdd(&s_hist[(x >> shift) & digits], 1u);
        }
        cluster.sync();
        // Bins in descending order, four a thread, summed over the cluster.
        int mine[kBins / kSelThreads], sum = 0;
#pragma unroll
        for (int j = 0; j < kBins / kSelThreads; ++j) {
            const int bin = kBins - 1 - (threadIdx.x * (kBins / kSelThreads) + j);
            int n = 0;
            for (int r = 0; r < ranks; ++r)
                n += static_cast<int>(cluster.map_shared_rank(s_hist, r)[bin]);
            mine[j] = n;
            sum += n;
        }
        int total;
        int before = block_scan(sum, total, s_warp);
        if (want > 0 && before < want && before + sum >= want) {
#pragma unroll
            for (int j = 0; j < kBins / kSelThreads; ++j) {
                if (before < want && before + mine[j] >= want) {
                    s_pick[0] = kBins - 1 - (threadIdx.x * (kBins / kSelThreads) + j);
                    s_pick[1] = want - before;
                }
                before += mine[j];
            }
        }
        cluster.sync();  // also: nobody reads this histogram any more
        if (want > 0) {
            key |= static_cast<uint32_t>(s_pick[0]) << shift;
            want = s_pick[1];
        }
    }
    // Free tokens above `key` stay, and the first `want` equal to it (want = 0: none do).
    const int wanted = want;
    const bool none = n_new - lo - (len - hi) <= 0;

    // Each warp owns a run of the segment.
    const int s0 = base, s1 = min(base + p.segment, len);
    const int n_seg = max(0, s1 - s0);
    const int run = ((n_seg + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;
    const int w0 = warp * run, w1 = min(w0 + run, n_seg);
    auto kind = [&](int i) -> int {  // 0 goes, 1 stays, 2 equal
        const int t = base + i;
        if (t < lo || t >= hi) return 1;
        if (none) return 0;
        const uint32_t x = s_keys[i];
        return x > key ? 1 : x == key ? 2 : 0;
    };
    int stay = 0, equal = 0;
    for (int i = w0 + lane; i < w0 + run; i += 32) {
        const int k = i < w1 ? kind(i) : 0;
        stay += __popc(__ballot_sync(0xffffffffu, k == 1));
        equal += __popc(__ballot_sync(0xffffffffu, k == 2));
    }
    int total_stay, total_equal;
    const int stay_before = block_scan(lane == 0 ? stay : 0, total_stay, s_warp);
    const int equal_before = block_scan(lane == 0 ? equal : 0, total_equal, s_warp);
    if (threadIdx.x == 0) {
        s_counts[0] = total_stay;
        s_counts[1] = total_equal;
    }
    cluster.sync();
    int g = __shfl_sync(0xffffffffu, stay_before, 0), e = __shfl_sync(0xffffffffu, equal_before, 0);
    for (int r = 0; r < rank; ++r) {
        const int* c = cluster.map_shared_rank(s_counts, r);
        g += c[0];
        e += c[1];
    }
    for (int i = w0 + lane; i < w0 + run; i += 32) {
        const int k = i < w1 ? kind(i) : 0;
        const uint32_t bs = __ballot_sync(0xffffffffu, k == 1), be = __ballot_sync(0xffffffffu, k == 2);
        const uint32_t below = (1u << lane) - 1u;
        const int gb = g + __popc(bs & below), eb = e + __popc(be & below);
        if (k == 1 || (k == 2 && eb < wanted)) idx[gb + min(eb, wanted)] = base + i;
        g += __popc(bs);
        e += __popc(be);
    }
    cluster.sync();  // no block leaves while another reads its shared memory
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

cudaError_t allow_select() {
    static std::atomic<uint64_t> done{0};
    return allow_shared_memory(reinterpret_cast<const void*>(select_tokens), kMaxSegment * 4, done);
}

}  // namespace

cudaError_t preload_evict_kernels() {
    cudaError_t e = allow_select();
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
    if (cache_len > static_cast<int64_t>(kMaxSegment) * kMaxCluster)
        return set_error(SC_ERR_UNSUPPORTED, "caches of %lld tokens: at most %d", (long long)cache_len,
                         kMaxSegment * kMaxCluster);
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
    // A cluster where one block cannot hold the scores, or where there are few long rows.
    int ranks = 1;
    while (ranks < kMaxCluster && (cache_len > static_cast<int64_t>(ranks) * kMaxSegment ||
                                   (rows * ranks * 2 <= 148 && cache_len > static_cast<int64_t>(ranks) * 4096)))
        ranks *= 2;
    sp.segment = static_cast<int32_t>(((cache_len + ranks - 1) / ranks + 31) / 32 * 32);
    cudaError_t e = allow_select();
    if (e != cudaSuccess) return cuda_error(e, "eviction set-up");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * ranks));
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(sp.segment) * 4;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(ranks);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, select_tokens, sp);
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
        move_rows_in_place<<<dim3(2 * mp.slices + 1, static_cast<unsigned>(rows)), kMoveThreads, 0, st>>>(mp);
    } else {
        const int64_t pieces = budget * (mp.row16 ? mp.row16 : 1);
        const int64_t per = kMoveThreads * kMoveUnroll;
        move_rows<<<dim3(static_cast<unsigned>((pieces + per - 1) / per), static_cast<unsigned>(rows), 3),
                    kMoveThreads, 0, st>>>(mp);
    }
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_error(e, "eviction move launch");
    return ok();
}
