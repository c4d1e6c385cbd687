// sc_attention.cuh — shared by the attention kernels: what a call holds, and the warp-level
// matrix, copy and exponential instructions they use.
#pragma once

#include "sc_common.cuh"

namespace sc {

// One call of the shared-prefix attention.  Tokens of q are packed over the sequences; rows of
// one KV head are (token, head of its group) pairs, token-major.  Strides count elements.
struct AttnParams {
    const void* q;
    int64_t q_t, q_h;
    const void* kp;  // prefix keys and values [P, Hkv, D]
    const void* vp;
    int64_t kp_t, kp_h, vp_t, vp_h;
    const void* kc;  // own caches [B, cap, Hkv, D], or a pool [n_pages, page, Hkv, D]
    const void* vc;
    int64_t kc_b, kc_t, kc_h, vc_b, vc_t, vc_h;
    const int32_t* page_table;  // null: dense caches
    int64_t pt_b;
    int64_t n_pages;
    const int32_t* cache_lens;  // null: every cache is full
    const int32_t* cu_q;        // [B + 1] first token of each sequence; null: nq each
    int32_t N, B, Hq, Hkv, G, D;
    int32_t nq;       // tokens a sequence, at most
    int32_t P, cap;   // prefix tokens; own cache tokens a sequence, at most
    int32_t page;     // tokens a page (dense: cap)
    FastDiv div_G, div_page;
    float scale_log2;  // scale * log2(e)
    int32_t n_pp, n_cp;  // parts of the prefix and of each own cache
    int32_t chunk_p;     // prefix tokens a part
    int32_t tiles_p, tiles_c;  // row tiles of the prefix, and at most of a sequence
    float* part_o;   // [n_pp + n_cp][N * Hq][D], not normalised
    float2* part_ml; // [n_pp + n_cp][N * Hq]: row maximum (log2 units) and sum
    void* out;
    int64_t o_t, o_h;
    float* lse;  // [N, Hq], or null
    int32_t* status;
};

constexpr float kNegInf = -__builtin_huge_valf();

// Where sequences begin in q.  A sequence whose starts decrease, leave the range of the first and the last
// one or are more than nq apart has no tokens (`of` is false), and its rows of the output are left alone.
struct Starts {
    const int32_t* cu;  // [B + 1], or null: nq each
    int first, last;    // tokens that sequences may have
    int nq;
    __device__ __forceinline__ Starts(const int32_t* cu_q, int B, int N, int most)
        : cu(cu_q), first(0), last(N), nq(most) {
        if (cu_q != nullptr) {
            first = max(cu_q[0], 0);
            last = max(min(cu_q[B], N), 0);
        }
    }
    __device__ __forceinline__ explicit Starts(const AttnParams& p) : Starts(p.cu_q, p.B, p.N, p.nq) {}
    __device__ __forceinline__ bool of(int b, int& tok0, int& n) const {
        tok0 = b * nq;
        n = nq;
        if (cu == nullptr) return true;
        const int a = cu[b], e = cu[b + 1];
        const bool fine = a >= first && e >= a && e <= last && e - a <= nq;
        tok0 = fine ? a : 0;
        n = fine ? e - a : 0;
        return fine;
    }
};
__device__ __forceinline__ int used_tokens(const AttnParams& p) { return Starts(p).last; }
__device__ __forceinline__ void sequence_tokens(const AttnParams& p, const Starts& starts, int b, int& tok0, int& n) {
    if (!starts.of(b, tok0, n) && threadIdx.x == 0 && p.status) atomicOr(p.status, SC_STATUS_BAD_SEQ_LEN);
}

// What is wrong with any sequence that device starts give, by one warp.  (Out of line, like in_sequence:
// few calls need it, and what lies between a kernel's instructions costs their fetches.)
static __device__ __noinline__ void report_sequences(const int32_t* cu_q, int B, int N, int nq, const int32_t* cache_lens,
                                                     int cap, int32_t* status) {
    const Starts starts(cu_q, B, N, nq);
    for (int b = threadIdx.x & 31; b < B; b += 32) {
        int tok0, n;
        bool fine = starts.of(b, tok0, n);
        if (cache_lens != nullptr) fine = fine && cache_lens[b] >= 0 && cache_lens[b] <= cap;
        if (!fine) atomicOr(status, SC_STATUS_BAD_SEQ_LEN);
    }
}

// Whether a token is some sequence's, for a whole warp.  Between starts that do not decrease a search
// finds its sequence; where that one is not fine, the others are asked in turn.
static __device__ __noinline__ bool in_sequence(const int32_t* cu_q, int B, int N, int nq, int tok) {
    const Starts starts(cu_q, B, N, nq);
    if (tok < starts.first || tok >= starts.last) return false;
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = B;  // cu_q[lo] <= tok < cu_q[hi]
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, i = lo + (lane + 1) * step;
        const uint32_t upto = __ballot_sync(0xffffffffu, i < hi && cu_q[i] <= tok);
        const int k = 32 - __clz(upto);  // the last of them, if any
        hi = min(hi, lo + (k + 1) * step);
        lo += k * step;
    }
    int tok0, n;
    if (starts.of(lo, tok0, n)) return true;
    for (int b0 = 0; b0 < B; b0 += 32) {
        const bool in = b0 + lane < B && starts.of(b0 + lane, tok0, n) && tok >= tok0 && tok < tok0 + n;
        if (__any_sync(0xffffffffu, in)) return true;
    }
    return false;
}

__device__ __forceinline__ int cache_length(const AttnParams& p, int b) {
    if (p.cache_lens == nullptr) return p.cap;
    const int len = p.cache_lens[b];
    if (len < 0 || len > p.cap) {
        if (threadIdx.x == 0 && p.status) atomicOr(p.status, SC_STATUS_BAD_SEQ_LEN);
        return 0;
    }
    return len;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes global -> shared; zeros instead when !valid (the source is then not read).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// c[16 x 8] += a[16 x 16] b[16 x 8], fp32 accumulation.
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value) {
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// An 8 x 8 matrix of 16-bit values, two a lane, transposed.
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(bit_cast_u32<__half2>(w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// ---- weights as 16-bit pieces ----
// Where memory bounds a kernel, a weight x >= 0 goes into its product with V as hi + lo, 2^-16 (bfloat16)
// or 2^-20 (float16) of x off.  hi is x rounded down and lo the rest plus 2^-12 x, so that lo is above
// zero wherever x is: an infinite value times either piece is that infinity, and their sum too (with a lo
// of zero or below it would be NaN).  float16 begins at 2^-24, so its weights are lifted: 2^16 for the
// largest, of which hi is float16's largest number and lo the rest.  A part's sums of weights (kUnlift) and of values (kUnlift, and the 2^-12 taken back) go out
// without either, so that its lse keeps its bits.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 16.f : 0.f;
template <typename T>
constexpr float kUnlift = std::is_same<T, __half>::value ? 0x1p-16f : 1.f;
template <typename T>
constexpr float kOnePiece = kUnlift<T> / (1.f + 0x1p-12f);
// What weights are taken from for a maximum m: it less the lift, or m itself where it is so large that the
// difference rounds to more.  (A lift of 2^k is exact up to maxima of 2^(24 + k).)
template <typename T>
__device__ __forceinline__ float lifted(float m, float lift) {
    if constexpr (!std::is_same<T, __half>::value) return m;
    const float base = m - lift;
    return m - base <= lift + 0.5f ? base : m;
}
template <typename T>
__device__ __forceinline__ void two_pieces(float x, float y, uint32_t& hi, uint32_t& lo) {
    float2 r;
    if constexpr (std::is_same<T, __half>::value) {
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
        r = unpack2<T>(hi);
    } else {
        const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
        hi = __byte_perm(a, b, 0x7632);
        r = make_float2(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u));
    }
    lo = pack2<T>(fmaf(x, 1.f + 0x1p-12f, -r.x), fmaf(y, 1.f + 0x1p-12f, -r.y));
}

// The tensor-core kernel (sc_attention_tile.cu), over the prefix for all rows together in `splits`
// parts, or (per_seq) over the prefix and then each sequence's own cache for the sequence's rows,
// output included: rounds of `sms` units, the last one's split into up to `splits` parts.
// chained: another kernel of the call is before it on the stream.
cudaError_t launch_attention_tiles(const AttnParams& a, bool half, bool per_seq, int tiles, int splits,
                                   int sms, int64_t units, bool chained, cudaStream_t s);
cudaError_t preload_attention_tile_kernels();

// The streaming kernel (sc_attention_stream.cu): few rows, parts of runs of 64-token steps, at least
// `least` of them; dp: head_dim padded to 64, 128 or 256; mt: 16-row tiles (0: one of 8 rows).  make_stream_maps is
// false where tensor maps cannot say the layout.
struct StreamMaps {
    alignas(64) unsigned char map[4][128];
    int box;
};
bool make_stream_maps(const AttnParams& a, bool half, bool with_prefix, StreamMaps* m);
cudaError_t launch_attention_stream(const AttnParams& a, const StreamMaps& m, bool half, bool with_prefix, int dp,
                                    int mt, int least, int blocks, bool chained, cudaStream_t s);
cudaError_t preload_attention_stream_kernels();

// ---- values that are not finite ----
// A token that some rows of a tile do not see has weight zero there, and 0 x infinity would be NaN.  So
// where a tile holds such tokens, values that are not finite leave the product: zeros take their
// place, the first token with +infinity and with -infinity (NaN: both) is kept for each column, and
// the rows that see it get them at the end.
constexpr int kNoToken = 0x7fffffff;
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}
// Two values with those that are not finite (all exponent bits set) made zero.
template <typename T>
__device__ __forceinline__ uint32_t finite_part(uint32_t v) {
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    if ((v & e) == e) v &= 0xffff0000u;
    if ((v >> 16 & e) == e) v &= 0xffffu;
    return v;
}
template <typename T>
__device__ __forceinline__ uint4 finite_part(uint4 v) {
    return make_uint4(finite_part<T>(v.x), finite_part<T>(v.y), finite_part<T>(v.z), finite_part<T>(v.w));
}
// One chunk (8 columns) of a token's values in shared memory; first: those columns of kNoToken-filled
// [2][columns].  Out of line: what it costs where nothing is odd is a load and a few comparisons.
template <typename T>
__device__ __noinline__ void take_out_odd(uint32_t at, int token, int* first, int columns, int* any) {
    const uint4 v = ld_shared_v4(at), f = finite_part<T>(v);
    if (f.x == v.x && f.y == v.y && f.z == v.z && f.w == v.w) return;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float2 x2 = unpack2<T>(w[e / 2]);
        const float x = e & 1 ? x2.y : x2.x;
        if (isfinite(x)) continue;
        if (!(x < 0.f)) atomicMin(first + e, token);
        if (!(x > 0.f)) atomicMin(first + columns + e, token);
    }
    st_shared_v4(at, f);
    *any = 1;
}
// Row of sums `o` that sees the tokens below `limit`.
static __device__ __noinline__ void add_odd(float* o, int n, const int* first, int columns, int limit) {
    for (int c = 0; c < n; ++c) {
        if (first[c] < limit) o[c] += -kNegInf;
        if (first[columns + c] < limit) o[c] += kNegInf;
    }
}

}  // namespace sc
