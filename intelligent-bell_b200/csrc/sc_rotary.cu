// sc_rotary.cu — rotary positions of new queries and keys: every (token, head) row of q and of
// k turned by its token's position, in one launch, in the half or the interleaved layout, over
// the whole head or its first rotary_dim elements.
//
// Mathematics.  For frequency i of a token at position p, with a = p * f_i and a factor m:
//   (y1, y2) = m (x1 cos a - x2 sin a, x2 cos a + x1 sin a)
// The pair (x1, x2) is (x[i], x[i + R/2]) in the half layout and (x[2i], x[2i + 1]) in the
// interleaved one; elements from R = rotary_dim on are passed through.  The inverse turns by
// -a and divides by m.
//
// Angles.  p * f_i in fp32 is off by up to 2^-24 p f_i radians, 0.03 at p = 10^6, so the angle
// is kept as a fraction of a turn in 64-bit fixed point: the host gives F_i = f_i / (2 pi) *
// 2^64 and the product p * F_i modulo 2^64 IS the fraction (whole turns fall off the top),
// exact but for F_i, which has a double's 53 bits (f_i <= 1: 2^-55 of a turn off, 2^-24 at p = 2^31).
// It goes as a signed fp32 number in [-1, 1) of half turns, 2^-25 of one off, to sincospif, which
// then needs no range reduction.
//
// What bounds it: HBM (two 16-bit values read and written for 3 multiplications).  A block
// loads the slices of its rows first, then tabulates its tokens' cosines and sines in shared
// memory while they are in flight (64 per token at R = 128, used by every head of q and k), then
// turns and stores.  32 + 8 heads of 128 for 8,192 tokens: 36.5 us, a plain copy of the same bytes
// 32.7.  Blocks of 128 threads with two items each in flight (one 36.9, four 36.8 us; blocks of 512
// threads 51.6).
#include <math.h>

#include "sc_common.cuh"

namespace sc {
namespace {

constexpr int kRThreads = 128;
constexpr int kMaxRotary = 512;       // frequencies travel as kernel parameters
constexpr int kMaxTokensPerBlock = 32;
constexpr int kTableEntries = 2048;   // float2 entries of the block's table

struct RotaryTensor {
    const void* x;
    void* out;
    int64_t x_b, x_t, x_h, x_d;
    int64_t o_b, o_t, o_h, o_d;
};

struct RotaryParams {
    RotaryTensor q, k;
    int32_t B, T, Hq, H;   // H = Hq + Hk rows a token
    int32_t D, R;          // head and rotary size
    int32_t interleaved;
    int32_t slices, items; // slices a row (turned, then passed through); items = H * slices
    int32_t turned;        // how many of a row's slices are turned
    int32_t tokens;        // tokens a block
    int32_t chunk;         // items of one token in one block (blockIdx.y picks which)
    FastDiv div_chunk, div_slices, div_T;
    const void* pos;
    int32_t pos_is_64;
    int64_t pos_b, pos_t;
    int64_t pos_start;
    float mult;            // of the cosine
    float mult_sin;        // of the sine (negative: inverse)
    uint64_t freq[kMaxRotary / 2];
};

__device__ __forceinline__ int64_t position(const RotaryParams& p, int32_t b, int32_t t) {
    if (p.pos == nullptr) return p.pos_start + t;
    const int64_t at = b * p.pos_b + t * p.pos_t;
    return p.pos_is_64 ? static_cast<const int64_t*>(p.pos)[at]
                       : static_cast<int64_t>(static_cast<const int32_t*>(p.pos)[at]);
}

__device__ __forceinline__ float2 turn_of(const RotaryParams& p, int64_t pos, int i) {
    const int64_t frac = static_cast<int64_t>(static_cast<uint64_t>(pos) * p.freq[i]);
    float s, c;
    sincospif(static_cast<float>(frac) * 0x1p-63f, &s, &c);
    return make_float2(c * p.mult, s * p.mult_sin);
}

template <typename T>
__device__ __forceinline__ float load1(const T* p) {
    return static_cast<float>(*p);
}

// N 32-bit words (N = 8, 4 or 2: one 32-, 16- or 8-byte access).  Plain loads: the rotation may
// run in place.
template <int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[N]) {
    if constexpr (N == 8) {
        asm volatile("ld.global.v8.u32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                       "=r"(w[6]), "=r"(w[7])
                     : "l"(p));
    } else if constexpr (N == 4) {
        const uint4 v = *static_cast<const uint4*>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
        const uint2 v = *static_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    }
}
template <int N>
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[N]) {
    if constexpr (N == 8)
        st_v8(p, w);
    else if constexpr (N == 4)
        st_v4(p, make_uint4(w[0], w[1], w[2], w[3]));
    else
        st_v2(p, make_uint2(w[0], w[1]));
}

// The words of a vector as floats and back.
template <typename T, int N, int F>
__device__ __forceinline__ void widen(const uint32_t (&w)[N], float (&x)[F]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(bit_cast_u32<__half2>(w[i]));
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}
template <typename T, int N, int F>
__device__ __forceinline__ void narrow(const float (&x)[F], uint32_t (&w)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
    }
}

// A slice: F frequencies of one row, as two vectors of VB = F * sizeof(T) bytes (the halves'
// parts in the half layout, two adjacent vectors in the interleaved one), or 2F elements behind
// the rotary part, which are copied.  Each thread has up to two slices, loaded before the table
// is made.
template <typename T, int VB>
__global__ void __launch_bounds__(kRThreads) rotary_vec(const __grid_constant__ RotaryParams p) {
    constexpr int F = VB / sizeof(T);
    constexpr int N = VB / 4;
    constexpr int kRounds = 2;
    __shared__ __align__(16) float2 s_cs[kTableEntries];
    const int half = p.R >> 1;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tokens;
    const int64_t all = static_cast<int64_t>(p.B) * p.T;
    const int n_tok = static_cast<int>(min(static_cast<int64_t>(p.tokens), all - first));
    const int base = blockIdx.y * p.chunk;
    const int n_items = min(p.chunk, p.items - base);

    uint32_t a[kRounds][N], b[kRounds][N];
    char* dst[kRounds];
    int second[kRounds], local[kRounds], slice[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        dst[r] = nullptr;
        const uint32_t idx = threadIdx.x + r * kRThreads;
        const int tok = static_cast<int>(fdiv(idx, p.div_chunk));
        const int item = base + static_cast<int>(idx) - tok * p.chunk;
        if (tok >= n_tok || item >= base + n_items) continue;
        const int row = static_cast<int>(fdiv(static_cast<uint32_t>(item), p.div_slices));
        const int sl = item - row * p.slices;
        const uint32_t tg = static_cast<uint32_t>(first + tok);
        const int bb = static_cast<int>(fdiv(tg, p.div_T));
        const int64_t t = static_cast<int64_t>(tg) - static_cast<int64_t>(bb) * p.T;
        const bool is_q = row < p.Hq;
        const RotaryTensor& x = is_q ? p.q : p.k;
        const int h = is_q ? row : row - p.Hq;
        const bool turn = sl < p.turned;
        const int e0 = !turn ? p.R + (sl - p.turned) * 2 * F : p.interleaved ? sl * 2 * F : sl * F;
        const int gap = turn && !p.interleaved ? half : F;
        const T* src = static_cast<const T*>(x.x) + bb * x.x_b + t * x.x_t + h * x.x_h + e0;
        load_words<N>(src, a[r]);
        load_words<N>(src + gap, b[r]);
        dst[r] = reinterpret_cast<char*>(static_cast<T*>(x.out) + bb * x.o_b + t * x.o_t +
                                         h * x.o_h + e0);
        second[r] = gap;
        local[r] = tok * half;
        slice[r] = turn ? sl * F : -1;
    }
    for (int e = threadIdx.x; e < n_tok * half; e += kRThreads) {
        const int tok = e / half, i = e - tok * half;
        const uint32_t tg = static_cast<uint32_t>(first + tok);
        const int bb = static_cast<int>(fdiv(tg, p.div_T));
        s_cs[e] = turn_of(p, position(p, bb, static_cast<int>(tg) - bb * p.T), i);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        if (dst[r] == nullptr) continue;
        if (slice[r] >= 0) {
            float x[F], y[F];
            widen<T, N, F>(a[r], x);
            widen<T, N, F>(b[r], y);
            const float2* cs = s_cs + local[r] + slice[r];
            if (p.interleaved) {
                // x and y are 2F consecutive elements: pairs lie side by side
#pragma unroll
                for (int i = 0; i < F; i += 2) {
                    const float2 u = cs[i / 2], v = cs[F / 2 + i / 2];
                    const float x1 = x[i], x2 = x[i + 1], y1 = y[i], y2 = y[i + 1];
                    x[i] = x1 * u.x - x2 * u.y;
                    x[i + 1] = x2 * u.x + x1 * u.y;
                    y[i] = y1 * v.x - y2 * v.y;
                    y[i + 1] = y2 * v.x + y1 * v.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < F; ++i) {
                    const float2 u = cs[i];
                    const float x1 = x[i], x2 = y[i];
                    x[i] = x1 * u.x - x2 * u.y;
                    y[i] = x2 * u.x + x1 * u.y;
                }
            }
            narrow<T, N, F>(x, a[r]);
            narrow<T, N, F>(y, b[r]);
        }
        store_words<N>(dst[r], a[r]);
        store_words<N>(dst[r] + static_cast<int64_t>(second[r]) * sizeof(T), b[r]);
    }
}

// Any strides and sizes: a thread turns one pair, or copies one or two elements behind the
// rotary part.
template <typename T>
__global__ void __launch_bounds__(kRThreads) rotary_any(const __grid_constant__ RotaryParams p) {
    const int pairs = (p.D + 1) >> 1;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * kRThreads + threadIdx.x;
    const int64_t rows = static_cast<int64_t>(p.B) * p.T * p.H;
    if (w >= rows * pairs) return;
    const int64_t row = w / pairs;
    const int i = static_cast<int>(w - row * pairs);
    const int64_t tg = row / p.H;
    const int hh = static_cast<int>(row - tg * p.H);
    const int bb = static_cast<int>(tg / p.T);
    const int64_t t = tg - static_cast<int64_t>(bb) * p.T;
    const RotaryTensor& x = hh < p.Hq ? p.q : p.k;
    const int h = hh < p.Hq ? hh : hh - p.Hq;
    const T* src = static_cast<const T*>(x.x) + bb * x.x_b + t * x.x_t + h * x.x_h;
    T* dst = static_cast<T*>(x.out) + bb * x.o_b + t * x.o_t + h * x.o_h;
    const int half = p.R >> 1;
    if (i >= half) {
        for (int e = 2 * i; e < min(2 * i + 2, p.D); ++e) dst[e * x.o_d] = src[e * x.x_d];
        return;
    }
    const int e1 = p.interleaved ? 2 * i : i, e2 = p.interleaved ? 2 * i + 1 : i + half;
    const float2 u = turn_of(p, position(p, bb, static_cast<int32_t>(t)), i);
    const float x1 = load1(src + e1 * x.x_d), x2 = load1(src + e2 * x.x_d);
    const float y1 = x1 * u.x - x2 * u.y, y2 = x2 * u.x + x1 * u.y;
    if constexpr (sizeof(T) == 4) {
        dst[e1 * x.o_d] = y1;
        dst[e2 * x.o_d] = y2;
    } else {
        dst[e1 * x.o_d] = from_float<T>(y1);
        dst[e2 * x.o_d] = from_float<T>(y2);
    }
}

template <typename T>
cudaError_t launch_rotary(const RotaryParams& p, int vb, dim3 grid, cudaStream_t s) {
    if (vb == 32)
        rotary_vec<T, 32><<<grid, kRThreads, 0, s>>>(p);
    else if (vb == 16)
        rotary_vec<T, 16><<<grid, kRThreads, 0, s>>>(p);
    else if (vb == 8)
        rotary_vec<T, 8><<<grid, kRThreads, 0, s>>>(p);
    else
        rotary_any<T><<<grid, kRThreads, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t preload_rotary_type() {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, rotary_vec<T, 32>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, rotary_vec<T, 16>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, rotary_vec<T, 8>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, rotary_any<T>);
    return e;
}

}  // namespace

cudaError_t preload_rotary_kernels() {
    cudaError_t e = preload_rotary_type<__half>();
    if (e == cudaSuccess) e = preload_rotary_type<__nv_bfloat16>();
    if (e == cudaSuccess) e = preload_rotary_type<float>();
    return e;
}

}  // namespace sc

using namespace sc;

extern "C" int32_t sc_rope_apply(int32_t batch, int64_t n_tokens, int32_t q_heads, int32_t k_heads,
                                 int32_t head_dim, int32_t rotary_dim, int32_t interleaved,
                                 const void* q, const int64_t* q_strides, const void* k,
                                 const int64_t* k_strides, int32_t dtype, const void* positions,
                                 int32_t positions_are_64, const int64_t* pos_strides,
                                 int64_t pos_start, const double* inv_freq, double factor,
                                 int32_t inverse, void* q_out, const int64_t* qo_strides,
                                 void* k_out, const int64_t* ko_strides, void* stream) {
    if (batch < 0 || n_tokens < 0 || q_heads < 0 || k_heads < 0 || head_dim < 0)
        return set_error(SC_ERR_INVALID_ARGUMENT, "negative size");
    if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
        return set_error(SC_ERR_INVALID_ARGUMENT,
                         "rotary_dim must be even and at most head_dim %d, got %d", head_dim,
                         rotary_dim);
    if (head_dim > kMaxHeadDim || rotary_dim > kMaxRotary)
        return set_error(SC_ERR_UNSUPPORTED, "head_dim %d (at most %d) or rotary_dim %d (at most %d)",
                         head_dim, kMaxHeadDim, rotary_dim, kMaxRotary);
    if (dtype != SC_DTYPE_F16 && dtype != SC_DTYPE_BF16 && dtype != SC_DTYPE_F32)
        return set_error(SC_ERR_INVALID_DTYPE, "dtype code %d: float16, bfloat16 or float32", dtype);
    if (!(factor > 0.0) || !isfinite(factor))
        return set_error(SC_ERR_INVALID_ARGUMENT, "factor must be positive and finite, got %g", factor);
    const int32_t kh = k ? k_heads : 0;
    const int64_t rows = size_product(batch, n_tokens, static_cast<int64_t>(q_heads) + kh);
    if (size_product(rows, (head_dim + 1) / 2) >= (int64_t(1) << 31) * kRThreads ||
        rows >= (int64_t(1) << 31) || size_product(static_cast<int64_t>(q_heads) + kh, head_dim) >= (int64_t(1) << 24))
        return set_error(SC_ERR_INVALID_ARGUMENT, "%lld rows in one call; split it", (long long)rows);
    if (rows == 0 || head_dim == 0) return ok();
    if ((q_heads && (!q || !q_out || !q_strides || !qo_strides)) ||
        (kh && (!k_out || !k_strides || !ko_strides)) || (rotary_dim && !inv_freq) ||
        (positions && !pos_strides))
        return set_error(SC_ERR_INVALID_ARGUMENT, "null pointer argument");

    RotaryParams p{};
    auto fill = [](RotaryTensor& t, const void* x, const int64_t* xs, void* o, const int64_t* os) {
        t.x = x, t.out = o;
        t.x_b = xs[0], t.x_t = xs[1], t.x_h = xs[2], t.x_d = xs[3];
        t.o_b = os[0], t.o_t = os[1], t.o_h = os[2], t.o_d = os[3];
    };
    if (q_heads) fill(p.q, q, q_strides, q_out, qo_strides);
    if (kh) fill(p.k, k, k_strides, k_out, ko_strides);
    p.B = batch, p.T = static_cast<int32_t>(n_tokens), p.Hq = q_heads, p.H = q_heads + kh;
    p.D = head_dim, p.R = rotary_dim, p.interleaved = interleaved != 0;
    p.pos = positions, p.pos_is_64 = positions_are_64, p.pos_start = pos_start;
    if (positions) p.pos_b = pos_strides[0], p.pos_t = pos_strides[1];
    p.mult = static_cast<float>(inverse ? 1.0 / factor : factor);
    p.mult_sin = inverse ? -p.mult : p.mult;
    for (int i = 0; i < rotary_dim / 2; ++i) {
        // The fraction of a turn a step makes, modulo 1, in units of 2^-64.
        const double turns = inv_freq[i] * 0.15915494309189533576888376337251436;  // 1 / (2 pi)
        if (!isfinite(turns) || fabs(turns) > 0x1p40)
            return set_error(SC_ERR_INVALID_ARGUMENT, "frequency %d is %g", i, inv_freq[i]);
        const double frac = turns - floor(turns);  // in [0, 1)
        const double scaled = frac * 0x1p64;
        p.freq[i] = scaled >= 0x1p64 ? 0 : static_cast<uint64_t>(scaled);
    }

    const int64_t esize = dtype == SC_DTYPE_F32 ? 4 : 2;
    const int half = rotary_dim / 2;
    auto fits = [&](int vb) {
        const int f = static_cast<int>(vb / esize);
        if (half % f != 0 || (head_dim - rotary_dim) % (2 * f) != 0) return false;
        auto one = [&](const RotaryTensor& t, int heads) {
            if (heads == 0) return true;
            auto al = [&](const void* a) { return reinterpret_cast<uintptr_t>(a) % vb == 0; };
            auto st = [&](int64_t s, int64_t n) { return n <= 1 || s % f == 0; };
            return t.x_d == 1 && t.o_d == 1 && al(t.x) && al(t.out) && st(t.x_b, batch) &&
                   st(t.x_t, n_tokens) && st(t.x_h, heads) && st(t.o_b, batch) &&
                   st(t.o_t, n_tokens) && st(t.o_h, heads);
        };
        return one(p.q, q_heads) && one(p.k, kh);
    };
    const int vb = fits(32) ? 32 : fits(16) ? 16 : fits(8) ? 8 : 0;
    p.div_T = make_fastdiv(static_cast<uint32_t>(p.T));
    dim3 grid;
    if (vb) {
        const int f = static_cast<int>(vb / esize);
        p.turned = half / f;
        p.slices = p.turned + (head_dim - rotary_dim) / (2 * f);
        p.div_slices = make_fastdiv(static_cast<uint32_t>(p.slices));
        p.items = p.H * p.slices;
        const int room = 2 * kRThreads;
        const int parts = (p.items + room - 1) / room;
        p.chunk = (p.items + parts - 1) / parts;
        p.div_chunk = make_fastdiv(static_cast<uint32_t>(p.chunk));
        int tokens = room / p.chunk;
        if (tokens > kMaxTokensPerBlock) tokens = kMaxTokensPerBlock;
        if (half && tokens > kTableEntries / half) tokens = kTableEntries / half;
        const int64_t all = static_cast<int64_t>(batch) * n_tokens;
        // few tokens: over as many SMs as there are
        if (tokens > (all + 147) / 148) tokens = static_cast<int>((all + 147) / 148);
        p.tokens = tokens < 1 ? 1 : tokens;
        grid = dim3(static_cast<unsigned>((all + p.tokens - 1) / p.tokens), parts);
    } else {
        const int64_t work = rows * ((head_dim + 1) / 2);
        grid = dim3(static_cast<unsigned>((work + kRThreads - 1) / kRThreads));
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == SC_DTYPE_F16    ? launch_rotary<__half>(p, vb, grid, s)
                          : dtype == SC_DTYPE_BF16 ? launch_rotary<__nv_bfloat16>(p, vb, grid, s)
                                                   : launch_rotary<float>(p, vb, grid, s);
    if (e != cudaSuccess) return cuda_error(e, "rotary launch");
    return ok();
}
