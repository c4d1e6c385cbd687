// sc_weights.cuh — one call of the attention weights, shared by its two kernels.
#pragma once

#include "sc_attention.cuh"

namespace sc {

struct WeightParams {
    const void* q;
    int64_t q_t, q_h;
    const void* k;
    int64_t k_b, k_t, k_h;
    const float* lse;  // [N, Hq]
    int64_t lse_t, lse_h;
    const float* scores;
    int64_t s_b, s_h;
    float* out;
    int64_t o_b, o_h;
    const int32_t* cache_lens;
    const int32_t* cu_q;
    int32_t N, B, Hq, Hkv, G, D, nq, S;
    int32_t causal;
    int32_t parts, chunk;  // blocks a (b, h), tokens a block
    int32_t row_room;      // queries that fit in shared memory (a multiple of 16)
    FastDiv div_G;
    float scale_log2;
    int32_t* status;
};

// The tensor-core kernel (sc_weights_tile.cu), where its tensor maps can say the layout; *taken
// tells.
cudaError_t launch_weight_tiles(const WeightParams& p, bool half, cudaStream_t s, bool* taken);
cudaError_t preload_weight_tile_kernels();

}  // namespace sc
