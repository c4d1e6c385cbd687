// sc_tile_waits.h — which products the softmax warps of attend_tiles wait for.  Plain C++, so that a
// model of the barriers can be run on the CPU with it.
#pragma once

#ifdef __CUDACC__
#define SC_HOST_DEVICE __host__ __device__
#else
#define SC_HOST_DEVICE
#endif

namespace sc {

// A wait names a phase of a barrier by its parity, so a warp may only wait for a phase when the one
// before it is over: with two open phases the answer would be that of the phase two before.  Phase
// i of o_full is over when the product of token tile i has reached the sums.  With two row tiles the
// scores of tile i follow the product of tile i - 1, so whoever has scores is at most one phase
// behind.  With one row tile they follow the product of tile i - 2, so before the last wait, for
// phase n_tiles - 1, phase n_tiles - 2 is waited for.  That is done before the last tile's weights
// are handed over (phase n_tiles - 1 cannot be over until every warp has): later the parity could
// be that of a phase that never ends.  Returns that phase, or -1: nothing to wait for.
SC_HOST_DEVICE constexpr int phase_before_weights(int n_q, int i, int n_tiles) {
    return n_q == 1 && i > 0 && i == n_tiles - 1 ? i - 1 : -1;
}

}  // namespace sc
