// Leaky states with input-dependent decay over packed sequences: what the forward and the backward kernels share.
#ifndef BPL_CSRC_STATE_SCAN_CUH_
#define BPL_CSRC_STATE_SCAN_CUH_

#include "sequence.cuh"

namespace bpl {

// Distance in tokens of the states kept for the backward pass.
constexpr uint32_t SCAN_TILE_TOKENS = 16;
constexpr uint32_t SCAN_MAX_STATE = 128;

// One launch over `n_chunks` runs of `chunk` tokens (a multiple of the tile; the last may be shorter).  A block holds CPB
// channels of one group and one chunk.
template<typename T>
struct ScanArgs {
    const T *x, *delta, *z, *B, *C, *dy;
    const float *A, *D, *bias, *initial;
    T *y;
    float *last, *saved;
    float *chunk_state, *chunk_time;      // [n_chunks][channels][state], [n_chunks][channels]
    long long x_stride, delta_stride, z_stride, B_stride, B_group, C_stride, C_group;
    Sequences seq;
    uint32_t channels, per_group, tiles, state, chunk, n_chunks;
    uint32_t row_copy, state_copy;        // bytes of one copy of x, delta, z and of B, C
    bool softplus, y_pairs, state_aligned;
};

// How a target shares its work out: lanes per channel, chunks of tokens, blocks of a group's channels.
struct ScanPlan2 {
    uint32_t lanes, chunk, n_chunks, tiles;
};

}  // namespace bpl

#endif  // BPL_CSRC_STATE_SCAN_CUH_
