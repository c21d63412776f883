// Leaky states with input-dependent decay over packed sequences: what the forward and the backward kernels share.
#ifndef BPL_CSRC_STATE_SCAN_CUH_
#define BPL_CSRC_STATE_SCAN_CUH_

#include <initializer_list>
#include <type_traits>

#include "sequence.cuh"

namespace bpl {

// Distance in tokens of the states kept for the backward pass.
constexpr uint32_t SCAN_TILE_TOKENS = 16;
constexpr uint32_t SCAN_MAX_STATE = 128;

constexpr int NS = 4;              // states of a lane
constexpr int CARRIERS = 128;      // threads of a block that bring tiles in and out, beside the walking ones
constexpr uint32_t CREW = CARRIERS / 2;

// lanes of a channel: a power of two
inline uint32_t lanes_for(uint32_t state) {
    uint32_t lanes = 1;
    while (lanes * NS < state) lanes *= 2;
    return lanes;
}

// Bytes that a copy of rows can move at once: 16 or 4 where addresses, distances and counts allow it, else 0.
template<typename T>
inline uint32_t copy_bytes(std::initializer_list<const void *> rows, std::initializer_list<long long> strides, uint32_t count) {
    for (uint32_t bytes : {16u, 4u}) {
        const uint32_t e = bytes / sizeof(T);
        bool ok = count % e == 0;
        for (const void *r : rows) ok &= reinterpret_cast<uintptr_t>(r) % bytes == 0;
        for (long long s : strides) ok &= s % e == 0;
        if (ok) return bytes;
    }
    return 0;
}

// Rows [tb, tb + TILE) within [from, to) of what lies `stride` elements apart, `count` elements each, into shared memory, by one warp; `mode`: 16 or 4 bytes at a time,
// or (0) element by element.
template<uint32_t TILE, typename T, int ROW>
__device__ __forceinline__ void fetch(T (*to_rows)[ROW], const T *base, long long stride, uint32_t tb, uint32_t from, uint32_t to,
                                      uint32_t count, uint32_t mode) {
    const uint32_t lane = threadIdx.x % 32;
    auto rows = [&](auto per_copy, auto copy) {
        constexpr uint32_t E = decltype(per_copy)::value, PER_ROW = ROW / E > 0 ? ROW / E : 1, COPIES = TILE * PER_ROW;
        if constexpr (PER_ROW <= 32) {           // a lane always the same elements of a row
            constexpr uint32_t J = 32 / PER_ROW;
            const uint32_t j0 = lane / PER_ROW, e = lane % PER_ROW * E;
            const T *at = base + (tb + j0) * stride + e;
            if (e >= count || (J > TILE && j0 >= TILE)) return;
            static_assert(J > TILE || TILE % J == 0, "whole rounds");
            if (tb >= from && tb + TILE <= to) {
#pragma unroll
                for (uint32_t j = 0; j < TILE; j += J, at += J * stride) copy(&to_rows[j0 + j][e], at);
            } else {
#pragma unroll 1
                for (uint32_t j = 0; j < TILE; j += J, at += J * stride)
                    if (tb + j0 + j >= from && tb + j0 + j < to) copy(&to_rows[j0 + j][e], at);
            }
        } else {
#pragma unroll 4
            for (uint32_t i = lane; i < COPIES; i += 32) {
                const uint32_t j = i / PER_ROW, e = i % PER_ROW * E, t = tb + j;
                if (t >= from && t < to && e < count) copy(&to_rows[j][e], base + t * stride + e);
            }
        }
    };
    if (mode == 16) rows(std::integral_constant<uint32_t, 16 / sizeof(T)>(), [](T *a, const T *b) { copy_async<16>(a, b); });
    else if (mode == 4) rows(std::integral_constant<uint32_t, 4 / sizeof(T)>(), [](T *a, const T *b) { copy_async<4>(a, b); });
    else rows(std::integral_constant<uint32_t, 1>(), [](T *a, const T *b) { *a = *b; });
}

template<typename T>
__device__ __forceinline__ void load_states(const T *at, pair (&v)[NS / 2]) {         // (8 bytes at once)
    static_assert(sizeof(T) == 2, "two bytes");
    const uint2 raw = *reinterpret_cast<const uint2 *>(at);
    const T *e = reinterpret_cast<const T *>(&raw);
    v[0] = load_pair(e);
    v[1] = load_pair(e + 2);
}
__device__ __forceinline__ void load_states(const float *at, pair (&v)[NS / 2]) {
    const float4 f = *reinterpret_cast<const float4 *>(at);
    v[0] = make_pair(f.x, f.y);
    v[1] = make_pair(f.z, f.w);
}

// A state (or its derivative) that passes a whole chunk: v 2^exponent, the exponent a sum over the chunk's tokens.  What single tokens
// would make of it: nothing grows out of zero however large the growth, an infinite one stays infinite however far the decay goes, and
// where 2^exponent alone leaves the range the product need not (it is taken in two halves, each at most the largest power of two: 2^254
// turns every other number into infinity).
__device__ __forceinline__ float through_chunk(float v, float exponent) {
    const float factor = ex2(exponent);
    if (factor > 0.0f && factor < INFINITY && fabsf(v) < INFINITY) return v * factor;
    const float half = ex2(fminf(0.5f * exponent, 127.0f));
    return isinf(v) ? v : v * half * half;
}
__device__ __forceinline__ pair through_chunk(pair v, pair exponent) {
    const float2 a = split(v), e = split(exponent);
    return make_pair(through_chunk(a.x, e.x), through_chunk(a.y, e.y));
}

// One launch over `n_chunks` runs of `chunk` tokens (a multiple of the tile; the last may be shorter).  A block holds CPB
// channels of one group and one chunk.
template<typename T>
struct ScanArgs {
    const T *x, *delta, *z, *B, *C;
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
struct StateScanPlan {
    uint32_t lanes, chunk, n_chunks, tiles;
};

}  // namespace bpl

#endif  // BPL_CSRC_STATE_SCAN_CUH_
