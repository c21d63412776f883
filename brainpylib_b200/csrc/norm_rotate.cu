// Queries and keys of a layer normed head by head and rotated by their positions, in one pass, and the gradient (no counterpart in
// brainpylib):
//
//     r = (mean x^2 + eps)^(-1/2);   n = r x w;   (a, b) -> (a cos - b sin, a sin + b cos),  angle = position * frequency
//     dz = dy turned back;   dw = sum dz r x;   dx = r (dz w - x r^2 mean(dz w x))
//
// Bound by memory.  A few neighbouring lanes hold a head of a token, each some pairs (a, b) as two runs of neighbouring elements, so
// that a pair never leaves its lane; sums over a head are shuffles.  Cosines and sines of a token are made once per block into
// shared memory: the angle in turns in twice 64 bits, its fraction in 32.  16,384 tokens of 40 heads of 128 in 16 bits, parts of a wider
// projection: 67 us, 5.0 TB/s; the gradient of 8192 tokens of 32 heads 49 us, 4.1 TB/s (elements of 16 bits each in a register of its own, which an
// array of them takes, 108 and 60: fewer blocks on an SM).
#include <initializer_list>
#include <type_traits>

#include "sequence.cuh"

namespace bpl {
namespace {

constexpr int ROTATE_THREADS = 256;
constexpr uint32_t MAX_SIZE = 256;              // elements of a head
constexpr uint32_t TABLE = 1024;                // cosines and sines of a block
constexpr uint32_t BLOCKS_PER_SM = 4;           // of the backward pass: blocks hold parts of the weights' gradients

// (two 16-byte words where they are more)
template<typename T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Vec {
    T v[V];
};

struct RotateHeads {
    const void *x, *dy;
    const void *weight;
    void *out;                   // forward: y, backward: dx
    long long row, head;         // of x; dy and out are dense
    uint32_t heads, per_head;    // per_head: 2^32 / heads, rounded up
    float *parts;                // [blocks][size]: the weight's gradient
};
struct RotateArgs {
    RotateHeads of[2];           // queries, keys
    const void *positions;
    const float *frequencies;
    uint32_t tokens, size, turned, per_block, tiles;     // turned: pairs that are rotated; per_block: tokens of a tile
    float eps, per_size;         // per_size: 1 / size
    bool wide_positions, wide_weights, weights_aligned;
};

// Where the elements of pair i of a head lie: the first at a, the second at b.  What is not rotated is paired all the same, with
// an angle of zero.
template<bool INTERLEAVED>
__device__ __forceinline__ void pair_at(const RotateArgs &p, uint32_t i, uint32_t &a, uint32_t &b) {
    if (INTERLEAVED) {
        a = 2 * i;
        b = a + 1;
    } else if (i < p.turned) {
        a = i;
        b = i + p.turned;
    } else {
        a = i + p.turned;
        b = a + p.size / 2 - p.turned;
    }
}

// V pairs of a lane: interleaved they are 2 V neighbouring elements, else two runs of V.  Elements of 16 bits are kept as the words they
// lie in (an array of them would take a register for each).
template<typename T, int V>
using Raw = std::conditional_t<sizeof(T) == 2 && V == 8, uint4, Vec<T, V>>;
template<typename T, int V>
__device__ __forceinline__ void elements(const Raw<T, V> &raw, float *to) {
    if constexpr (sizeof(T) == 2 && V == 8) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = split(load_pair(reinterpret_cast<const T *>(&w[k])));
            to[2 * k] = f.x;
            to[2 * k + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) to[k] = to_float(raw.v[k]);
    }
}
template<typename T, int V>
__device__ __forceinline__ Raw<T, V> raw_of(const float *from) {
    Raw<T, V> raw;
    if constexpr (sizeof(T) == 2 && V == 8) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) store_pair(reinterpret_cast<T *>(&w[k]), make_float2(from[2 * k], from[2 * k + 1]));
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) raw.v[k] = from_float<T>(from[k]);
    }
    return raw;
}
template<typename T, int V, bool INTERLEAVED>
struct Pairs {
    Raw<T, V> lo, hi;
    __device__ __forceinline__ void load(const T *at, uint32_t a, uint32_t b) {
        lo = *reinterpret_cast<const Raw<T, V> *>(at + a);
        hi = *reinterpret_cast<const Raw<T, V> *>(at + (INTERLEAVED ? a + V : b));
    }
    __device__ __forceinline__ void store(T *at, uint32_t a, uint32_t b) const {
        *reinterpret_cast<Raw<T, V> *>(at + a) = lo;
        *reinterpret_cast<Raw<T, V> *>(at + (INTERLEAVED ? a + V : b)) = hi;
    }
    __device__ __forceinline__ void floats(float (&a)[V], float (&b)[V]) const {
        float all[2 * V];
        elements<T, V>(lo, all);
        elements<T, V>(hi, all + V);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            a[k] = all[INTERLEAVED ? 2 * k : k];
            b[k] = all[INTERLEAVED ? 2 * k + 1 : V + k];
        }
    }
    __device__ __forceinline__ void set(const float (&a)[V], const float (&b)[V]) {
        float all[2 * V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            all[INTERLEAVED ? 2 * k : k] = a[k];
            all[INTERLEAVED ? 2 * k + 1 : V + k] = b[k];
        }
        lo = raw_of<T, V>(all);
        hi = raw_of<T, V>(all + V);
    }
};

template<int LANES>
__device__ __forceinline__ float over_lanes(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
    return v;
}

__device__ __forceinline__ double position_of(const RotateArgs &p, uint32_t t) {
    return p.wide_positions ? static_cast<double>(static_cast<const long long *>(p.positions)[t])
                            : static_cast<double>(static_cast<const int *>(p.positions)[t]);
}

// The angle position * frequency in turns, without whole ones: at most half a turn.  Its product with 1 / (2 pi) in twice 64 bits, so
// that positions up to 2^53 leave 32 bits of the fraction (64 bits alone: 2^-53 of the angle, all 32 of them from 2^28 turns on).
__device__ __forceinline__ float turns_of(double position, double frequency) {
    constexpr double PER_TURN = 0.15915494309189535, PER_TURN_REST = -9.839338337591243e-18;
    const double angle = position * frequency, angle_rest = fma(position, frequency, -angle);
    const double turns = angle * PER_TURN;
    const double rest = fma(angle, PER_TURN, -turns) + fma(angle, PER_TURN_REST, angle_rest * PER_TURN);
    const double part = (turns - rint(turns)) + rest;          // (the rest may be whole turns itself, of angles beyond 2^53)
    return static_cast<float>(part - rint(part));
}

// A block takes tiles of `per_block` tokens, in turn; LANES lanes a head, ITER groups of V pairs a lane.
template<typename T, int V, int LANES, int ITER, bool INTERLEAVED, bool BACKWARD>
__global__ __launch_bounds__(ROTATE_THREADS, BACKWARD ? 2 : 3) void norm_rotate_kernel(const RotateArgs p) {
    constexpr uint32_t GROUPS = ROTATE_THREADS / LANES;
    constexpr int AHEAD = 1;                         // heads of a round (two: 86 us against 68 for 16,384 tokens of 40 heads of 128)
    constexpr uint32_t PAIRS = LANES * ITER * V, FOUR = V < 4 ? V : 4;
    static_assert(TABLE % PAIRS == 0, "whole tokens");
    // of the pairs of a token: four neighbouring ones of every lane next to those of the next lane, so that lanes reach all banks
    __shared__ alignas(16) float cosines[TABLE], sines[TABLE];
    auto place = [](uint32_t i) { return i / (LANES * V) * (LANES * V) + i % V / FOUR * (LANES * FOUR) + i % (LANES * V) / V * FOUR + i % FOUR; };
    __shared__ float sums[BACKWARD ? ROTATE_THREADS / 32 : 1][BACKWARD ? MAX_SIZE : 1];
    const uint32_t part = threadIdx.x % LANES, group = threadIdx.x / LANES, pairs = p.size / 2;
    uint32_t a[ITER], b[ITER], first[ITER];
    bool there[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        first[i] = (i * LANES + part) * V;
        there[i] = first[i] < pairs;
        pair_at<INTERLEAVED>(p, there[i] ? first[i] : 0u, a[i], b[i]);
    }
    float dw[2][ITER][2][V] = {};                    // (backward) of queries' and keys' weights
    for (uint32_t tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
        const uint32_t t0 = tile * p.per_block, n = min(p.per_block, p.tokens - t0);
        if (tile != blockIdx.x) __syncthreads();
        for (uint32_t i = threadIdx.x; i < n * p.turned; i += ROTATE_THREADS) {
            const uint32_t t = i / p.turned, f = i % p.turned;
            float s, c;
            sincospif(2.0f * turns_of(position_of(p, t0 + t), static_cast<double>(p.frequencies[f])), &s, &c);
            cosines[t * PAIRS + place(f)] = c;
            sines[t * PAIRS + place(f)] = BACKWARD ? -s : s;
        }
        __syncthreads();
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const RotateHeads &h = p.of[which];
            float wa[ITER][V], wb[ITER][V];
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                if (h.weight != nullptr && there[i] && p.wide_weights && V % 4 == 0 && p.weights_aligned) {
                    Pairs<float, V, INTERLEAVED> w;
                    w.load(static_cast<const float *>(h.weight), a[i], b[i]);
                    w.floats(wa[i], wb[i]);
                } else if (h.weight != nullptr && there[i] && !p.wide_weights && V > 1 && p.weights_aligned) {
                    Pairs<T, V, INTERLEAVED> w;
                    w.load(static_cast<const T *>(h.weight), a[i], b[i]);
                    w.floats(wa[i], wb[i]);
                } else {
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        wa[i][k] = wb[i][k] = 1.0f;
                        if (h.weight != nullptr && there[i]) {
                            const uint32_t ia = INTERLEAVED ? a[i] + 2 * k : a[i] + k, ib = INTERLEAVED ? ia + 1 : b[i] + k;
                            wa[i][k] = p.wide_weights ? static_cast<const float *>(h.weight)[ia] : to_float(static_cast<const T *>(h.weight)[ia]);
                            wb[i][k] = p.wide_weights ? static_cast<const float *>(h.weight)[ib] : to_float(static_cast<const T *>(h.weight)[ib]);
                        }
                    }
                }
            }
            const uint32_t rows = n * h.heads;
            // (all lanes of a warp go through the same rounds: sums over lanes are shuffles of the whole warp; the heads of the next round
            // are on their way while those of this one are worked on)
            Pairs<T, V, INTERLEAVED> x[AHEAD][ITER], dy[AHEAD][ITER], x_next[AHEAD][ITER], dy_next[AHEAD][ITER];
            auto request = [&](uint32_t base) {
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    const uint32_t row = base + j * GROUPS + group;
                    if (row >= rows) continue;
                    const uint32_t token = h.heads > 1 ? __umulhi(row, h.per_head) : row, head = row - token * h.heads;
                    const T *at = static_cast<const T *>(h.x) + (t0 + token) * h.row + head * h.head;
#pragma unroll
                    for (int i = 0; i < ITER; ++i)
                        if (there[i]) {
                            x_next[j][i].load(at, a[i], b[i]);
                            if (BACKWARD)
                                dy_next[j][i].load(static_cast<const T *>(h.dy) + (static_cast<size_t>(t0) * h.heads + row) * p.size, a[i], b[i]);
                        }
                }
            };
            request(0);
            for (uint32_t base = 0; base < rows; base += AHEAD * GROUPS) {
                uint32_t token[AHEAD], row[AHEAD];
                bool mine[AHEAD];
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    row[j] = base + j * GROUPS + group;
                    mine[j] = row[j] < rows;
                    token[j] = mine[j] ? (h.heads > 1 ? __umulhi(row[j], h.per_head) : row[j]) : 0u;
#pragma unroll
                    for (int i = 0; i < ITER; ++i) {
                        x[j][i] = x_next[j][i];
                        if (BACKWARD) dy[j][i] = dy_next[j][i];
                    }
                }
                request(base + AHEAD * GROUPS);
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    float xa[ITER][V], xb[ITER][V], square = 0.0f;
#pragma unroll
                    for (int i = 0; i < ITER; ++i) {
                        if (mine[j] && there[i]) {
                            x[j][i].floats(xa[i], xb[i]);
#pragma unroll
                            for (int k = 0; k < V; ++k) square += xa[i][k] * xa[i][k] + xb[i][k] * xb[i][k];
                        }
                    }
                    const float r = rsqrtf(fmaf(over_lanes<LANES>(square), p.per_size, p.eps));
                    T *to = static_cast<T *>(h.out) + (static_cast<size_t>(t0) * h.heads + row[j]) * p.size;
                    float za[ITER][V], zb[ITER][V], dot = 0.0f;
#pragma unroll
                    for (int i = 0; i < ITER; ++i) {
                        if (!mine[j] || !there[i]) continue;
                        if (BACKWARD) {
                            dy[j][i].floats(za[i], zb[i]);
                        } else {
#pragma unroll
                            for (int k = 0; k < V; ++k) {
                                za[i][k] = xa[i][k] * r * wa[i][k];
                                zb[i][k] = xb[i][k] * r * wb[i][k];
                            }
                        }
                        if (first[i] < p.turned) {
                            const uint32_t from = token[j] * PAIRS + i * (LANES * V) + part * FOUR;
#pragma unroll
                            for (int q = 0; q < V; q += FOUR) {
                                const Vec<float, FOUR> c = *reinterpret_cast<const Vec<float, FOUR> *>(cosines + from + q / FOUR * (LANES * FOUR));
                                const Vec<float, FOUR> d = *reinterpret_cast<const Vec<float, FOUR> *>(sines + from + q / FOUR * (LANES * FOUR));
#pragma unroll
                                for (int e = 0; e < FOUR; ++e) {
                                    if (INTERLEAVED && first[i] + q + e >= p.turned) continue;      // (else whole lanes)
                                    const float ta = za[i][q + e] * c.v[e] - zb[i][q + e] * d.v[e];
                                    zb[i][q + e] = za[i][q + e] * d.v[e] + zb[i][q + e] * c.v[e];
                                    za[i][q + e] = ta;
                                }
                            }
                        }
#pragma unroll
                        for (int k = 0; k < V; ++k) {
                            if (BACKWARD) {
                                const float na = xa[i][k] * r, nb = xb[i][k] * r;       // normed
                                dw[which][i][0][k] += za[i][k] * na;
                                dw[which][i][1][k] += zb[i][k] * nb;
                                za[i][k] *= wa[i][k];
                                zb[i][k] *= wb[i][k];
                                dot += za[i][k] * na + zb[i][k] * nb;
                                xa[i][k] = na;
                                xb[i][k] = nb;
                            }
                        }
                    }
                    if (BACKWARD) {
                        const float mean = over_lanes<LANES>(dot) * p.per_size;
#pragma unroll
                        for (int i = 0; i < ITER; ++i) {
                            if (!mine[j] || !there[i]) continue;
#pragma unroll
                            for (int k = 0; k < V; ++k) {
                                za[i][k] = r * (za[i][k] - xa[i][k] * mean);
                                zb[i][k] = r * (zb[i][k] - xb[i][k] * mean);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < ITER; ++i)
                        if (mine[j] && there[i]) {
                            Pairs<T, V, INTERLEAVED> y;
                            y.set(za[i], zb[i]);
                            y.store(to, a[i], b[i]);
                        }
                }
            }
        }
    }
    if constexpr (BACKWARD) {
        // the block's parts of the weights' gradients: lanes of a warp that hold the same pairs, then the warps, in order
        const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            if (p.of[which].weight == nullptr) continue;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ITER; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        float v = dw[which][i][half][k];
#pragma unroll
                        for (int o = LANES; o < 32; o <<= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
                        if (lane < LANES && there[i]) {
                            const uint32_t at = INTERLEAVED ? a[i] + 2 * k + half : (half ? b[i] : a[i]) + k;
                            sums[warp][at] = v;
                        }
                    }
            __syncthreads();
            for (uint32_t e = threadIdx.x; e < p.size; e += ROTATE_THREADS) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < ROTATE_THREADS / 32; ++w) v += sums[w][e];
                p.of[which].parts[static_cast<size_t>(blockIdx.x) * p.size + e] = v;
            }
        }
    }
}

// The parts of all blocks added up, in 64 bits: 32 columns to a block, warp w the blocks w, w + 8, ... of the first kernel, then the warps
// in order.
template<typename T>
__global__ __launch_bounds__(256) void rotate_sum_kernel(const float *q_parts, const float *k_parts, void *dq_weight, void *dk_weight, uint32_t size,
                                                         uint32_t blocks, bool wide) {
    __shared__ double sums[8][32];
    pdl_wait();
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, e = blockIdx.x * 32 + lane;
    const float *parts = blockIdx.y == 0 ? q_parts : k_parts;
    void *out = blockIdx.y == 0 ? dq_weight : dk_weight;
    if (out == nullptr) return;
    double sum = 0.0;
    if (e < size) {
#pragma unroll 8
        for (uint32_t b = warp; b < blocks; b += 8) sum += static_cast<double>(__ldcg(parts + static_cast<size_t>(b) * size + e));
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || e >= size) return;
    for (int w = 1; w < 8; ++w) sum += sums[w][lane];
    if (wide) static_cast<float *>(out)[e] = static_cast<float>(sum);
    else static_cast<T *>(out)[e] = from_float<T>(static_cast<float>(sum));
}

// ---- launches ------------------------------------------------------------------------------------------------------------
const bpl_norm_rotate_descriptor *checked(const char *opaque, size_t opaque_len, const char *what) {
    const auto *d = unpack<bpl_norm_rotate_descriptor>(opaque, opaque_len);
    if (d == nullptr) return nullptr;
    if (d->dtype > BPL_BFLOAT16 || (d->weight_dtype != d->dtype && d->weight_dtype != BPL_FLOAT) || d->size < 2 || d->size > MAX_SIZE ||
        d->size % 2 != 0 || d->rotated > d->size || d->rotated % 2 != 0 || d->tokens >= (1u << 31) || d->q_heads > 65535 ||
        d->k_heads > 65535) {
        set_status(BPL_ERR_ARGUMENT, what);
        return nullptr;
    }
    return d;
}

bool given(void **b, std::initializer_list<int> which, const char *what) {
    for (int i : which)
        if (b[i] == nullptr) {
            set_status(BPL_ERR_ARGUMENT, what);
            return false;
        }
    return true;
}

// Tokens of a tile: eight, which the table has room for, so that weights and angles are made for some heads at once; fewer where SMs
// would be idle.  (Rows of a tile stay below 2^16 heads, and so do products of their number with that of heads below 2^32: see `per_head`.)
uint32_t tile_tokens(const bpl_norm_rotate_descriptor &d) {
    const uint32_t heads = d.q_heads > d.k_heads ? d.q_heads : d.k_heads;
    uint32_t n = 8;
    while (n > 1 && n * heads > 65535) n /= 2;
    const uint32_t spread = d.tokens / (4 * static_cast<uint32_t>(sm_count()));
    if (n > spread) n = spread;
    return n < 1 ? 1 : n;
}
uint32_t backward_blocks(const bpl_norm_rotate_descriptor &d) {
    const uint32_t n = tile_tokens(d), tiles = (d.tokens + n - 1) / n, most = BLOCKS_PER_SM * static_cast<uint32_t>(sm_count());
    return tiles < most ? tiles : most;
}

template<typename T, int V, int LANES, int ITER>
void launch(cudaStream_t stream, const RotateArgs &p, bool interleaved, bool backward, uint32_t blocks) {
    if (backward) {
        if (interleaved) norm_rotate_kernel<T, V, LANES, ITER, true, true><<<blocks, ROTATE_THREADS, 0, stream>>>(p);
        else norm_rotate_kernel<T, V, LANES, ITER, false, true><<<blocks, ROTATE_THREADS, 0, stream>>>(p);
    } else {
        if (interleaved) norm_rotate_kernel<T, V, LANES, ITER, true, false><<<blocks, ROTATE_THREADS, 0, stream>>>(p);
        else norm_rotate_kernel<T, V, LANES, ITER, false, false><<<blocks, ROTATE_THREADS, 0, stream>>>(p);
    }
}

// Whether V pairs of a lane can be moved at once: runs begin at multiples of V elements of 16 bytes in all operands.
bool aligned(const RotateArgs &p, const bpl_norm_rotate_descriptor &d, uint32_t v, bool backward) {
    const uint32_t pairs = p.size / 2;
    bool ok = pairs % v == 0 && (p.turned % v == 0 || (d.flags & BPL_ROTATE_INTERLEAVED) != 0) && p.size % v == 0;
    for (const RotateHeads &h : p.of)
        ok &= h.row % v == 0 && (h.heads < 2 || h.head % v == 0) && aligned16(h.x) && aligned16(h.out) && (!backward || aligned16(h.dy));
    return ok;
}

template<typename T>
void run(cudaStream_t stream, RotateArgs p, const bpl_norm_rotate_descriptor &d, bool backward) {
    constexpr int V = 16 / sizeof(T);
    const bool interleaved = (d.flags & BPL_ROTATE_INTERLEAVED) != 0;
    p.per_block = tile_tokens(d);
    p.tiles = (d.tokens + p.per_block - 1) / p.per_block;
    const uint32_t blocks = backward ? backward_blocks(d) : p.tiles, pairs = p.size / 2;
    if (aligned(p, d, V, backward)) {
        const uint32_t lanes = pairs / V;
        if (lanes <= 8) return launch<T, V, 8, 1>(stream, p, interleaved, backward, blocks);
        if (lanes <= 16) return launch<T, V, 16, 1>(stream, p, interleaved, backward, blocks);
        if constexpr (V == 4) return launch<T, V, 32, 1>(stream, p, interleaved, backward, blocks);
    }
    if (pairs <= 32) return launch<T, 1, 32, 1>(stream, p, interleaved, backward, blocks);
    if (pairs <= 64) return launch<T, 1, 32, 2>(stream, p, interleaved, backward, blocks);
    launch<T, 1, 32, 4>(stream, p, interleaved, backward, blocks);
}

void norm_rotate_any(cudaStream_t stream, const RotateArgs &p, const bpl_norm_rotate_descriptor &d, bool backward) {
    if (d.dtype == BPL_FLOAT) run<float>(stream, p, d, backward);
    else if (d.dtype == BPL_HALF) run<__half>(stream, p, d, backward);
    else run<__nv_bfloat16>(stream, p, d, backward);
}

uint32_t per_head(uint32_t heads) { return heads > 1 ? static_cast<uint32_t>(((1ull << 32) + heads - 1) / heads) : 0; }

// what both passes read: buffers 0 to 5
RotateArgs arguments(void **b, const bpl_norm_rotate_descriptor &d) {
    RotateArgs p = {};
    p.of[0] = RotateHeads{b[0], nullptr, b[4], nullptr, d.q_stride, d.q_head_stride, d.q_heads, per_head(d.q_heads), nullptr};
    p.of[1] = RotateHeads{b[1], nullptr, b[5], nullptr, d.k_stride, d.k_head_stride, d.k_heads, per_head(d.k_heads), nullptr};
    p.positions = b[2];
    p.frequencies = static_cast<const float *>(b[3]);
    p.tokens = d.tokens; p.size = d.size; p.turned = d.rotated / 2; p.eps = d.eps;
    p.per_size = 1.0f / static_cast<float>(d.size);
    p.wide_positions = (d.flags & BPL_ROTATE_WIDE_POSITIONS) != 0;
    p.wide_weights = d.weight_dtype == BPL_FLOAT;
    p.weights_aligned = aligned16(b[4]) && aligned16(b[5]);
    return p;
}

}  // namespace

size_t norm_rotate_backward_workspace_bytes(const char *opaque, size_t opaque_len) {
    if (opaque == nullptr || opaque_len != sizeof(bpl_norm_rotate_descriptor)) return 0;
    const auto &d = *reinterpret_cast<const bpl_norm_rotate_descriptor *>(opaque);
    return d.size > MAX_SIZE ? 0 : sizeof(float) * 2 * static_cast<size_t>(backward_blocks(d)) * d.size;
}

}  // namespace bpl

using namespace bpl;

extern "C" {

void norm_rotate(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "norm_rotate: heads of 2 to 256 elements, an even number, fewer than 2^31 tokens");
    if (d == nullptr || d->tokens == 0 || d->q_heads + d->k_heads == 0) return;
    if ((d->q_heads > 0 && !given(buffers, {0, 6}, "norm_rotate: null buffer")) ||
        (d->k_heads > 0 && !given(buffers, {1, 7}, "norm_rotate: null buffer")) || !given(buffers, {2}, "norm_rotate: null buffer") ||
        (d->rotated > 0 && !given(buffers, {3}, "norm_rotate: null buffer")))
        return;
    RotateArgs p = arguments(buffers, *d);
    p.of[0].out = buffers[6];
    p.of[1].out = buffers[7];
    norm_rotate_any(stream, p, *d, false);
    launch_ok();
}

void norm_rotate_backward(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "norm_rotate_backward: heads of 2 to 256 elements, an even number, fewer than 2^31 tokens");
    if (d == nullptr) return;
    const bool weights = buffers[4] != nullptr || buffers[5] != nullptr, rows = d->tokens > 0 && d->q_heads + d->k_heads > 0;
    if ((buffers[4] != nullptr && !given(buffers, {10}, "norm_rotate_backward: null buffer")) ||
        (buffers[5] != nullptr && !given(buffers, {11}, "norm_rotate_backward: null buffer")))
        return;
    if (rows && ((d->q_heads > 0 && !given(buffers, {0, 6, 8}, "norm_rotate_backward: null buffer")) ||
                 (d->k_heads > 0 && !given(buffers, {1, 7, 9}, "norm_rotate_backward: null buffer")) ||
                 !given(buffers, {2}, "norm_rotate_backward: null buffer") ||
                 (d->rotated > 0 && !given(buffers, {3}, "norm_rotate_backward: null buffer")) ||
                 (weights && !given(buffers, {12}, "norm_rotate_backward: null buffer"))))
        return;
    RotateArgs p = arguments(buffers, *d);
    const uint32_t blocks = rows ? backward_blocks(*d) : 0;
    for (int i = 0; i < 2; ++i) {
        p.of[i].dy = buffers[6 + i];
        p.of[i].out = buffers[8 + i];
        p.of[i].parts = static_cast<float *>(buffers[12]) + (buffers[12] ? static_cast<size_t>(i) * blocks * d->size : 0);
    }
    if (rows) norm_rotate_any(stream, p, *d, true);
    if (weights) {
        const dim3 grid((d->size + 31) / 32, 2);
        const bool wide = d->weight_dtype == BPL_FLOAT;
        if (d->dtype == BPL_HALF)
            launch_dependent(rotate_sum_kernel<__half>, grid, dim3(256), 0, stream, p.of[0].parts, p.of[1].parts, buffers[4] ? buffers[10] : nullptr,
                             buffers[5] ? buffers[11] : nullptr, d->size, blocks, wide);
        else
            launch_dependent(rotate_sum_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, p.of[0].parts, p.of[1].parts,
                             buffers[4] ? buffers[10] : nullptr, buffers[5] ? buffers[11] : nullptr, d->size, blocks, wide);
    }
    launch_ok();
}

}  // extern "C"
