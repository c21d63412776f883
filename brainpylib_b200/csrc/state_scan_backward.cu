// The gradient of state_scan.  With dY = dy silu(z) (dy without a gate) and a[t] = exp(dt A):
//
//     q[t] = C[t] dY[t] + a[t + 1] q[t + 1]          the derivative by h[t], from the last token to the first
//     dC = sum over channels of dY h;  dB = sum over channels of q dt x;  dx = D dY + dt sum_n q B
//     d(dt) = x sum_n q B + sum_n q a h[t - 1] A;  dA = sum over tokens of q a h[t - 1] dt
//
// A block walks its tokens tile by tile from the last to the first.  The states of a tile are computed once more from the one
// that the forward pass kept in front of it; they and the decays stay in registers for the way back.  Sums over channels are
// left as one part per block and token, sums over tokens as one part per chunk, and added up in a fixed order by a last kernel:
// the same call gives the same bits.
#include <initializer_list>

#include "state_scan.cuh"

namespace bpl {
namespace {

constexpr int BACK_THREADS = 128;
constexpr int BACK_WARPS = BACK_THREADS / 32;
constexpr uint32_t TILE = SCAN_TILE_TOKENS;

template<typename T>
struct BackArgs {
    const T *x, *delta, *z, *B, *C, *dy;
    const float *A, *D, *bias, *initial, *saved, *d_last;
    T *dx, *d_delta, *d_z;
    float *d_initial;
    float *part_BC;                    // [tiles][tokens][groups][2][state]
    float *part_A, *part_D, *part_bias;   // [n_chunks][channels](state)
    float *chunk_state, *chunk_time;
    long long x_stride, delta_stride, z_stride, B_stride, B_group, C_stride, C_group;
    Sequences seq;
    uint32_t channels, groups, per_group, tiles, state, chunk, n_chunks;
    bool softplus;
};

// Sums V values over the CW channels of a warp (lanes LANES apart); a lane is left with V / min(V, CW) of the sums, from
// value (channel % min(V, CW)) * (V / min(V, CW)) on, in v[0 ..].
template<int V, int CW, int LANES>
__device__ __forceinline__ void sum_over_channels(float (&v)[V], const int channel) {
    constexpr int K = V < CW ? V : CW;
#pragma unroll
    for (int half = V / 2, bit = K / 2; bit > 0; half /= 2, bit /= 2) {
        const bool upper = (channel & bit) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float give = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor_sync(FULL_MASK, give, bit * LANES);
        }
    }
#pragma unroll
    for (int bit = K; bit < CW; bit *= 2) {
#pragma unroll
        for (int i = 0; i < V / K; ++i) v[i] += __shfl_xor_sync(FULL_MASK, v[i], bit * LANES);
    }
}

template<int NS, int LANES>
struct BackShared {
    static constexpr int CPB = BACK_THREADS / LANES, NP = NS * LANES, Y_ROW = CPB + 32 / LANES;
    float dt[TILE][CPB][2];
    float dY[TILE][CPB];
    float B[TILE][NP], C[TILE][NP];
    float sums[3][TILE][Y_ROW];
    float part[BACK_WARPS][TILE][2][NP];
};

// ENDS: only what a chunk hands to the one in front of it when nothing comes from behind, and the time that passes in it.
template<typename T, int NS, int LANES, bool ENDS>
__global__ void __launch_bounds__(BACK_THREADS)
state_scan_backward_kernel(const BackArgs<T> p) {
    using Shared = BackShared<NS, LANES>;
    constexpr int CPB = Shared::CPB, NP = Shared::NP, PAIRS = NS / 2, CW = 32 / LANES, V = 2 * NS;
    constexpr int K = LANES < static_cast<int>(TILE) ? LANES : static_cast<int>(TILE), KV = V < CW ? V : CW;
    extern __shared__ __align__(16) unsigned char raw_shared[];
    Shared &sh = *reinterpret_cast<Shared *>(raw_shared);

    const uint32_t tid = threadIdx.x, warp = tid / 32, local = tid / LANES, part = tid % LANES;
    const uint32_t group = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles, k_chunk = blockIdx.y;
    const uint32_t c_first = tile * CPB, c_count = min(static_cast<uint32_t>(CPB), p.per_group - c_first);
    const uint32_t c0 = group * p.per_group + c_first, channel = c0 + local;
    const bool valid = local < c_count;
    const uint32_t n0 = part * NS;
    const Sequences seq = p.seq;
    const uint32_t first = seq.first(), last = seq.last();

    const uint32_t from = k_chunk * p.chunk;
    uint32_t to = min(from + p.chunk, seq.tokens);
    if (ENDS) {                       // only where the sequence at the chunk's first token began before it
        if (k_chunk == 0 || from >= last || from <= first) return;
        const uint32_t s = seq.of(from);
        if (seq.begin(s) >= from) return;
        to = min(to, max(seq.end(s), from));
    }
    const uint32_t live_from = max(from, first), live_to = min(to, last);

    pair A2[PAIRS], g[PAIRS], dA[PAIRS];
#pragma unroll
    for (int k = 0; k < PAIRS; ++k) {
        float a[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t n = n0 + 2 * k + i;
            a[i] = valid && n < p.state ? p.A[static_cast<size_t>(channel) * p.state + n] * LOG2_E : 0.0f;
        }
        A2[k] = make_pair(a[0], a[1]);
        g[k] = 0;
        dA[k] = 0;
    }
    float time = 0.0f, d_D = 0.0f, d_bias = 0.0f;

    auto load_state = [&](pair (&to_pairs)[PAIRS], const float *at) {
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
            float v[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) v[i] = valid && n0 + 2 * k + i < p.state ? __ldcg(at + n0 + 2 * k + i) : 0.0f;
            to_pairs[k] = make_pair(v[0], v[1]);
        }
    };
    auto store_state = [&](const pair (&pairs)[PAIRS], float *at) {
        if (!valid) return;
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
            const float2 v = split(pairs[k]);
            if (n0 + 2 * k < p.state) at[n0 + 2 * k] = v.x;
            if (n0 + 2 * k + 1 < p.state) at[n0 + 2 * k + 1] = v.y;
        }
    };
    auto state_of = [&](uint32_t row) { return (static_cast<size_t>(row) * p.channels + channel) * p.state; };
    auto load_or_zero = [&](pair (&to_pairs)[PAIRS], const float *base, uint32_t row) {
        if (base != nullptr) {
            load_state(to_pairs, base + state_of(row));
        } else {
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) to_pairs[k] = 0;
        }
    };

    // what reaches the chunk's last token from the chunks behind it
    uint32_t next_begin = 0xffffffffu;         // where the sequence of the token behind the tile begins
    if (live_from < live_to && live_to == to && to < last && !ENDS) {
        const uint32_t s = seq.of(to);
        next_begin = seq.begin(s);
        if (next_begin < to) {
            const uint32_t s_end = max(seq.end(s), to + 1);
            for (uint32_t j = min((s_end - 1) / p.chunk, p.n_chunks - 1); j > k_chunk; --j) {
                const float passed = valid ? __ldcg(p.chunk_time + static_cast<size_t>(j) * p.channels + channel) : 0.0f;
                const pair dt = make_pair(passed, passed);
                pair own[PAIRS];
                load_state(own, p.chunk_state + state_of(j));
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) g[k] = fma2(g[k], ex2_pair(mul2(dt, A2[k])), own[k]);
            }
        }
    }

    const uint32_t n_tiles = to > from ? (to - from + TILE - 1) / TILE : 0;
    for (uint32_t i_tile = n_tiles; i_tile-- > 0;) {
        const uint32_t tb = from + i_tile * TILE;
        // ---- stage
        for (uint32_t i = tid; i < TILE * CPB; i += BACK_THREADS) {
            const uint32_t j = i / CPB, c = i % CPB, t = tb + j;
            float dt = 0.0f, in = 0.0f, dY = 0.0f;
            if (c < c_count && t >= live_from && t < live_to) {
                dt = to_float(p.delta[t * p.delta_stride + c0 + c]) + (p.bias ? p.bias[c0 + c] : 0.0f);
                if (p.softplus) dt = softplus(dt);
                if (!ENDS) in = dt * to_float(p.x[t * p.x_stride + c0 + c]);
                dY = to_float(p.dy[static_cast<size_t>(t) * p.channels + c0 + c]);
                if (p.z != nullptr) dY *= silu(to_float(p.z[t * p.z_stride + c0 + c]));
            }
            sh.dt[j][c][0] = dt;
            sh.dt[j][c][1] = in;
            sh.dY[j][c] = dY;
        }
        for (uint32_t i = tid; i < TILE * NP; i += BACK_THREADS) {
            const uint32_t j = i / NP, n = i % NP, t = tb + j;
            const bool use = n < p.state && t >= live_from && t < live_to;
            if (!ENDS) sh.B[j][n] = use ? to_float(p.B[t * p.B_stride + group * p.B_group + n]) : 0.0f;
            sh.C[j][n] = use ? to_float(p.C[t * p.C_stride + group * p.C_group + n]) : 0.0f;
        }
        // bit j: token tb + j is the first, the last of its sequence
        uint32_t starts = 0, ends = 0;
        if (next_begin >= tb || tb < live_from || tb + TILE > live_to) {
            const uint32_t t = tb + tid % TILE;
            bool start = false, end = false;
            if (t >= live_from && t < live_to) {
                const uint32_t s = seq.of(t);
                start = seq.begin(s) == t;
                end = seq.end(s) == t + 1;
            }
            starts = __ballot_sync(FULL_MASK, start) & 0xffffu;
            ends = __ballot_sync(FULL_MASK, end) & 0xffffu;
            next_begin = tb >= live_from && tb < live_to ? seq.begin(seq.of(tb)) : 0xffffffffu;
        }
        __syncthreads();

        if (ENDS) {
            float passed = 0.0f;
#pragma unroll
            for (int j = TILE - 1; j >= 0; --j) {
                const float dtj = sh.dt[j][local][0], dY = sh.dY[j][local];
                const pair dt = make_pair(dtj, dtj), dy = make_pair(dY, dY);
                if (ends >> j & 1) load_or_zero(g, p.d_last, seq.of(tb + j));
                passed += dtj;
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) {
                    const pair c = *reinterpret_cast<const pair *>(&sh.C[j][n0 + 2 * k]);
                    g[k] = mul2(fma2(c, dy, g[k]), decay_pair(dt, A2[k]));
                }
            }
            time += passed;
            __syncthreads();
            continue;
        }

        // ---- forwards through the tile: states and decays into registers
        pair before[PAIRS], h[TILE][PAIRS], keep[TILE][PAIRS];
        load_state(before, p.saved + state_of(tb / TILE));
#pragma unroll
        for (int j0 = 0; j0 < static_cast<int>(TILE); j0 += K) {
            float y[K];
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const int j = j0 + i;
                pair prev[PAIRS];
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) prev[k] = j ? h[j ? j - 1 : 0][k] : before[k];
                if (starts >> j & 1) load_or_zero(prev, p.initial, seq.of(tb + j));
                const float2 d = *reinterpret_cast<const float2 *>(sh.dt[j][local]);
                const pair dt = make_pair(d.x, d.x), in = make_pair(d.y, d.y);
                pair sum = 0;
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) {
                    const pair b = *reinterpret_cast<const pair *>(&sh.B[j][n0 + 2 * k]);
                    const pair c = *reinterpret_cast<const pair *>(&sh.C[j][n0 + 2 * k]);
                    keep[j][k] = decay_pair(dt, A2[k]);
                    h[j][k] = fma2(prev[k], keep[j][k], mul2(in, b));
                    sum = k == 0 ? mul2(h[j][k], c) : fma2(h[j][k], c, sum);
                }
                y[i] = sum2(sum);
            }
            const float sum = sum_over_lanes<K, LANES>(y, part);
            if (part < K) sh.sums[0][j0 + part][local] = sum;
        }
        // ---- and back
        pair dA_tile[PAIRS];
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) dA_tile[k] = 0;
#pragma unroll
        for (int j0 = static_cast<int>(TILE) - K; j0 >= 0; j0 -= K) {
            float qB[K], wA[K];
#pragma unroll
            for (int i = K - 1; i >= 0; --i) {
                const int j = j0 + i;
                const float2 d = *reinterpret_cast<const float2 *>(sh.dt[j][local]);
                const float dYj = sh.dY[j][local];
                const pair dt = make_pair(d.x, d.x), in = make_pair(d.y, d.y), dy = make_pair(dYj, dYj);
                if (ends >> j & 1) load_or_zero(g, p.d_last, seq.of(tb + j));
                pair prev[PAIRS];
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) prev[k] = j ? h[j ? j - 1 : 0][k] : before[k];
                if (starts >> j & 1) load_or_zero(prev, p.initial, seq.of(tb + j));
                pair sum_qB = 0, sum_wA = 0;
                float v[V];
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) {
                    const pair b = *reinterpret_cast<const pair *>(&sh.B[j][n0 + 2 * k]);
                    const pair c = *reinterpret_cast<const pair *>(&sh.C[j][n0 + 2 * k]);
                    const pair q = fma2(c, dy, g[k]);
                    const float2 to_B = split(mul2(q, in)), to_C = split(mul2(dy, h[j][k]));
                    v[2 * k] = to_B.x;
                    v[2 * k + 1] = to_B.y;
                    v[NS + 2 * k] = to_C.x;
                    v[NS + 2 * k + 1] = to_C.y;
                    sum_qB = k == 0 ? mul2(q, b) : fma2(q, b, sum_qB);
                    g[k] = mul2(q, keep[j][k]);
                    const pair w = mul2(g[k], prev[k]);
                    sum_wA = k == 0 ? mul2(w, A2[k]) : fma2(w, A2[k], sum_wA);
                    dA_tile[k] = fma2(w, dt, dA_tile[k]);
                }
                qB[i] = sum2(sum_qB);
                wA[i] = sum2(sum_wA);
                if (starts >> j & 1) {
                    if (p.d_initial != nullptr) store_state(g, p.d_initial + state_of(seq.of(tb + j)));
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) g[k] = 0;
                }
                const int cw = (tid % 32) / LANES;
                sum_over_channels<V, CW, LANES>(v, cw);
                if (cw < KV) {
                    constexpr int R = V / KV;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const int at = cw * R + r;             // 0 .. NS - 1: of B, NS .. 2 NS - 1: of C
                        sh.part[warp][j][at / NS][n0 + at % NS] = v[r];
                    }
                }
            }
            const float sum_b = sum_over_lanes<K, LANES>(qB, part), sum_a = sum_over_lanes<K, LANES>(wA, part);
            if (part < K) {
                sh.sums[1][j0 + part][local] = sum_b;
                sh.sums[2][j0 + part][local] = sum_a;
            }
        }
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) dA[k] = add2(dA[k], dA_tile[k]);
        __syncthreads();

        // ---- per token and channel
        for (uint32_t i = tid; i < TILE * CPB; i += BACK_THREADS) {
            const uint32_t j = i / CPB, c = i % CPB, t = tb + j;
            if (c >= c_count || t >= to) continue;
            const size_t at = static_cast<size_t>(t) * p.channels + c0 + c;
            float dx = 0.0f, dd = 0.0f, dz = 0.0f;
            if (t >= live_from && t < live_to) {
                const float x = to_float(p.x[t * p.x_stride + c0 + c]), dY = sh.dY[j][c], dt = sh.dt[j][c][0];
                const float D = p.D ? p.D[c0 + c] : 0.0f, qB = sh.sums[1][j][c];
                dx = fmaf(dt, qB, D * dY);
                dd = fmaf(x, qB, sh.sums[2][j][c] * LN_2);
                if (p.softplus) dd *= sigmoid(to_float(p.delta[t * p.delta_stride + c0 + c]) + (p.bias ? p.bias[c0 + c] : 0.0f));
                d_D = fmaf(dY, x, d_D);
                d_bias += dd;
                if (p.z != nullptr) {
                    const float z = to_float(p.z[t * p.z_stride + c0 + c]), s = sigmoid(z);
                    dz = to_float(p.dy[at]) * fmaf(D, x, sh.sums[0][j][c]) * (s * fmaf(z, 1.0f - s, 1.0f));
                }
            }
            p.dx[at] = from_float<T>(dx);
            p.d_delta[at] = from_float<T>(dd);
            if (p.d_z != nullptr) p.d_z[at] = from_float<T>(dz);
        }
        // ---- the block's part of the sums over channels
        for (uint32_t i = tid; i < TILE * 2 * NP; i += BACK_THREADS) {
            const uint32_t j = i / (2 * NP), which = i / NP % 2, n = i % NP, t = tb + j;
            if (n >= p.state || t >= to) continue;
            float sum = 0.0f;
            if (t >= live_from && t < live_to) {
#pragma unroll
                for (int w = 0; w < BACK_WARPS; ++w) sum += sh.part[w][j][which][n];
            }
            p.part_BC[(((static_cast<size_t>(tile) * seq.tokens + t) * p.groups + group) * 2 + which) * p.state + n] = sum;
        }
        __syncthreads();
    }

    if (ENDS) {
        store_state(g, p.chunk_state + state_of(k_chunk));
        if (valid && part == 0) p.chunk_time[static_cast<size_t>(k_chunk) * p.channels + channel] = time;
        return;
    }
    store_state(dA, p.part_A + state_of(k_chunk));
    // a thread's token sums belong to channel tid % CPB; LANES threads share one
    static_assert(sizeof(sh.part) >= 2 * BACK_THREADS * sizeof(float), "room for two sums a thread");
    float *const sums = &sh.part[0][0][0][0];
    sums[tid] = d_D;
    sums[BACK_THREADS + tid] = d_bias;
    __syncthreads();
    if (tid < c_count) {
        float a = 0.0f, b = 0.0f;
        for (int i = 0; i < LANES; ++i) {
            a += sums[i * CPB + tid];
            b += sums[BACK_THREADS + i * CPB + tid];
        }
        p.part_D[static_cast<size_t>(k_chunk) * p.channels + c0 + tid] = a;
        p.part_bias[static_cast<size_t>(k_chunk) * p.channels + c0 + tid] = b;
    }
    if (p.d_initial != nullptr) {                       // sequences without a token hand their gradient on
        for (uint32_t s = k_chunk; s < seq.count; s += p.n_chunks) {
            if (seq.end(s) > seq.begin(s)) continue;
            load_or_zero(g, p.d_last, s);
            store_state(g, p.d_initial + state_of(s));
        }
    }
}

// Adds the parts up in their order: dB and dC (values of `rows` groups of tokens), then dA, dD and the bias'.
template<typename T>
struct SumArgs {
    const float *part_BC, *part_A, *part_D, *part_bias;
    T *d_B, *d_C;
    float *d_A, *d_D, *d_bias;
    size_t n_BC, n_A, n_C;          // tokens * groups * 2 * state, channels * state, channels
    uint32_t tiles, n_chunks, state;
};

template<typename T>
__global__ void __launch_bounds__(256)
state_scan_sum_kernel(const SumArgs<T> p) {
    const size_t step = static_cast<size_t>(gridDim.x) * blockDim.x, me = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    for (size_t i = me; i < p.n_BC; i += step) {
        float sum = 0.0f;
        for (uint32_t k = 0; k < p.tiles; ++k) sum += p.part_BC[k * p.n_BC + i];
        const size_t row = i / (2 * p.state), at = i % (2 * p.state);
        (at < p.state ? p.d_B : p.d_C)[row * p.state + at % p.state] = from_float<T>(sum);
    }
    for (size_t i = me; i < p.n_A; i += step) {
        float sum = 0.0f;
        for (uint32_t k = 0; k < p.n_chunks; ++k) sum += p.part_A[k * p.n_A + i];
        p.d_A[i] = sum;
    }
    for (size_t i = me; i < p.n_C; i += step) {
        float a = 0.0f, b = 0.0f;
        for (uint32_t k = 0; k < p.n_chunks; ++k) {
            a += p.part_D[k * p.n_C + i];
            b += p.part_bias[k * p.n_C + i];
        }
        if (p.d_D != nullptr) p.d_D[i] = a;
        if (p.d_bias != nullptr) p.d_bias[i] = b;
    }
}

struct BackPlan {
    uint32_t per_lane, lanes, chunk, n_chunks, tiles;
    size_t BC, A, C, bytes;
};

BackPlan plan_backward(const bpl_state_scan_descriptor &d) {
    BackPlan q;
    q.per_lane = d.state <= 64 ? 2 : 4;
    q.lanes = 1;
    while (q.lanes * q.per_lane < d.state) q.lanes *= 2;
    const uint32_t per_block = BACK_THREADS / q.lanes, per_group = d.channels / d.groups;
    q.tiles = (per_group + per_block - 1) / per_block;
    const uint64_t blocks = static_cast<uint64_t>(q.tiles) * d.groups, want = 4ull * sm_count();
    uint64_t chunks = blocks ? want / blocks : 1;
    const uint64_t most = (d.tokens + 63) / 64;
    chunks = chunks > most ? most : chunks;
    if (chunks < 1) chunks = 1;
    const uint64_t chunk = (d.tokens + chunks - 1) / chunks;
    q.chunk = static_cast<uint32_t>((chunk + TILE - 1) / TILE * TILE);
    if (q.chunk == 0) q.chunk = TILE;
    q.n_chunks = (d.tokens + q.chunk - 1) / q.chunk;
    if (q.n_chunks < 1) q.n_chunks = 1;
    q.BC = static_cast<size_t>(d.tokens) * d.groups * 2 * d.state;
    q.A = static_cast<size_t>(d.channels) * d.state;
    q.C = d.channels;
    q.bytes = sizeof(float) * (q.BC * q.tiles + q.n_chunks * (2 * q.A + 3 * q.C));
    return q;
}

template<typename T, int NS, int LANES, bool ENDS>
bool launch(cudaStream_t stream, const BackArgs<T> &p) {
    constexpr unsigned bytes = sizeof(BackShared<NS, LANES>);
    if (!allow_shared<state_scan_backward_kernel<T, NS, LANES, ENDS>>(bytes)) {
        set_status(BPL_ERR_CUDA, "state_scan_backward: shared memory");
        return false;
    }
    state_scan_backward_kernel<T, NS, LANES, ENDS><<<dim3(p.tiles * p.groups, p.n_chunks), BACK_THREADS, bytes, stream>>>(p);
    return true;
}

template<typename T, int NS, int LANES>
bool run_backward(cudaStream_t stream, const BackArgs<T> &p) {
    return (p.n_chunks == 1 || launch<T, NS, LANES, true>(stream, p)) && launch<T, NS, LANES, false>(stream, p);
}

template<typename T>
void backward(cudaStream_t stream, void **b, const bpl_state_scan_descriptor &d) {
    const BackPlan q = plan_backward(d);
    BackArgs<T> p = {};
    p.x = static_cast<const T *>(b[0]);
    p.delta = static_cast<const T *>(b[1]);
    p.A = static_cast<const float *>(b[2]);
    p.B = static_cast<const T *>(b[3]);
    p.C = static_cast<const T *>(b[4]);
    p.D = static_cast<const float *>(b[5]);
    p.z = static_cast<const T *>(b[6]);
    p.bias = static_cast<const float *>(b[7]);
    p.initial = static_cast<const float *>(b[9]);
    p.saved = static_cast<const float *>(b[10]);
    p.dy = static_cast<const T *>(b[11]);
    p.d_last = static_cast<const float *>(b[12]);
    p.dx = static_cast<T *>(b[13]);
    p.d_delta = static_cast<T *>(b[14]);
    p.d_z = static_cast<T *>(b[19]);
    p.d_initial = static_cast<float *>(b[21]);
    float *ws = static_cast<float *>(b[22]);
    p.part_BC = ws;
    p.part_A = p.part_BC + q.BC * q.tiles;
    p.chunk_state = p.part_A + q.n_chunks * q.A;
    p.part_D = p.chunk_state + q.n_chunks * q.A;
    p.part_bias = p.part_D + q.n_chunks * q.C;
    p.chunk_time = p.part_bias + q.n_chunks * q.C;
    p.x_stride = d.x_stride; p.delta_stride = d.delta_stride; p.z_stride = d.z_stride;
    p.B_stride = d.B_stride; p.B_group = d.B_group_stride; p.C_stride = d.C_stride; p.C_group = d.C_group_stride;
    p.seq = Sequences{static_cast<const int *>(b[8]), d.sequences, d.length, d.tokens};
    p.channels = d.channels; p.groups = d.groups; p.per_group = d.channels / d.groups; p.tiles = q.tiles; p.state = d.state;
    p.chunk = q.chunk; p.n_chunks = q.n_chunks; p.softplus = (d.flags & BPL_SCAN_SOFTPLUS) != 0;
    bool ok;
    if (q.per_lane == 4) ok = run_backward<T, 4, 32>(stream, p);
    else if (q.lanes == 1) ok = run_backward<T, 2, 1>(stream, p);
    else if (q.lanes == 2) ok = run_backward<T, 2, 2>(stream, p);
    else if (q.lanes == 4) ok = run_backward<T, 2, 4>(stream, p);
    else if (q.lanes == 8) ok = run_backward<T, 2, 8>(stream, p);
    else if (q.lanes == 16) ok = run_backward<T, 2, 16>(stream, p);
    else ok = run_backward<T, 2, 32>(stream, p);
    if (!ok) return;
    SumArgs<T> s = {};
    s.part_BC = p.part_BC; s.part_A = p.part_A; s.part_D = p.part_D; s.part_bias = p.part_bias;
    s.d_A = static_cast<float *>(b[15]);
    s.d_B = static_cast<T *>(b[16]);
    s.d_C = static_cast<T *>(b[17]);
    s.d_D = static_cast<float *>(b[18]);
    s.d_bias = static_cast<float *>(b[20]);
    s.n_BC = q.BC; s.n_A = q.A; s.n_C = q.C; s.tiles = q.tiles; s.n_chunks = q.n_chunks; s.state = d.state;
    const size_t most = q.BC > q.A ? q.BC : q.A;
    const size_t blocks = (most + 255) / 256;
    state_scan_sum_kernel<T><<<static_cast<unsigned>(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, stream>>>(s);
}

}  // namespace

size_t state_scan_backward_workspace_bytes(const char *opaque, size_t opaque_len) {
    if (opaque == nullptr || opaque_len != sizeof(bpl_state_scan_descriptor)) return 0;
    const auto &d = *reinterpret_cast<const bpl_state_scan_descriptor *>(opaque);
    return d.state < 1 || d.state > SCAN_MAX_STATE || d.groups < 1 ? 0 : plan_backward(d).bytes;
}

}  // namespace bpl

using namespace bpl;

extern "C" void state_scan_backward(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = unpack<bpl_state_scan_descriptor>(opaque, opaque_len);
    if (d == nullptr || d->channels == 0) return;
    if (d->dtype > BPL_BFLOAT16 || d->state < 1 || d->state > SCAN_MAX_STATE || d->groups < 1 || d->channels % d->groups != 0 ||
        d->tokens >= (1u << 31)) {
        set_status(BPL_ERR_ARGUMENT, "state_scan_backward: 1..128 states, channels a multiple of groups, fewer than 2^31 tokens");
        return;
    }
    bool given = true;
    for (int i : {2, 15, 22}) given &= buffers[i] != nullptr;
    if (d->tokens > 0)
        for (int i : {0, 1, 3, 4, 10, 11, 13, 14, 16, 17}) given &= buffers[i] != nullptr;
    // a gradient where there is an operand
    const int pairs[4][2] = {{5, 18}, {6, 19}, {7, 20}, {9, 21}};
    for (const auto &io : pairs) given &= buffers[io[0]] == nullptr || buffers[io[1]] != nullptr;
    if (!given) {
        set_status(BPL_ERR_ARGUMENT, "state_scan_backward: null buffer");
        return;
    }
    if (d->dtype == BPL_FLOAT) backward<float>(stream, buffers, *d);
    else if (d->dtype == BPL_HALF) backward<__half>(stream, buffers, *d);
    else backward<__nv_bfloat16>(stream, buffers, *d);
    launch_ok();
}
