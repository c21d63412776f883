// The gradient of state_scan.  With dY = dy silu(z) (dy without a gate) and a[t] = exp(dt A):
//
//     q[t] = C[t] dY[t] + a[t + 1] q[t + 1]          the derivative by h[t], from the last token to the first
//     dC = sum over channels of dY h;  dB = sum over channels of q dt x;  dx = D dY + dt sum_n q B
//     d(dt) = x sum_n q B + sum_n q a h[t - 1] A;  dA = sum over tokens of q a h[t - 1] dt
//
// A block walks its tokens tile by tile from the last to the first.  The states of a group of tokens are computed once more
// from the one that the forward pass kept in front of the tile, and stay in registers for the way back.  Sums over channels are
// left as one part per block and token, sums over tokens as one part per chunk, and added up in a fixed order by a last kernel:
// the same call gives the same bits.
#include <algorithm>

#include "state_scan.cuh"

namespace bpl {
namespace {

constexpr uint32_t TILE = SCAN_TILE_TOKENS;
constexpr int GROUP = 4;                   // tokens whose states are in registers at once
__host__ __device__ constexpr int walkers(int lanes) { return lanes == 1 ? 64 : 128; }

template<typename T>
struct BackArgs {
    const T *x, *delta, *z, *B, *C, *dy;
    const float *A, *D, *bias, *initial, *saved, *d_last;
    T *dx, *d_delta, *d_z;
    float *d_initial;
    float *part_BC;                    // [tiles of a launch][tokens][groups][2][state]
    float *part_A, *part_D, *part_bias;   // [n_chunks][channels](state)
    float *chunk_state, *chunk_time;
    long long x_stride, delta_stride, z_stride, B_stride, B_group, C_stride, C_group;
    Sequences seq;
    uint32_t channels, groups, per_group, tile0, tiles, state, chunk, n_chunks;      // tiles tile0 .. tile0 + tiles - 1 of every group
    uint32_t row_copy, state_copy;
    bool softplus, out_pairs, state_aligned;
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

// Shared memory of a block: a ring of copies as in the forward pass; times, inputs and cotangents as floats for the tile that is
// turned, the one that is walked and the one that is read out; sums of the latter two.
template<typename T, int LANES>
struct BackShared {
    static constexpr int WALKERS = walkers(LANES), CPB = WALKERS / LANES, NP = NS * LANES, Y_ROW = CPB + (LANES < 32 ? 32 / LANES : 2);
    static_assert(CPB % 2 == 0 && Y_ROW % 2 == 0 && sizeof(T) * CPB * TILE % 16 == 0 && sizeof(T) * NP * TILE % 16 == 0,
                  "alignment of pairs and copies");
    static constexpr int RING = 5;
    struct Raw {
        T x[TILE][CPB], delta[TILE][CPB], z[TILE][CPB], dy[TILE][CPB];
        alignas(16) T B[TILE][NP], C[TILE][NP];
    } raw[RING];
    float step[3][TILE][CPB][2], dY[3][TILE][CPB];          // dt and dt x; dy times the gate
    float sums[2][3][TILE][Y_ROW];                          // over a channel's states: h C, q B, q a h A
    float part[2][WALKERS / 32][TILE][2][NP];               // over a warp's channels: of B and C
    alignas(16) float middle[TILE / GROUP - 1][WALKERS][NS];
    int odd[2][CREW / 32];                                  // whether an operand is infinite, by turning warps
};

// Blocks that share an SM.
template<typename T, int LANES>
constexpr int RESIDENT = sizeof(BackShared<T, LANES>) <= 113 * 1024 ? 2 : 1;

// A lane holds NS neighbouring states of a channel, LANES lanes share a channel.  As in the forward pass a part of the block walks
// and two crews bring tiles in and out.
// What bounds it: the sums over channels and states, exchanged between lanes, and the bytes that lanes take from shared memory; so
// the decays of the way back are computed once more instead of being kept.  8192 tokens of 2048 channels, 16 states: 525 us (floor: 58
// for each time that the exponentials are taken), the pass over chunks' ends 100, the sums 16.  Code in front of which instructions wait
// counts as well: eight tokens' states in registers took a tenth more, three blocks to an SM a quarter.
// ENDS: only what a chunk hands to the one in front of it when nothing comes from behind, and the time that passes in it.
// PADDED: lanes hold more states than there are, or a block more channels.  Those are zero and add zeros to the sums, but for infinities,
// which times 0 are no numbers: tiles with such go the way of the bounds, where what is not there is cleared.
// (Registers are capped for two blocks to an SM where shared memory has room for two; elsewhere, 5 to 8 and 65 to 128 states and up to
// four, the cap would only spill.)
template<typename T, int LANES, bool ENDS, bool PADDED>
__global__ void __launch_bounds__(walkers(LANES) + CARRIERS, RESIDENT<T, LANES>)
state_scan_backward_kernel(const BackArgs<T> p) {
    using Shared = BackShared<T, LANES>;
    constexpr int CPB = Shared::CPB, NP = Shared::NP, PAIRS = NS / 2, CW = 32 / LANES, V = 2 * NS, RING = Shared::RING;
    constexpr int WALKERS = Shared::WALKERS;
    constexpr int K = LANES < GROUP ? LANES : GROUP, KV = V < CW ? V : CW, R = V / KV;
    constexpr int FLUSH = R < GROUP ? GROUP / R : 1;      // tokens whose sums over channels wait in registers
    static_assert(GROUP % K == 0 && GROUP % FLUSH == 0, "whole groups");
    extern __shared__ __align__(16) unsigned char raw_shared[];
    Shared &sh = *reinterpret_cast<Shared *>(raw_shared);

    const bool walker = threadIdx.x < WALKERS;
    const uint32_t tid = walker ? threadIdx.x : threadIdx.x - WALKERS, warp = tid / 32, local = tid / LANES, part = tid % LANES;
    const uint32_t group = blockIdx.x / p.tiles, tile = p.tile0 + blockIdx.x % p.tiles, k_chunk = blockIdx.y;
    const uint32_t c_first = tile * CPB, c_count = min(static_cast<uint32_t>(CPB), p.per_group - c_first);
    const uint32_t c0 = group * p.per_group + c_first, channel = c0 + local;
    const bool valid = walker && local < c_count;
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
    const uint32_t n_tiles = to > from ? (to - from + TILE - 1) / TILE : 0;
    auto begin_of = [&](uint32_t i) { return from + (n_tiles - 1 - i) * TILE; };        // tiles are counted from the last

    // ---- the parts of a tile's way
    auto request = [&](uint32_t i, uint32_t place) {
        if (i < n_tiles) {
            typename Shared::Raw &r = sh.raw[place];
            const uint32_t tb = begin_of(i);
            if (tid / 32 == 2) {
                fetch<TILE>(r.dy, p.dy + c0, static_cast<long long>(p.channels), tb, live_from, live_to, c_count, p.row_copy);
                if (p.z != nullptr) fetch<TILE>(r.z, p.z + c0, p.z_stride, tb, live_from, live_to, c_count, p.row_copy);
                fetch<TILE>(r.C, p.C + group * p.C_group, p.C_stride, tb, live_from, live_to, p.state, p.state_copy);
            } else {
                fetch<TILE>(r.delta, p.delta + c0, p.delta_stride, tb, live_from, live_to, c_count, p.row_copy);
                if (!ENDS) fetch<TILE>(r.x, p.x + c0, p.x_stride, tb, live_from, live_to, c_count, p.row_copy);
                if (!ENDS) fetch<TILE>(r.B, p.B + group * p.B_group, p.B_stride, tb, live_from, live_to, p.state, p.state_copy);
            }
        }
        copies_commit();
    };
    const bool turner = !walker && tid < CREW;
    const uint32_t mate = tid % CREW, e2 = mate % (CPB / 2) * 2, j2 = mate / (CPB / 2);
    constexpr uint32_t J_STEP = CREW / (CPB / 2), TURNS = J_STEP > TILE ? 1 : TILE / J_STEP;
    const bool has0 = e2 < c_count, has1 = e2 + 1 < c_count, at_work = J_STEP <= TILE || j2 < TILE;
    pair bias = 0, D = 0;
    if (p.bias != nullptr) bias = make_pair(has0 ? p.bias[c0 + e2] : 0.0f, has1 ? p.bias[c0 + e2 + 1] : 0.0f);
    if (!ENDS && p.D != nullptr) D = make_pair(has0 ? p.D[c0 + e2] : 0.0f, has1 ? p.D[c0 + e2 + 1] : 0.0f);
    auto turn = [&](uint32_t i, uint32_t place, uint32_t at) {
        if (i >= n_tiles) return;
        typename Shared::Raw &r = sh.raw[place];
        const uint32_t tb = begin_of(i);
        pair dt[TURNS], in[TURNS], dY[TURNS];
        if (at_work) {
#pragma unroll
            for (uint32_t q = 0; q < TURNS; ++q) {
                const uint32_t j = j2 + q * J_STEP;
                dt[q] = add2(load_pair(&r.delta[j][e2]), bias);
                if (!ENDS) in[q] = load_pair(&r.x[j][e2]);
                dY[q] = load_pair(&r.dy[j][e2]);
                if (p.z != nullptr) {
                    const float2 z = split(load_pair(&r.z[j][e2]));
                    dY[q] = mul2(dY[q], make_pair(silu(z.x), silu(z.y)));
                }
            }
            if (p.softplus)
#pragma unroll
                for (uint32_t q = 0; q < TURNS; ++q) dt[q] = softplus_pair(dt[q]);
#pragma unroll
            for (uint32_t q = 0; q < TURNS; ++q) {
                const uint32_t j = j2 + q * J_STEP, t = tb + j;
                const bool live0 = t >= live_from && t < live_to && has0, live1 = t >= live_from && t < live_to && has1;
                const float2 d = split(dt[q]), u = ENDS ? make_float2(0.0f, 0.0f) : split(mul2(dt[q], in[q])), y = split(dY[q]);
                *reinterpret_cast<float4 *>(sh.step[at][j][e2]) =
                    make_float4(live0 ? d.x : 0.0f, live0 ? u.x : 0.0f, live1 ? d.y : 0.0f, live1 ? u.y : 0.0f);
                store_pair(&sh.dY[at][j][e2], make_float2(live0 ? y.x : 0.0f, live1 ? y.y : 0.0f));
            }
        }
        if (p.state < NP || tb < live_from || tb + TILE > live_to)
            for (uint32_t k = mate; k < TILE * NP; k += CREW) {
                const uint32_t j = k / NP, n = k % NP, t = tb + j;
                if (n < p.state && t >= live_from && t < live_to) continue;
                r.B[j][n] = from_float<T>(0.0f);
                r.C[j][n] = from_float<T>(0.0f);
            }
        if constexpr (PADDED) {
            bool odd = false;
            const auto see = [&odd](float a, float b) { odd |= !(fmaxf(fabsf(a), fabsf(b)) < INFINITY); };
            if (at_work)
#pragma unroll 1
                for (uint32_t q = 0; q < TURNS; ++q) {
                    const uint32_t j = j2 + q * J_STEP;
                    const float4 v = *reinterpret_cast<const float4 *>(sh.step[at][j][e2]);
                    const float2 y = split(load_pair(&sh.dY[at][j][e2]));
                    see(v.x, v.z);
                    see(v.y, v.w);
                    see(y.x, y.y);
                }
            if (c_count < CPB)          // (channels that are not there meet the operands that all channels share)
                for (uint32_t k = mate; k < TILE * NP; k += CREW) {
                    const uint32_t t = tb + k / NP;
                    if (k % NP < p.state && t >= live_from && t < live_to) see(to_float(r.B[k / NP][k % NP]), to_float(r.C[k / NP][k % NP]));
                }
            odd = __any_sync(FULL_MASK, odd);
            if (tid % 32 == 0) sh.odd[i & 1][tid / 32] = odd;
        }
    };
    const bool store_pairs = (p.channels & 1u) == 0 && (c0 & 1u) == 0 && p.out_pairs && has1;
    float2 d_D = make_float2(0.0f, 0.0f), d_bias = d_D;          // of a thread's two channels
    auto read_out = [&](uint32_t i, uint32_t place, uint32_t at) {
        const typename Shared::Raw &r = sh.raw[place];
        const uint32_t tb = begin_of(i);
        if (at_work) {
            float2 d_D_tile = make_float2(0.0f, 0.0f), d_bias_tile = d_D_tile;
#pragma unroll 2
            for (uint32_t q = 0; q < TURNS; ++q) {
                const uint32_t j = j2 + q * J_STEP, t = tb + j;
                const bool live = t >= live_from && t < live_to;
                const pair x = load_pair(&r.x[j][e2]), dY = load_pair(&sh.dY[at][j][e2]);
                const pair qB = load_pair(&sh.sums[i & 1][1][j][e2]);
                const float4 st = *reinterpret_cast<const float4 *>(sh.step[at][j][e2]);
                const pair through_state = mul2(make_pair(st.x, st.z), qB);
                float2 dx = split(p.D != nullptr ? fma2(D, dY, through_state) : through_state);
                float2 dd = split(fma2(load_pair(&sh.sums[i & 1][2][j][e2]), make_pair(LN_2, LN_2), mul2(x, qB)));
                if (p.softplus) {
                    const float2 raw = split(add2(load_pair(&r.delta[j][e2]), bias));
                    dd.x *= sigmoid(raw.x);
                    dd.y *= sigmoid(raw.y);
                }
                float2 dz = make_float2(0.0f, 0.0f);
                if (p.z != nullptr) {
                    const float2 z = split(load_pair(&r.z[j][e2])), dy = split(load_pair(&r.dy[j][e2]));
                    const pair sum = load_pair(&sh.sums[i & 1][0][j][e2]);
                    const float2 y = split(p.D != nullptr ? fma2(D, x, sum) : sum);
                    const float s0 = sigmoid(z.x), s1 = sigmoid(z.y);
                    dz = make_float2(dy.x * y.x * (s0 * fmaf(z.x, 1.0f - s0, 1.0f)), dy.y * y.y * (s1 * fmaf(z.y, 1.0f - s1, 1.0f)));
                }
                const float2 yx = split(mul2(dY, x));
                if (live) {
                    d_D_tile.x += yx.x;
                    d_D_tile.y += yx.y;
                    d_bias_tile.x += dd.x;
                    d_bias_tile.y += dd.y;
                } else {
                    dx = dd = dz = make_float2(0.0f, 0.0f);
                }
                if (t < to) {
                    const size_t o = static_cast<size_t>(t) * p.channels + c0 + e2;
                    if (store_pairs) {
                        store_pair(p.dx + o, dx);
                        store_pair(p.d_delta + o, dd);
                        if (p.d_z != nullptr) store_pair(p.d_z + o, dz);
                    } else {
                        if (has0) {
                            p.dx[o] = from_float<T>(dx.x);
                            p.d_delta[o] = from_float<T>(dd.x);
                            if (p.d_z != nullptr) p.d_z[o] = from_float<T>(dz.x);
                        }
                        if (has1) {
                            p.dx[o + 1] = from_float<T>(dx.y);
                            p.d_delta[o + 1] = from_float<T>(dd.y);
                            if (p.d_z != nullptr) p.d_z[o + 1] = from_float<T>(dz.y);
                        }
                    }
                }
            }
            d_D.x += d_D_tile.x;
            d_D.y += d_D_tile.y;
            d_bias.x += d_bias_tile.x;
            d_bias.y += d_bias_tile.y;
        }
        // the block's part of the sums over channels
        const bool whole = tb >= live_from && tb + TILE <= live_to;
#pragma unroll 4
        for (uint32_t k = mate; k < TILE * 2 * NP; k += CREW) {
            const uint32_t j = k / (2 * NP), which = k / NP % 2, n = k % NP, t = tb + j;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WALKERS / 32; ++w) sum += sh.part[i & 1][w][j][which][n];
            if (!whole && !(t >= live_from && t < live_to)) sum = 0.0f;
            if (n < p.state && t < to)
                p.part_BC[(((static_cast<size_t>(tile - p.tile0) * seq.tokens + t) * p.groups + group) * 2 + which) * p.state + n] = sum;
        }
    };

    if (!walker && !turner)
#pragma unroll 1
        for (uint32_t i = 0; i < RING - 2; ++i) request(i, i);

    // ---- walking
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
    float time = 0.0f;
    const bool by_vectors = p.state % 4 == 0 && p.state_aligned;
    auto load_state = [&](pair (&to_pairs)[PAIRS], const float *at) {
        if (by_vectors) {
            const float4 v = valid && n0 < p.state ? __ldcg(reinterpret_cast<const float4 *>(at + n0)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            to_pairs[0] = make_pair(v.x, v.y);
            to_pairs[1] = make_pair(v.z, v.w);
            return;
        }
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
    if (walker && live_from < live_to && live_to == to && to < last && !ENDS) {
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
                for (int k = 0; k < PAIRS; ++k) g[k] = add2(through_chunk(g[k], mul2(dt, A2[k])), own[k]);
            }
        }
    }
    pair before[PAIRS], then[PAIRS];           // the kept states in front of this tile and of the next
#pragma unroll
    for (int k = 0; k < PAIRS; ++k) before[k] = then[k] = 0;
    if (!ENDS && walker && n_tiles > 0) load_state(then, p.saved + state_of(begin_of(0) / TILE));

    auto only_there = [&](pair v, int k) {
        const float2 f = split(v);
        return make_pair(valid && n0 + 2 * k < p.state ? f.x : 0.0f, valid && n0 + 2 * k + 1 < p.state ? f.y : 0.0f);
    };

    // BOUNDED: sequences begin or end in the tile, tokens belong to none, or operands are infinite.  (Without them there is no branch
    // between tokens, so that one token's loads and exponentials run beside another's chain.)
    auto walk_tile = [&](uint32_t i, const typename Shared::Raw &r, uint32_t tb, uint32_t at, uint32_t starts, uint32_t ends, uint32_t dead,
                         auto bounded) {
        constexpr bool BOUNDED = decltype(bounded)::value;
        if (ENDS) {
            float passed = 0.0f;
#pragma unroll
            for (int j = TILE - 1; j >= 0; --j) {
                const float dtj = sh.step[at][j][local][0], dYj = sh.dY[at][j][local];
                const pair dt = make_pair(dtj, dtj), dY = make_pair(dYj, dYj);
                if (BOUNDED && (ends >> j & 1)) load_or_zero(g, p.d_last, seq.of(tb + j));
                passed += dtj;
                pair c[PAIRS];
                load_states(&r.C[j][n0], c);
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) g[k] = mul2(fma2(c[k], dY, g[k]), decay_pair(dt, A2[k]));
            }
            time += passed;
            return;
        }
        // forwards through the tile, GROUP tokens at a time: the state in front of every group into shared memory (a thread's own)
        // (a token of no sequence finds no state, not the one that the sequence in front has left, which may be infinite)
        auto enter = [&](uint32_t j, pair (&state)[PAIRS]) {
            if (!BOUNDED) return;
            if (starts >> j & 1) load_or_zero(state, p.initial, seq.of(tb + j));
            else if (dead >> j & 1) load_or_zero(state, nullptr, 0);
        };
        auto forward = [&](uint32_t j, const pair (&state)[PAIRS], pair (&after)[PAIRS]) {
            const float2 d = *reinterpret_cast<const float2 *>(sh.step[at][j][local]);
            const pair dt = make_pair(d.x, d.x), in = make_pair(d.y, d.y);
            pair b[PAIRS];
            load_states(&r.B[j][n0], b);
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) {
                after[k] = fma2(state[k], decay_pair(dt, A2[k]), mul2(in, b[k]));
                if (BOUNDED && PADDED) after[k] = only_there(after[k], k);
            }
        };
        pair middle[PAIRS], dA_tile[PAIRS];
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
            middle[k] = before[k];
            dA_tile[k] = 0;
        }
        ulonglong2 *const middles = reinterpret_cast<ulonglong2 *>(sh.middle[0][0]) + tid;      // WALKERS apart
#pragma unroll 1
        for (int j0 = 0; j0 < static_cast<int>(TILE) - GROUP; j0 += GROUP) {
#pragma unroll
            for (int m = 0; m < GROUP; ++m) {
                enter(j0 + m, middle);
                forward(j0 + m, middle, middle);
            }
            middles[j0 / GROUP * WALKERS] = make_ulonglong2(middle[0], middle[1]);
        }
        // the groups, the last one first: forwards with the states into registers, and back
        const int cw = (tid % 32) / LANES;
#pragma unroll 1
        for (int j0 = static_cast<int>(TILE) - GROUP; j0 >= 0; j0 -= GROUP) {
            pair h[GROUP][PAIRS], start[PAIRS];
            start[0] = before[0];
            start[1] = before[1];
            if (j0 > 0) {
                const ulonglong2 v = middles[(j0 / GROUP - 1) * WALKERS];
                start[0] = v.x;
                start[1] = v.y;
            }
#pragma unroll
            for (int m = 0; m < GROUP; ++m) {
                pair prev[PAIRS];
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) prev[k] = m ? h[m ? m - 1 : 0][k] : start[k];
                enter(j0 + m, prev);
                forward(j0 + m, prev, h[m]);
            }
            // (results are written in groups, so that loads need not wait for stores)
            float waiting[FLUSH][R], sum_y[GROUP / K], sum_b[GROUP / K], sum_a[GROUP / K];
#pragma unroll
            for (int m0 = GROUP - K; m0 >= 0; m0 -= K) {
                float hC[K], qB[K], wA[K];
#pragma unroll
                for (int e = K - 1; e >= 0; --e) {
                    const int m = m0 + e, j = j0 + m;
                    const float2 d = *reinterpret_cast<const float2 *>(sh.step[at][j][local]);
                    const float dYj = sh.dY[at][j][local];
                    const pair dt = make_pair(d.x, d.x), in = make_pair(d.y, d.y), dY = make_pair(dYj, dYj);
                    if (BOUNDED && (ends >> j & 1)) load_or_zero(g, p.d_last, seq.of(tb + j));
                    pair prev[PAIRS], b[PAIRS], c[PAIRS];
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) prev[k] = m ? h[m ? m - 1 : 0][k] : start[k];
                    enter(j, prev);
                    load_states(&r.B[j][n0], b);
                    load_states(&r.C[j][n0], c);
                    pair sum_hC = 0, sum_qB = 0, sum_wA = 0;
                    float v[V];
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) {
                        pair q = fma2(c[k], dY, g[k]);
                        if (BOUNDED && PADDED) q = only_there(q, k);
                        const float2 to_B = split(mul2(q, in)), to_C = split(mul2(dY, h[m][k]));
                        v[2 * k] = to_B.x;
                        v[2 * k + 1] = to_B.y;
                        v[NS + 2 * k] = to_C.x;
                        v[NS + 2 * k + 1] = to_C.y;
                        sum_hC = k == 0 ? mul2(h[m][k], c[k]) : fma2(h[m][k], c[k], sum_hC);
                        sum_qB = k == 0 ? mul2(q, b[k]) : fma2(q, b[k], sum_qB);
                        g[k] = mul2(q, decay_pair(dt, A2[k]));
                        if (BOUNDED && PADDED) g[k] = only_there(g[k], k);
                        const pair w = mul2(g[k], prev[k]);
                        sum_wA = k == 0 ? mul2(w, A2[k]) : fma2(w, A2[k], sum_wA);
                        dA_tile[k] = fma2(w, dt, dA_tile[k]);
                    }
                    hC[e] = sum2(sum_hC);
                    qB[e] = sum2(sum_qB);
                    wA[e] = sum2(sum_wA);
                    if (BOUNDED && (starts >> j & 1)) {
                        if (p.d_initial != nullptr) store_state(g, p.d_initial + state_of(seq.of(tb + j)));
#pragma unroll
                        for (int k = 0; k < PAIRS; ++k) g[k] = 0;
                    }
                    sum_over_channels<V, CW, LANES>(v, cw);
#pragma unroll
                    for (int f = 0; f < R; ++f) waiting[m % FLUSH][f] = v[f];
                    if (m % FLUSH == 0 && cw < KV) {
#pragma unroll
                        for (int u = 0; u < FLUSH; ++u)
#pragma unroll
                            for (int f = 0; f < R; ++f) {
                                const int o = cw * R + f;              // 0 .. NS - 1: of B, NS .. 2 NS - 1: of C
                                sh.part[i & 1][warp][j + u][o / NS][n0 + o % NS] = waiting[u][f];
                            }
                    }
                }
                sum_y[m0 / K] = sum_over_lanes<K, LANES>(hC, part);
                sum_b[m0 / K] = sum_over_lanes<K, LANES>(qB, part);
                sum_a[m0 / K] = sum_over_lanes<K, LANES>(wA, part);
            }
            if (part < K)
#pragma unroll
                for (int m = 0; m < GROUP; m += K) {
                    sh.sums[i & 1][0][j0 + m + part][local] = sum_y[m / K];
                    sh.sums[i & 1][1][j0 + m + part][local] = sum_b[m / K];
                    sh.sums[i & 1][2][j0 + m + part][local] = sum_a[m / K];
                }
        }
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) dA[k] = add2(dA[k], dA_tile[k]);
    };

    auto walk = [&](uint32_t i, uint32_t place, uint32_t at) {
        const uint32_t tb = begin_of(i);
        const typename Shared::Raw &r = sh.raw[place];
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) before[k] = then[k];
        if (!ENDS && i + 1 < n_tiles) load_state(then, p.saved + state_of(tb / TILE - 1));
        if (tb >= live_to || tb + TILE <= live_from) return;        // (nothing is read from a tile without a token of a sequence)
        // bit j: token tb + j is the first, the last of its sequence, or of none
        uint32_t starts = 0, ends = 0, dead = 0;
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
            dead = __ballot_sync(FULL_MASK, t < live_from || t >= live_to) & 0xffffu;
            next_begin = tb >= live_from && tb < live_to ? seq.begin(seq.of(tb)) : 0xffffffffu;
        }
        bool odd = false;
        if constexpr (PADDED) odd = (sh.odd[i & 1][0] | sh.odd[i & 1][1]) != 0;
        if ((starts | ends | dead) == 0 && !odd) walk_tile(i, r, tb, at, 0u, 0u, 0u, std::false_type());
        else walk_tile(i, r, tb, at, starts, ends, dead, std::true_type());
    };

    if (!walker) copies_wait<RING - 4>();        // tiles 0 and 1 are there
    __syncthreads();
    if (turner) turn(0, 0, 0);
    __syncthreads();
    uint32_t before_place = RING - 1, here = 0, next = 1, ahead = RING - 2;      // places in the ring of tiles i - 1, i, i + 1, i + RING - 2
    uint32_t behind = 2, at = 0, coming = 1;                                     // of the turned tiles i - 1, i, i + 1
    for (uint32_t i = 0; i <= n_tiles; ++i) {
        if (walker) {
            if (i < n_tiles) walk(i, here, at);
        } else if (turner) {
            turn(i + 1, next, coming);
        } else {
            request(i + RING - 2, ahead);
            if (!ENDS && i > 0) read_out(i - 1, before_place, behind);
            copies_wait<RING - 4>();
        }
        __syncthreads();
        before_place = here;
        here = next;
        next = next + 1 == RING ? 0 : next + 1;
        ahead = ahead + 1 == RING ? 0 : ahead + 1;
        behind = at;
        at = coming;
        coming = coming + 1 == 3 ? 0 : coming + 1;
    }

    if (ENDS) {
        store_state(g, p.chunk_state + state_of(k_chunk));
        if (valid && part == 0) p.chunk_time[static_cast<size_t>(k_chunk) * p.channels + channel] = time;
        return;
    }
    store_state(dA, p.part_A + state_of(k_chunk));
    // a reading thread's token sums belong to its two channels; J_STEP threads share them
    static_assert(sizeof(sh.part) >= 4 * CREW * sizeof(float), "room for four sums a thread");
    float4 *const token_sums = reinterpret_cast<float4 *>(&sh.part[0][0][0][0][0]);
    if (!walker && !turner) token_sums[mate] = make_float4(d_D.x, d_D.y, d_bias.x, d_bias.y);
    __syncthreads();
    if (!walker && !turner && mate < CPB / 2) {
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t q = 0; q < J_STEP && q < TILE; ++q) {
            const float4 v = token_sums[q * (CPB / 2) + mate];
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
        const size_t o = static_cast<size_t>(k_chunk) * p.channels + c0 + 2 * mate;
        if (2 * mate < c_count) {
            p.part_D[o] = sum.x;
            p.part_bias[o] = sum.z;
        }
        if (2 * mate + 1 < c_count) {
            p.part_D[o + 1] = sum.y;
            p.part_bias[o + 1] = sum.w;
        }
    }
    if (p.d_initial != nullptr) {                       // sequences without a token hand their gradient on
        for (uint32_t s = k_chunk; s < seq.count; s += p.n_chunks) {
            if (seq.end(s) > seq.begin(s)) continue;
            load_or_zero(g, p.d_last, s);
            store_state(g, p.d_initial + state_of(s));
        }
    }
}

// Adds the parts up in their order: dB and dC, whose tiles may come in several launches (`so_far`: the sum over the tiles in front),
// then dA, dD and the bias'.
template<typename T>
struct SumArgs {
    const float *part_BC, *part_A, *part_D, *part_bias;
    float *so_far;
    bool first, last;
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
        float sum = p.first ? 0.0f : p.so_far[i];
        for (uint32_t k = 0; k < p.tiles; ++k) sum += p.part_BC[k * p.n_BC + i];
        if (!p.last) {
            p.so_far[i] = sum;
            continue;
        }
        const size_t row = i / (2 * p.state), at = i % (2 * p.state);
        (at < p.state ? p.d_B : p.d_C)[row * p.state + at % p.state] = from_float<T>(sum);
    }
    if (!p.last) return;
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

template<typename T>
uint32_t resident(uint32_t lanes) {
    switch (lanes) {
        case 1: return RESIDENT<T, 1>;
        case 2: return RESIDENT<T, 2>;
        case 4: return RESIDENT<T, 4>;
        case 8: return RESIDENT<T, 8>;
        case 16: return RESIDENT<T, 16>;
        default: return RESIDENT<T, 32>;
    }
}

struct BackPlan {
    uint32_t lanes, chunk, n_chunks, tiles, at_once;     // tiles of a launch
    size_t BC, A, C, bytes;
};

// Chunks of tokens for `blocks` blocks of channels: the number that takes the least time when two blocks share an SM, an SM with one
// block takes 0.61 of the time of one with two, and the pass in front, over all chunks but one, costs 0.14 of the main one.  Few
// channels: two blocks for every SM.  No chunk shorter than 64 tokens.  (With the forward pass, 1400 tokens of 2756 channels, 64
// states: two blocks for every SM 1.11 ms, this 0.95; 65,536 tokens of 128 channels: 16 chunks 1.09 ms, 74 chunks 0.49.)  The costs are
// those of 9 to 64 states, in 32 bits 9 to 32; elsewhere an SM has shared memory for one block, and its two come one after the other.
uint32_t chunks_for(uint64_t blocks, uint32_t tokens) {
    const uint64_t sms = static_cast<uint64_t>(sm_count());
    if (blocks * 8 <= sms) {
        const uint64_t chunks = blocks == 0 ? 1 : 2 * sms / blocks, most = tokens / 64;
        return static_cast<uint32_t>(most < 1 ? 1 : chunks < most ? chunks : most);
    }
    uint32_t best = 1;
    double least = 0.0;
    for (uint32_t c = 1; c <= 16 && (c == 1 || static_cast<uint64_t>(c) * 64 <= tokens); ++c) {
        const uint64_t all = blocks * c, rest = all % (2 * sms);
        const double rounds = static_cast<double>(all / (2 * sms)) + (rest == 0 ? 0.0 : rest <= sms ? 0.61 : 1.0);
        const double time = rounds / c * (1.0 + 0.14 * (c - 1) / c);
        if (c == 1 || time < least) {
            least = time;
            best = c;
        }
    }
    return best;
}

constexpr uint64_t PARTS_BYTES = 2ull << 30;

BackPlan plan_backward(const bpl_state_scan_descriptor &d) {
    BackPlan q;
    q.lanes = lanes_for(d.state);
    const uint32_t per_block = walkers(q.lanes) / q.lanes, per_group = d.channels / d.groups;
    q.tiles = (per_group + per_block - 1) / per_block;
    const uint64_t chunks = chunks_for(static_cast<uint64_t>(q.tiles) * d.groups, d.tokens);
    const uint64_t chunk = (d.tokens + chunks - 1) / chunks;
    q.chunk = static_cast<uint32_t>((chunk + TILE - 1) / TILE * TILE);
    if (q.chunk == 0) q.chunk = TILE;
    q.n_chunks = (d.tokens + q.chunk - 1) / q.chunk;
    if (q.n_chunks < 1) q.n_chunks = 1;
    q.BC = static_cast<size_t>(d.tokens) * d.groups * 2 * d.state;
    q.A = static_cast<size_t>(d.channels) * d.state;
    q.C = d.channels;
    // Parts of dB and dC grow with tiles and state, the square of the state: a launch holds no more tiles than PARTS_BYTES have room for,
    // in whole rounds over the card, but one round at least.  (16,384 tokens of 4096 channels, 128 states: 2.9 GB with
    // the results instead of 17.6, 40.6 ms before and 41.3 so.)
    const uint64_t per_tile = static_cast<uint64_t>(d.groups) * q.n_chunks;
    const uint64_t card = static_cast<uint64_t>(sm_count()) * (d.dtype == BPL_FLOAT ? resident<float>(q.lanes) : resident<__half>(q.lanes));
    const uint64_t round = per_tile < card ? card / per_tile : 1, room = q.BC ? PARTS_BYTES / (sizeof(float) * q.BC) : q.tiles;
    q.at_once = room >= q.tiles ? q.tiles : static_cast<uint32_t>(std::min<uint64_t>(q.tiles, std::max(round, room / round * round)));
    const size_t kept = q.BC * (q.at_once + (q.at_once < q.tiles ? 1 : 0));
    q.bytes = sizeof(float) * (kept + q.n_chunks * (2 * q.A + 3 * q.C));
    return q;
}

template<typename T, int LANES, bool ENDS, bool PADDED>
bool launch(cudaStream_t stream, const BackArgs<T> &p) {
    constexpr unsigned bytes = sizeof(BackShared<T, LANES>);
    static_assert(bytes <= 227 * 1024, "shared memory of a block");
    if (!allow_shared<state_scan_backward_kernel<T, LANES, ENDS, PADDED>>(bytes)) {
        set_status(BPL_ERR_CUDA, "state_scan_backward: shared memory");
        return false;
    }
    state_scan_backward_kernel<T, LANES, ENDS, PADDED><<<dim3(p.tiles * p.groups, p.n_chunks), walkers(LANES) + CARRIERS, bytes, stream>>>(p);
    return true;
}

template<typename T, int LANES>
bool run_backward(cudaStream_t stream, BackArgs<T> p, SumArgs<T> s, uint32_t at_once) {
    if (p.n_chunks > 1 && !launch<T, LANES, true, false>(stream, p)) return false;
    const bool full = p.state == NS * LANES && p.per_group % BackShared<T, LANES>::CPB == 0;
    const size_t blocks = (std::max(s.n_BC, s.n_A) + 255) / 256;
    const unsigned most = 8u * static_cast<unsigned>(sm_count());
    for (const uint32_t tiles = p.tiles; p.tile0 < tiles; p.tile0 += at_once) {
        p.tiles = s.tiles = std::min(at_once, tiles - p.tile0);
        if (!(full ? launch<T, LANES, false, false>(stream, p) : launch<T, LANES, false, true>(stream, p))) return false;
        s.first = p.tile0 == 0;
        s.last = p.tile0 + p.tiles == tiles;
        state_scan_sum_kernel<T><<<static_cast<unsigned>(std::min<size_t>(blocks, most)), 256, 0, stream>>>(s);
    }
    return true;
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
    p.part_A = p.part_BC + q.BC * (q.at_once + (q.at_once < q.tiles ? 1 : 0));
    p.chunk_state = p.part_A + q.n_chunks * q.A;
    p.part_D = p.chunk_state + q.n_chunks * q.A;
    p.part_bias = p.part_D + q.n_chunks * q.C;
    p.chunk_time = p.part_bias + q.n_chunks * q.C;
    p.x_stride = d.x_stride; p.delta_stride = d.delta_stride; p.z_stride = d.z_stride;
    p.B_stride = d.B_stride; p.B_group = d.B_group_stride; p.C_stride = d.C_stride; p.C_group = d.C_group_stride;
    p.seq = Sequences{static_cast<const int *>(b[8]), d.sequences, d.length, d.tokens};
    p.channels = d.channels; p.groups = d.groups; p.per_group = d.channels / d.groups; p.tiles = q.tiles; p.state = d.state;
    p.chunk = q.chunk; p.n_chunks = q.n_chunks; p.softplus = (d.flags & BPL_SCAN_SOFTPLUS) != 0;
    const uint32_t per_block = walkers(q.lanes) / q.lanes;
    p.row_copy = copy_bytes<T>({p.x, p.delta, p.z, p.dy}, {d.x_stride, d.delta_stride, p.z ? d.z_stride : 0, d.channels}, p.per_group);
    if (p.row_copy > per_block * sizeof(T)) p.row_copy = 4;
    p.state_copy = copy_bytes<T>({p.B, p.C}, {d.B_stride, d.C_stride, d.groups > 1 ? d.B_group_stride : 0, d.groups > 1 ? d.C_group_stride : 0},
                                 d.state);
    p.out_pairs = true;
    for (const void *o : {static_cast<const void *>(p.dx), static_cast<const void *>(p.d_delta), static_cast<const void *>(p.d_z)})
        p.out_pairs &= reinterpret_cast<uintptr_t>(o) % (2 * sizeof(T)) == 0;
    p.state_aligned = true;
    for (const void *a : {static_cast<const void *>(p.initial), static_cast<const void *>(p.saved), static_cast<const void *>(p.d_last),
                          static_cast<const void *>(p.chunk_state)})
        p.state_aligned &= aligned16(a);
    SumArgs<T> s = {};
    s.part_BC = p.part_BC; s.part_A = p.part_A; s.part_D = p.part_D; s.part_bias = p.part_bias;
    s.so_far = p.part_BC + q.BC * q.at_once;
    s.d_A = static_cast<float *>(b[15]);
    s.d_B = static_cast<T *>(b[16]);
    s.d_C = static_cast<T *>(b[17]);
    s.d_D = static_cast<float *>(b[18]);
    s.d_bias = static_cast<float *>(b[20]);
    s.n_BC = q.BC; s.n_A = q.A; s.n_C = q.C; s.n_chunks = q.n_chunks; s.state = d.state;
    switch (q.lanes) {
        case 1: run_backward<T, 1>(stream, p, s, q.at_once); break;
        case 2: run_backward<T, 2>(stream, p, s, q.at_once); break;
        case 4: run_backward<T, 4>(stream, p, s, q.at_once); break;
        case 8: run_backward<T, 8>(stream, p, s, q.at_once); break;
        case 16: run_backward<T, 16>(stream, p, s, q.at_once); break;
        default: run_backward<T, 32>(stream, p, s, q.at_once);
    }
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
    if (d == nullptr) return;
    if (d->dtype > BPL_BFLOAT16 || d->state < 1 || d->state > SCAN_MAX_STATE || d->groups < 1 || d->channels % d->groups != 0 ||
        d->tokens >= (1u << 31)) {
        set_status(BPL_ERR_ARGUMENT, "state_scan_backward: 1..128 states, channels a multiple of groups, fewer than 2^31 tokens");
        return;
    }
    bool given = true;
    if (d->channels > 0)
        for (int i : {2, 15, 22}) given &= buffers[i] != nullptr;
    if (d->channels > 0 && d->tokens > 0)
        for (int i : {0, 1, 3, 4, 10, 11, 13, 14}) given &= buffers[i] != nullptr;
    if (d->tokens > 0)
        for (int i : {16, 17}) given &= buffers[i] != nullptr;
    // a gradient where there is an operand
    const int pairs[4][2] = {{5, 18}, {6, 19}, {7, 20}, {9, 21}};
    for (const auto &io : pairs) given &= buffers[io[0]] == nullptr || buffers[io[1]] != nullptr;
    if (!given) {
        set_status(BPL_ERR_ARGUMENT, "state_scan_backward: null buffer");
        return;
    }
    if (!sequences_fit(*d, buffers[8])) {
        set_status(BPL_ERR_ARGUMENT, "state_scan_backward: 2^31 sequences, or sequences and their length are not the tokens");
        return;
    }
    if (d->channels == 0) {                // the sums over no channels
        const size_t bytes = static_cast<size_t>(d->tokens) * d->groups * d->state * (d->dtype == BPL_FLOAT ? 4 : 2);
        for (int i : {16, 17})
            if (bytes > 0 && cudaMemsetAsync(buffers[i], 0, bytes, stream) != cudaSuccess) break;
        launch_ok();
        return;
    }
    if (d->dtype == BPL_FLOAT) backward<float>(stream, buffers, *d);
    else if (d->dtype == BPL_HALF) backward<__half>(stream, buffers, *d);
    else backward<__nv_bfloat16>(stream, buffers, *d);
    launch_ok();
}
