// Leaky states whose decay and input are selected by the data, over packed sequences (no counterpart in brainpylib; the
// whole-sequence form of a leaky update such as lif_exp_step's):
//
//     dt = delta + bias (through the softplus if asked);  h[t, n] = exp(dt A[n]) h[t - 1, n] + dt x B[t, n]
//     y = sum_n C[t, n] h[t, n] + D x;  y = y * silu(z) if there is a gate
//
// for every channel on its own; channels of a group share B and C.
#include "state_scan.cuh"

namespace bpl {
namespace {

constexpr uint32_t SLICE = SCAN_TILE_TOKENS, TILE = 2 * SLICE;  // tokens that a warp walks at once, tokens staged at once
__host__ __device__ constexpr int walkers(int lanes) { return lanes == 1 ? 64 : 128; }

// Shared memory of a block.  Tiles arrive as they lie in memory in a ring of copies, are turned to floats two tiles deep, and
// leave as sums two tiles deep: one barrier a tile.
template<typename T, int LANES>
struct ScanShared {
    // (rows of sums apart by banks, and at even places: they are read as pairs)
    static constexpr int WALKERS = walkers(LANES), CPB = WALKERS / LANES, NP = NS * LANES, Y_ROW = CPB + (LANES < 32 ? 32 / LANES : 2);
    static_assert(CPB % 2 == 0 && NP % 2 == 0 && Y_ROW % 2 == 0 && sizeof(T) * CPB * TILE % 16 == 0 && sizeof(T) * NP * TILE % 16 == 0,
                  "alignment of pairs and copies");
    // the tiles read out, walked and turned, and two on their way (one where B and C of 128 floats fill the memory)
    static constexpr int RING = sizeof(T) * NP > 256 ? 4 : 5;
    struct Raw {
        T x[TILE][CPB], delta[TILE][CPB], z[TILE][CPB];
        alignas(16) T B[TILE][NP], C[TILE][NP];             // (walked as they are)
    } raw[RING];
    float step[2][TILE][CPB][2];                             // dt, dt x
    float y[2][TILE][Y_ROW];
    int odd[2][CREW / 32];                                   // whether a time or an input is no finite number, by turning warps
};
template<typename T, int LANES>
constexpr bool fits = sizeof(ScanShared<T, LANES>) <= 227 * 1024;

// A lane holds NS neighbouring states of a channel in registers (as pairs) and walks the tokens; LANES lanes share a channel.
// Its floor are the exponentials, one for every token, channel and state, 16 of them per clock and SM (16,384 tokens of 4096 channels, 16
// states: 231 us); it takes 725, as a walking warp's token takes 87 clocks where its exponentials take 32: with 128 blocks there is one
// walking warp to a scheduler, which waits for its own instructions (issue slots taken 52 %, exponentials' pipe 36 %).  Measured and
// slower: half of the decays as polynomials (the arithmetic pipe has no room), two states a lane and eight lanes (928 us against 836
// then), two warps in turn on one channel (884), loads a group ahead by hand (1200 and more: spills).
// ENDS: only the state that a chunk leaves behind when it starts from zero, and the time that passes in it.
// PADDED: lanes hold more states than there are.  Those stay zero, as their rates, inputs and read-outs are, but for an infinite time or
// input, which times 0 is no number: tiles with such go the way of the bounds, where the states are cleared.  (A form of its own, as
// the walk with full lanes took 3 to 8 % longer with the same conditions in its text; with padded ones they cost 1 to 4 %, 8192 tokens of
// 4096 channels, 10 states: 395 to 406 us, and 9 % with 50 states in 16 bits.)
template<typename T, int LANES, bool ENDS, bool PADDED>
__global__ void __launch_bounds__(walkers(LANES) + CARRIERS, 2)
state_scan_kernel(const ScanArgs<T> p) {
    using Shared = ScanShared<T, LANES>;
    constexpr int CPB = Shared::CPB, NP = Shared::NP, PAIRS = NS / 2, RING = Shared::RING, WALKERS = Shared::WALKERS;
    constexpr int K = LANES < static_cast<int>(SLICE) ? LANES : static_cast<int>(SLICE);
    extern __shared__ __align__(16) unsigned char raw_shared[];
    Shared &sh = *reinterpret_cast<Shared *>(raw_shared);

    const bool walker = threadIdx.x < WALKERS;
    const uint32_t tid = walker ? threadIdx.x : threadIdx.x - WALKERS, local = tid / LANES, part = tid % LANES;
    const uint32_t group = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles, k_chunk = blockIdx.y;
    const uint32_t c_first = tile * CPB, c_count = min(static_cast<uint32_t>(CPB), p.per_group - c_first);
    const uint32_t c0 = group * p.per_group + c_first;               // first channel of the block
    const uint32_t channel = c0 + local;
    const bool valid = walker && local < c_count;
    const uint32_t n0 = part * NS;
    const Sequences seq = p.seq;
    const uint32_t first = seq.first(), last = seq.last();

    uint32_t from = k_chunk * p.chunk;
    const uint32_t to = min(from + p.chunk, seq.tokens);
    if (ENDS) {                       // only where the sequence at the chunk's end goes on behind it
        if (to >= last || to <= first || k_chunk + 1 >= p.n_chunks) return;
        const uint32_t begin = seq.begin(seq.of(to));
        if (begin >= to) return;
        if (begin > from) from = begin / TILE * TILE;
    }
    const uint32_t live_from = max(from, first), live_to = min(to, last);
    const uint32_t n_tiles = to > from ? (to - from + TILE - 1) / TILE : 0;

    // ---- the parts of a tile's way
    auto request = [&](uint32_t i, uint32_t place) {                // tile i into the ring, by two warps
        if (i < n_tiles) {
            typename Shared::Raw &r = sh.raw[place];
            const uint32_t tb = from + i * TILE;
            if (tid / 32 == 2) {
                fetch<TILE>(r.x, p.x + c0, p.x_stride, tb, live_from, live_to, c_count, p.row_copy);
                if (!ENDS && p.z != nullptr) fetch<TILE>(r.z, p.z + c0, p.z_stride, tb, live_from, live_to, c_count, p.row_copy);
            } else {
                fetch<TILE>(r.delta, p.delta + c0, p.delta_stride, tb, live_from, live_to, c_count, p.row_copy);
                fetch<TILE>(r.B, p.B + group * p.B_group, p.B_stride, tb, live_from, live_to, p.state, p.state_copy);
                if (!ENDS) fetch<TILE>(r.C, p.C + group * p.C_group, p.C_stride, tb, live_from, live_to, p.state, p.state_copy);
            }
        }
        copies_commit();
    };
    // 64 threads turn, 64 request and read out; each always the same two neighbouring channels
    const bool turner = !walker && tid < CREW;
    const uint32_t mate = tid % CREW, e2 = mate % (CPB / 2) * 2, j2 = mate / (CPB / 2);
    constexpr uint32_t J_STEP = CREW / (CPB / 2);
    static_assert(CPB / 2 <= static_cast<int>(CREW) && CREW % (CPB / 2) == 0, "a row for every crew");
    const bool has0 = e2 < c_count, has1 = e2 + 1 < c_count;
    pair bias = 0, D = 0;
    if (p.bias != nullptr) bias = make_pair(has0 ? p.bias[c0 + e2] : 0.0f, has1 ? p.bias[c0 + e2 + 1] : 0.0f);
    if (!ENDS && p.D != nullptr) D = make_pair(has0 ? p.D[c0 + e2] : 0.0f, has1 ? p.D[c0 + e2 + 1] : 0.0f);
    // (both without branches around the arithmetic, and all loads in front of all stores, which might else be of the same place for
    // all that the compiler knows: so a thread's tokens run side by side.  What lies in the ring for a token or a channel that is
    // not there is computed with and dropped.)
    constexpr uint32_t TURNS = J_STEP > TILE ? 1 : TILE / J_STEP;
    auto turn = [&](uint32_t i, uint32_t place) {
        if (i >= n_tiles) return;
        typename Shared::Raw &r = sh.raw[place];
        const uint32_t tb = from + i * TILE;
        pair dt[TURNS], in[TURNS];
        const bool at_work = J_STEP <= TILE || j2 < TILE;
#pragma unroll
        for (uint32_t q = 0; q < TURNS; ++q) {
            dt[q] = at_work ? load_pair(&r.delta[j2 + q * J_STEP][e2]) : 0;
            in[q] = at_work ? load_pair(&r.x[j2 + q * J_STEP][e2]) : 0;
        }
#pragma unroll
        for (uint32_t q = 0; q < TURNS; ++q) dt[q] = add2(dt[q], bias);
        if (p.softplus)
#pragma unroll
            for (uint32_t q = 0; q < TURNS; ++q) dt[q] = softplus_pair(dt[q]);
#pragma unroll
        for (uint32_t q = 0; q < TURNS; ++q) in[q] = mul2(dt[q], in[q]);
        if (at_work)
#pragma unroll
            for (uint32_t q = 0; q < TURNS; ++q) {
                const uint32_t j = j2 + q * J_STEP, t = tb + j;
                const bool live = t >= live_from && t < live_to;
                const float2 d = split(dt[q]), u = split(in[q]);
                const float d0 = live && has0 ? d.x : 0.0f, u0 = live && has0 ? u.x : 0.0f;
                const float d1 = live && has1 ? d.y : 0.0f, u1 = live && has1 ? u.y : 0.0f;
                *reinterpret_cast<float4 *>(sh.step[i & 1][j][e2]) = make_float4(d0, u0, d1, u1);
            }
        if constexpr (PADDED) {          // (read back: kept in registers it took 4 to 9 % longer with 10 states)
            bool odd = false;
            if (at_work)
#pragma unroll 1
                for (uint32_t q = 0; q < TURNS; ++q) {
                    const float4 v = *reinterpret_cast<const float4 *>(sh.step[i & 1][j2 + q * J_STEP][e2]);
                    odd |= !(fmaxf(fabsf(v.x), fabsf(v.z)) < INFINITY && fmaxf(fabsf(v.y), fabsf(v.w)) < INFINITY);
                }
            odd = __any_sync(FULL_MASK, odd);
            if (tid % 32 == 0) sh.odd[i & 1][tid / 32] = odd;
        }
        // states that are not there, and tokens: zeros for B and C
        if (p.state < NP || tb < live_from || tb + TILE > live_to)
            for (uint32_t k = mate; k < TILE * NP; k += CREW) {
                const uint32_t j = k / NP, n = k % NP, t = tb + j;
                if (n < p.state && t >= live_from && t < live_to) continue;
                r.B[j][n] = from_float<T>(0.0f);
                r.C[j][n] = from_float<T>(0.0f);
            }
    };
    // the sums of the tile's tokens, skip and gate, one rounding
    const bool store_pairs = (p.channels & 1u) == 0 && (c0 & 1u) == 0 && p.y_pairs;
    auto read_out = [&](uint32_t i, uint32_t place) {
        const typename Shared::Raw &r = sh.raw[place];
        const uint32_t tb = from + i * TILE;
        if (J_STEP > TILE && j2 >= TILE) return;
        pair y[TURNS];
        float2 z[TURNS];
#pragma unroll
        for (uint32_t q = 0; q < TURNS; ++q) {
            const uint32_t j = j2 + q * J_STEP;
            y[q] = load_pair(&sh.y[i & 1][j][e2]);
            if (p.D != nullptr) y[q] = fma2(D, load_pair(&r.x[j][e2]), y[q]);
            if (p.z != nullptr) z[q] = split(load_pair(&r.z[j][e2]));
        }
        if (p.z != nullptr)
#pragma unroll
            for (uint32_t q = 0; q < TURNS; ++q) y[q] = mul2(y[q], make_pair(silu(z[q].x), silu(z[q].y)));
        T *at = p.y + static_cast<size_t>(tb + j2) * p.channels + c0 + e2;
#pragma unroll
        for (uint32_t q = 0; q < TURNS; ++q, at += static_cast<size_t>(J_STEP) * p.channels) {
            const uint32_t t = tb + j2 + q * J_STEP;
            const bool live = t >= live_from && t < live_to;
            const float2 v = split(y[q]), w = make_float2(live ? v.x : 0.0f, live ? v.y : 0.0f);
            if (t < to) {
                if (store_pairs && has1) {
                    store_pair(at, w);
                } else {
                    if (has0) at[0] = from_float<T>(w.x);
                    if (has1) at[1] = from_float<T>(w.y);
                }
            }
        }
    };

    if (!walker && !turner)
#pragma unroll 1
        for (uint32_t i = 0; i < RING - 2; ++i) request(i, i);

    pair A2[PAIRS], h[PAIRS];
#pragma unroll
    for (int k = 0; k < PAIRS; ++k) {
        float a[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t n = n0 + 2 * k + i;
            a[i] = valid && n < p.state ? p.A[static_cast<size_t>(channel) * p.state + n] * LOG2_E : 0.0f;
        }
        A2[k] = make_pair(a[0], a[1]);
        h[k] = 0;
    }
    float time = 0.0f;

    const bool by_vectors = p.state % 4 == 0 && p.state_aligned;
    auto load_state = [&](const float *at) {       // at: the channel's states
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
            float v[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) v[i] = valid && n0 + 2 * k + i < p.state ? __ldcg(at + n0 + 2 * k + i) : 0.0f;
            h[k] = make_pair(v[0], v[1]);
        }
    };
    auto store_state = [&](float *at) {
        if (!valid) return;
        if (by_vectors) {
            const float2 a = split(h[0]), b = split(h[1]);
            if (n0 < p.state) *reinterpret_cast<float4 *>(at + n0) = make_float4(a.x, a.y, b.x, b.y);
            return;
        }
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
            const float2 v = split(h[k]);
            if (n0 + 2 * k < p.state) at[n0 + 2 * k] = v.x;
            if (n0 + 2 * k + 1 < p.state) at[n0 + 2 * k + 1] = v.y;
        }
    };
    auto zero_state = [&]() {
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) h[k] = 0;
    };
    auto state_of = [&](uint32_t row) { return (static_cast<size_t>(row) * p.channels + channel) * p.state; };

    auto only_there = [&](pair v, int k) {
        const float2 f = split(v);
        return make_pair(n0 + 2 * k < p.state ? f.x : 0.0f, n0 + 2 * k + 1 < p.state ? f.y : 0.0f);
    };

    // the state that reaches the chunk's first live token from the chunks in front
    uint32_t s = seq.count, s_begin = 0, s_end = 0;  // and the sequence that it stands in
    if (live_from < live_to) {
        s = seq.of(live_from);
        s_begin = seq.begin(s);
        s_end = seq.end(s);
        if (!ENDS && walker && s_begin < live_from) {
            for (uint32_t j = s_begin / p.chunk; j < k_chunk; ++j) {
                const float passed = valid ? __ldcg(p.chunk_time + static_cast<size_t>(j) * p.channels + channel) : 0.0f;
                const pair dt = make_pair(passed, passed);
                pair keep[PAIRS];
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) keep[k] = h[k];
                load_state(p.chunk_state + state_of(j));
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) h[k] = add2(through_chunk(keep[k], mul2(dt, A2[k])), h[k]);
                if constexpr (PADDED)
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) h[k] = only_there(h[k], k);
            }
        }
    }

    // what a token brings: the decay and the input of every state, and its read-out
    struct Token {
        pair keep[PAIRS], in[PAIRS], c[PAIRS];
        float time;
    };
    auto token = [&](uint32_t i, uint32_t j, uint32_t place) {
        Token k;
        const float2 d = *reinterpret_cast<const float2 *>(sh.step[i & 1][j][local]);
        const pair dt = make_pair(d.x, d.x), in = make_pair(d.y, d.y);
        k.time = d.x;
        pair b[PAIRS];
        load_states(&sh.raw[place].B[j][n0], b);
        if (!ENDS) load_states(&sh.raw[place].C[j][n0], k.c);
#pragma unroll
        for (int q = 0; q < PAIRS; ++q) {
            k.keep[q] = decay_pair(dt, A2[q]);
            k.in[q] = mul2(in, b[q]);
        }
        return k;
    };
    auto step = [&](const Token &k, auto bounded) -> float {
        pair y = 0;
#pragma unroll
        for (int q = 0; q < PAIRS; ++q) {
            h[q] = fma2(h[q], k.keep[q], k.in[q]);
            if constexpr (PADDED && decltype(bounded)::value) h[q] = only_there(h[q], q);
            if (!ENDS) y = q == 0 ? mul2(h[q], k.c[q]) : fma2(h[q], k.c[q], y);
        }
        return ENDS ? k.time : sum2(y);
    };
    // Tokens inside one sequence.  The chain of states is short; what takes long are loads, exponentials and the exchange of sums
    // between lanes.  So a token's work stands beside that of the token K further on, whose exponentials are under way meanwhile,
    // and a group's sums are exchanged while the next group is walked.
    auto walk = [&](uint32_t i, uint32_t j0, uint32_t place) {
        constexpr uint32_t GROUPS = SLICE / K;
        float passed = 0.0f, sums[GROUPS], y[2][K];
        Token at[2][K];
#pragma unroll
        for (int q = 0; q < K; ++q) at[0][q] = token(i, j0 + q, place);
#pragma unroll
        for (uint32_t g = 0; g <= GROUPS; ++g) {
            if (g > 0 && !ENDS) sums[g > 0 ? g - 1 : 0] = sum_over_lanes<K, LANES>(y[(g + 1) & 1], part);
            if (g < GROUPS)
#pragma unroll
                for (int q = 0; q < K; ++q) {
                    if (g + 1 < GROUPS) at[(g + 1) & 1][q] = token(i, j0 + (g + 1) * K + q, place);
                    y[g & 1][q] = step(at[g & 1][q], std::false_type());
                    passed += y[g & 1][q];
                }
        }
        if (ENDS) time += passed;              // (summed by slices: a long run's time keeps its precision)
        // written at the end: a store in between would keep the loads behind it from starting early
        if (!ENDS && (LANES == K || part < K))
#pragma unroll
            for (uint32_t g = 0; g < GROUPS; ++g) sh.y[i & 1][j0 + g * K + part % K][local] = sums[g];
    };
    auto walk_bounds = [&](uint32_t i, uint32_t j0, uint32_t tb, uint32_t place) {   // tokens that sequences begin or end in
        float passed = 0.0f;
#pragma unroll 1
        for (uint32_t j = j0; j < j0 + SLICE; ++j) {
            const uint32_t t = tb + j;
            if (t < live_from || t >= live_to) continue;
            if (t == s_begin) {
                time = passed = 0.0f;
                if (p.initial != nullptr) load_state(p.initial + state_of(s));
                else zero_state();
            }
            float y = step(token(i, j, place), std::true_type());
            if (ENDS) {
                passed += y;
            } else {
                y = sum_over_lanes<K, LANES>(y);
                if (part == 0) sh.y[i & 1][j][local] = y;
            }
            if (t + 1 >= s_end) {
                if (!ENDS && p.last != nullptr) store_state(p.last + state_of(s));
                while (++s < seq.count && (s_end = seq.end(s)) <= t + 1) {}
                s_begin = s < seq.count ? seq.begin(s) : 0xffffffffu;
                if (s >= seq.count) s_end = 0xffffffffu;
            }
        }
        if (ENDS) time += passed;
    };

    if (!walker) copies_wait<RING - 4>();        // tiles 0 and 1 are there
    __syncthreads();
    if (turner) turn(0, 0);
    __syncthreads();
    uint32_t before = RING - 1, here = 0, next = 1, ahead = RING - 2;      // places in the ring of tiles i - 1, i, i + 1, i + RING - 2
    for (uint32_t i = 0; i <= n_tiles; ++i) {
        if (walker) {
            const uint32_t tb = from + i * TILE;
            bool odd = false;
            if constexpr (PADDED) odd = i < n_tiles && (sh.odd[i & 1][0] | sh.odd[i & 1][1]) != 0;
#pragma unroll 1
            for (uint32_t j0 = 0; j0 < TILE && tb + j0 < to && i < n_tiles; j0 += SLICE) {
                if (!ENDS && p.saved != nullptr) store_state(p.saved + state_of((tb + j0) / SLICE));
                if (!odd && tb + j0 >= live_from && s_begin < tb + j0 && s_end > tb + j0 + SLICE && tb + j0 + SLICE <= live_to)
                    walk(i, j0, here);
                else
                    walk_bounds(i, j0, tb, here);
            }
        } else if (turner) {
            turn(i + 1, next);
        } else {
            request(i + RING - 2, ahead);       // into the place of tile i - 2, which has been read out
            if (!ENDS && i > 0) read_out(i - 1, before);
            copies_wait<RING - 4>();            // tile i + 2 is there
        }
        __syncthreads();
        before = here;
        here = next;
        next = next + 1 == RING ? 0 : next + 1;
        ahead = ahead + 1 == RING ? 0 : ahead + 1;
    }

    if (ENDS) {
        store_state(p.chunk_state + state_of(k_chunk));
        if (valid && part == 0) p.chunk_time[static_cast<size_t>(k_chunk) * p.channels + channel] = time;
    } else if (p.last != nullptr) {           // sequences without a token leave the state they came with
        for (uint32_t q = k_chunk; q < seq.count; q += p.n_chunks) {
            if (seq.end(q) > seq.begin(q)) continue;
            if (p.initial != nullptr) load_state(p.initial + state_of(q));
            else zero_state();
            store_state(p.last + state_of(q));
        }
    }
}

// ---- one token per running sequence ----------------------------------------------------------------------------------
struct StepArgs {
    const void *x, *delta, *z, *B, *C;
    const float *A, *D, *bias;
    const int *slots;
    float *state;
    void *y;
    long long x_stride, delta_stride, z_stride, B_stride, B_group, C_stride, C_group;
    uint32_t rows, pool, channels, per_group, n, tiles;
    bool softplus, vector, pairs;         // vector: four states at once; pairs: two of B and C
};

constexpr int STEP_THREADS = 128;

// The state of a row, -1 for padding, -2 for one behind the pool.
__device__ __forceinline__ int slot_of(const StepArgs &p, const uint32_t row) {
    const int slot = p.slots != nullptr ? p.slots[row] : static_cast<int>(row);
    return slot < 0 ? -1 : slot >= static_cast<int>(p.pool) ? -2 : slot;
}
// Whether an earlier row has the same state; by the whole block, with a barrier.
__device__ __forceinline__ bool taken(const StepArgs &p, const uint32_t row, const int slot) {
    bool mine = false;
    if (p.slots != nullptr)
        for (uint32_t i = threadIdx.x; i < row; i += STEP_THREADS) mine |= p.slots[i] == slot;
    return __syncthreads_or(mine) != 0;
}

__device__ __forceinline__ float4 load_four(const float *at, uint32_t n0, uint32_t n, bool vector) {
    if (vector) return *reinterpret_cast<const float4 *>(at + n0);
    return make_float4(at[n0], n0 + 1 < n ? at[n0 + 1] : 0.0f, n0 + 2 < n ? at[n0 + 2] : 0.0f, n0 + 3 < n ? at[n0 + 3] : 0.0f);
}
__device__ __forceinline__ void store_four(float *at, uint32_t n0, uint32_t n, bool vector, float4 v) {
    if (vector) {
        *reinterpret_cast<float4 *>(at + n0) = v;
        return;
    }
    at[n0] = v.x;
    if (n0 + 1 < n) at[n0 + 1] = v.y;
    if (n0 + 2 < n) at[n0 + 2] = v.z;
    if (n0 + 3 < n) at[n0 + 3] = v.w;
}
// four states through one token, of which `there` are; their part of the read-out (an infinite time or input times 0 is no number:
// states that are not there are cleared)
__device__ __forceinline__ float step_four(float4 &h, const float4 A, const float4 B, const float4 C, float dt, float in, uint32_t there) {
    h.x = fmaf(h.x, decay(dt, A.x * LOG2_E), in * B.x);
    h.y = there > 1 ? fmaf(h.y, decay(dt, A.y * LOG2_E), in * B.y) : 0.0f;
    h.z = there > 2 ? fmaf(h.z, decay(dt, A.z * LOG2_E), in * B.z) : 0.0f;
    h.w = there > 3 ? fmaf(h.w, decay(dt, A.w * LOG2_E), in * B.w) : 0.0f;
    return fmaf(h.x, C.x, h.y * C.y) + fmaf(h.z, C.z, h.w * C.w);
}

// four neighbouring operands of a row
template<typename T>
__device__ __forceinline__ float4 row_four(const T *at, uint32_t n0, uint32_t n, bool pairs) {
    if (pairs) {
        const float2 a = split(load_pair(at + n0)), b = split(load_pair(at + n0 + 2));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return make_float4(to_float(at[n0]), n0 + 1 < n ? to_float(at[n0 + 1]) : 0.0f, n0 + 2 < n ? to_float(at[n0 + 2]) : 0.0f,
                       n0 + 3 < n ? to_float(at[n0 + 3]) : 0.0f);
}
// the read-out of a channel as it is written
template<typename T>
__device__ __forceinline__ void store_step(const StepArgs &p, uint32_t row, uint32_t channel, int slot, float sum, float x, float z, float D) {
    if (p.D != nullptr) sum = fmaf(D, x, sum);
    if (p.z != nullptr) sum *= silu(z);
    static_cast<T *>(p.y)[static_cast<size_t>(row) * p.channels + channel] =
        from_float<T>(slot >= 0 ? sum : slot == -1 ? 0.0f : __int_as_float(0x7fffffff));
}

// In both kernels a state is read before it is known whether an earlier row takes it (what is read then is dropped, and nothing is
// written): two latencies of memory in a row instead of three.

// LANES lanes to a channel, Q times four states to a lane (neighbouring lanes read neighbouring ones).  Few channels and rows: Q = 1, so
// that all loads of a call are on their way at once (one row of 2048 channels, 16 states: 2.3 us on the device).  Many, of more than 16
// states: Q = 2, as every lane computes time step and gate (64 rows of 4096 channels, 128 states: Q = 1 102 us, 2 82, 4 96; 64 states:
// 45, 40, 41, 3.4 TB/s).
template<typename T, int LANES, int Q>
__global__ void __launch_bounds__(STEP_THREADS)
state_scan_step_kernel(const StepArgs p) {
    constexpr uint32_t CPB = STEP_THREADS / LANES;
    const uint32_t row = blockIdx.y, part = threadIdx.x % LANES, channel = blockIdx.x * CPB + threadIdx.x / LANES;
    const bool valid = channel < p.channels;
    int slot = slot_of(p, row);
    float x = 0.0f, dt = 0.0f, z = 0.0f, D = 0.0f;
    if (valid) {
        x = to_float(static_cast<const T *>(p.x)[row * p.x_stride + channel]);
        dt = to_float(static_cast<const T *>(p.delta)[row * p.delta_stride + channel]) + (p.bias != nullptr ? p.bias[channel] : 0.0f);
        if (p.z != nullptr) z = to_float(static_cast<const T *>(p.z)[row * p.z_stride + channel]);
        if (p.D != nullptr) D = p.D[channel];
    }
    const T *B = static_cast<const T *>(p.B) + row * p.B_stride + channel / p.per_group * p.B_group;
    const T *C = static_cast<const T *>(p.C) + row * p.C_stride + channel / p.per_group * p.C_group;
    float *at = p.state + (static_cast<size_t>(max(slot, 0)) * p.channels + channel) * p.n;
    float4 A[Q], b[Q], c[Q], h[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const uint32_t n0 = (part + q * LANES) * 4;
        if (!valid || n0 >= p.n) continue;
        A[q] = load_four(p.A + static_cast<size_t>(channel) * p.n, n0, p.n, p.vector);
        b[q] = row_four(B, n0, p.n, p.pairs);
        c[q] = row_four(C, n0, p.n, p.pairs);
        if (slot >= 0) h[q] = load_four(at, n0, p.n, p.vector);
    }
    if (taken(p, row, slot) && slot >= 0) slot = -2;
    if (p.softplus) dt = softplus(dt);
    float sum = 0.0f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const uint32_t n0 = (part + q * LANES) * 4;
        if (!valid || n0 >= p.n || slot < 0) continue;
        sum += step_four(h[q], A[q], b[q], c[q], dt, dt * x, p.n - n0);
        store_four(at, n0, p.n, p.vector, h[q]);
    }
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) sum += __shfl_xor_sync(FULL_MASK, sum, m);
    if (valid && part == 0) store_step<T>(p, row, channel, slot, sum, x, z, D);
}

// Many channels and rows of at most 16 states: a thread to a channel, so that time step and gate are computed once; the row's B and C
// stand in shared memory.  Bound by memory: a state is read and written once (250 rows of 4096 channels, 16 states: 33 us on the
// device, 4 TB/s; two rows a thread 36, four 41, lanes of four states 47).
constexpr uint32_t ROWS_MAX_STATE = 16;

template<typename T>
__global__ void __launch_bounds__(STEP_THREADS)
state_scan_step_rows_kernel(const StepArgs p) {
    __shared__ __align__(16) float s_B[ROWS_MAX_STATE], s_C[ROWS_MAX_STATE];
    const uint32_t row = blockIdx.y, group = blockIdx.x / p.tiles, in_group = blockIdx.x % p.tiles * STEP_THREADS + threadIdx.x;
    const uint32_t channel = group * p.per_group + in_group;
    const bool valid = in_group < p.per_group;
    int slot = slot_of(p, row);
    float x = 0.0f, dt = 0.0f, z = 0.0f, D = 0.0f;
    if (valid) {
        x = to_float(static_cast<const T *>(p.x)[row * p.x_stride + channel]);
        dt = to_float(static_cast<const T *>(p.delta)[row * p.delta_stride + channel]) + (p.bias != nullptr ? p.bias[channel] : 0.0f);
        if (p.z != nullptr) z = to_float(static_cast<const T *>(p.z)[row * p.z_stride + channel]);
        if (p.D != nullptr) D = p.D[channel];
    }
    if (threadIdx.x < 2 * ROWS_MAX_STATE) {
        const uint32_t n = threadIdx.x % ROWS_MAX_STATE;
        const bool of_B = threadIdx.x < ROWS_MAX_STATE;
        const T *from = of_B ? static_cast<const T *>(p.B) + row * p.B_stride + group * p.B_group
                             : static_cast<const T *>(p.C) + row * p.C_stride + group * p.C_group;
        (of_B ? s_B : s_C)[n] = n < p.n ? to_float(from[n]) : 0.0f;
    }
    const float *A = p.A + static_cast<size_t>(channel) * p.n;
    float *at = p.state + (static_cast<size_t>(max(slot, 0)) * p.channels + channel) * p.n;
    float4 h[ROWS_MAX_STATE / 4], rate[ROWS_MAX_STATE / 4];
#pragma unroll
    for (uint32_t n0 = 0; n0 < ROWS_MAX_STATE; n0 += 4) {
        if (!valid || n0 >= p.n) continue;
        rate[n0 / 4] = load_four(A, n0, p.n, p.vector);
        if (slot >= 0) h[n0 / 4] = load_four(at, n0, p.n, p.vector);
    }
    if (taken(p, row, slot) && slot >= 0) slot = -2;      // (and its barrier stands between B, C and their use)
    if (!valid) return;
    if (p.softplus) dt = softplus(dt);
    float sum = 0.0f;
#pragma unroll
    for (uint32_t n0 = 0; n0 < ROWS_MAX_STATE; n0 += 4) {
        if (slot < 0 || n0 >= p.n) continue;
        sum += step_four(h[n0 / 4], rate[n0 / 4], *reinterpret_cast<const float4 *>(s_B + n0), *reinterpret_cast<const float4 *>(s_C + n0),
                         dt, dt * x, p.n - n0);
        store_four(at, n0, p.n, p.vector, h[n0 / 4]);
    }
    store_step<T>(p, row, channel, slot, sum, x, z, D);
}

// ---- launches --------------------------------------------------------------------------------------------------------
const bpl_state_scan_descriptor *checked(const char *opaque, size_t opaque_len, const char *what) {
    const auto *d = unpack<bpl_state_scan_descriptor>(opaque, opaque_len);
    if (d == nullptr) return nullptr;
    if (d->dtype > BPL_BFLOAT16 || d->state < 1 || d->state > SCAN_MAX_STATE || d->groups < 1 || d->channels % d->groups != 0 ||
        d->tokens >= (1u << 31)) {
        set_status(BPL_ERR_ARGUMENT, what);
        return nullptr;
    }
    return d;
}

}  // namespace

StateScanPlan plan_state_scan(const bpl_state_scan_descriptor &d) {
    StateScanPlan q;
    q.lanes = lanes_for(d.state);
    const uint32_t per_block = walkers(q.lanes) / q.lanes, per_group = d.channels / d.groups;
    q.tiles = (per_group + per_block - 1) / per_block;
    // The pass in front, over all chunks but one, costs half of the main one, so tokens are cut into chunks only where the channels
    // fill less than two thirds of the SMs: then to two blocks for an SM (8192 packed tokens of 2048 channels: one chunk 399 us,
    // four 195, nine 221; 16,384 tokens of 4096 channels: one chunk 757, two 844).  No chunk is shorter than 64 tokens.  (Shared memory
    // has room for two blocks with 9 to 128 states, in 32 bits with 9 to 64; elsewhere an SM walks its two one after the other.)
    const uint64_t blocks = static_cast<uint64_t>(q.tiles) * d.groups, sms = sm_count(), most = (d.tokens + 63) / 64;
    uint64_t chunks = blocks == 0 || blocks * 3 > sms * 2 ? 1 : 2 * sms / blocks;
    chunks = chunks > most ? most : chunks;
    if (chunks < 1) chunks = 1;
    const uint64_t chunk = (d.tokens + chunks - 1) / chunks;
    q.chunk = static_cast<uint32_t>((chunk + TILE - 1) / TILE * TILE);
    if (q.chunk == 0) q.chunk = TILE;
    q.n_chunks = (d.tokens + q.chunk - 1) / q.chunk;
    if (q.n_chunks < 1) q.n_chunks = 1;
    return q;
}

size_t state_scan_workspace_bytes(const char *opaque, size_t opaque_len) {
    if (opaque == nullptr || opaque_len != sizeof(bpl_state_scan_descriptor)) return 0;
    const auto &d = *reinterpret_cast<const bpl_state_scan_descriptor *>(opaque);
    if (d.state < 1 || d.state > SCAN_MAX_STATE || d.groups < 1) return 0;
    const StateScanPlan q = plan_state_scan(d);
    return q.n_chunks > 1 ? sizeof(float) * q.n_chunks * static_cast<size_t>(d.channels) * (d.state + 1) : 0;
}

namespace {

template<typename T, int LANES, bool ENDS, bool PADDED>
bool launch(cudaStream_t stream, const ScanArgs<T> &p, uint32_t groups) {
    constexpr unsigned bytes = sizeof(ScanShared<T, LANES>);
    static_assert(fits<T, LANES>, "shared memory of a block");
    if (!allow_shared<state_scan_kernel<T, LANES, ENDS, PADDED>>(bytes)) {
        set_status(BPL_ERR_CUDA, "state_scan: shared memory");
        return false;
    }
    state_scan_kernel<T, LANES, ENDS, PADDED><<<dim3(p.tiles * groups, p.n_chunks), walkers(LANES) + CARRIERS, bytes, stream>>>(p);
    return true;
}

template<typename T, int LANES>
void run_scan(cudaStream_t stream, const ScanArgs<T> &p, uint32_t groups) {
    if (p.n_chunks > 1 && !launch<T, LANES, true, false>(stream, p, groups)) return;
    if (p.state < NS * LANES) launch<T, LANES, false, true>(stream, p, groups);
    else launch<T, LANES, false, false>(stream, p, groups);
}

template<typename T>
void scan(cudaStream_t stream, void **b, const bpl_state_scan_descriptor &d) {
    const StateScanPlan q = plan_state_scan(d);
    ScanArgs<T> p = {};
    p.x = static_cast<const T *>(b[0]);
    p.delta = static_cast<const T *>(b[1]);
    p.A = static_cast<const float *>(b[2]);
    p.B = static_cast<const T *>(b[3]);
    p.C = static_cast<const T *>(b[4]);
    p.D = static_cast<const float *>(b[5]);
    p.z = static_cast<const T *>(b[6]);
    p.bias = static_cast<const float *>(b[7]);
    p.initial = static_cast<const float *>(b[9]);
    p.y = static_cast<T *>(b[10]);
    p.last = static_cast<float *>(b[11]);
    p.saved = static_cast<float *>(b[12]);
    p.chunk_state = static_cast<float *>(b[13]);
    p.chunk_time = p.chunk_state ? p.chunk_state + static_cast<size_t>(q.n_chunks) * d.channels * d.state : nullptr;
    p.x_stride = d.x_stride; p.delta_stride = d.delta_stride; p.z_stride = d.z_stride;
    p.B_stride = d.B_stride; p.B_group = d.B_group_stride; p.C_stride = d.C_stride; p.C_group = d.C_group_stride;
    p.seq = Sequences{static_cast<const int *>(b[8]), d.sequences, d.length, d.tokens};
    p.channels = d.channels; p.per_group = d.channels / d.groups; p.tiles = q.tiles; p.state = d.state;
    p.chunk = q.chunk; p.n_chunks = q.n_chunks; p.softplus = (d.flags & BPL_SCAN_SOFTPLUS) != 0;
    const uint32_t per_block = walkers(q.lanes) / q.lanes;
    p.row_copy = copy_bytes<T>({p.x, p.delta, p.z}, {d.x_stride, d.delta_stride, p.z ? d.z_stride : 0}, p.per_group);
    if (p.row_copy > per_block * sizeof(T)) p.row_copy = 4;
    p.state_copy = copy_bytes<T>({p.B, p.C}, {d.B_stride, d.C_stride, d.groups > 1 ? d.B_group_stride : 0, d.groups > 1 ? d.C_group_stride : 0},
                                 d.state);
    p.y_pairs = reinterpret_cast<uintptr_t>(p.y) % (2 * sizeof(T)) == 0;
    p.state_aligned = true;
    for (const void *a : {static_cast<const void *>(p.last), static_cast<const void *>(p.saved), static_cast<const void *>(p.chunk_state)})
        p.state_aligned &= aligned16(a);
    switch (q.lanes) {
        case 1: return run_scan<T, 1>(stream, p, d.groups);
        case 2: return run_scan<T, 2>(stream, p, d.groups);
        case 4: return run_scan<T, 4>(stream, p, d.groups);
        case 8: return run_scan<T, 8>(stream, p, d.groups);
        case 16: return run_scan<T, 16>(stream, p, d.groups);
        default: return run_scan<T, 32>(stream, p, d.groups);
    }
}

template<typename T, int LANES, int Q = 1>
void launch_step(cudaStream_t stream, const StepArgs &p) {
    constexpr uint32_t per_block = STEP_THREADS / LANES;
    state_scan_step_kernel<T, LANES, Q><<<dim3((p.channels + per_block - 1) / per_block, p.rows), STEP_THREADS, 0, stream>>>(p);
}

template<typename T>
void step(cudaStream_t stream, StepArgs p) {
    p.pairs = p.n % 4 == 0 && p.B_stride % 2 == 0 && p.C_stride % 2 == 0 &&
              (p.channels == p.per_group || (p.B_group % 2 == 0 && p.C_group % 2 == 0)) &&
              reinterpret_cast<uintptr_t>(p.B) % (2 * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(p.C) % (2 * sizeof(T)) == 0;
    // Many: 256 channels and rows for every SM (4096 channels, 16 states, a thread to a channel against lanes: 10 rows 3.85 us against
    // 3.6, 16 rows 4.4 against 4.6, 250 rows 33 against 47).
    if (static_cast<uint64_t>(p.channels) * p.rows >= 256ull * sm_count()) {
        if (p.n > 64) return launch_step<T, 16, 2>(stream, p);
        if (p.n > 32) return launch_step<T, 8, 2>(stream, p);
        if (p.n > ROWS_MAX_STATE) return launch_step<T, 4, 2>(stream, p);
        p.tiles = (p.per_group + STEP_THREADS - 1) / STEP_THREADS;
        const dim3 grid(p.tiles * (p.channels / p.per_group), p.rows);
        state_scan_step_rows_kernel<T><<<grid, STEP_THREADS, 0, stream>>>(p);
        return;
    }
    switch (lanes_for(p.n)) {
        case 1: return launch_step<T, 1>(stream, p);
        case 2: return launch_step<T, 2>(stream, p);
        case 4: return launch_step<T, 4>(stream, p);
        case 8: return launch_step<T, 8>(stream, p);
        case 16: return launch_step<T, 16>(stream, p);
        default: return launch_step<T, 32>(stream, p);
    }
}

bool all_given(void **b, std::initializer_list<int> which, const char *what) {
    for (int i : which)
        if (b[i] == nullptr) {
            set_status(BPL_ERR_ARGUMENT, what);
            return false;
        }
    return true;
}

}  // namespace
}  // namespace bpl

using namespace bpl;

extern "C" {

void state_scan(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "state_scan: 1..128 states, channels a multiple of groups, fewer than 2^31 tokens");
    if (d == nullptr || d->channels == 0) return;
    if ((d->tokens > 0 && !all_given(buffers, {0, 1, 3, 4, 10}, "state_scan: null buffer")) || !all_given(buffers, {2}, "state_scan: null buffer"))
        return;
    if (!sequences_fit(*d, buffers[8])) {
        set_status(BPL_ERR_ARGUMENT, "state_scan: 2^31 sequences, or sequences and their length are not the tokens");
        return;
    }
    if (d->sequences == 0 && d->tokens == 0) return;
    if (state_scan_workspace_bytes(opaque, opaque_len) > 0 && !all_given(buffers, {13}, "state_scan: no workspace")) return;
    if (d->dtype == BPL_FLOAT) scan<float>(stream, buffers, *d);
    else if (d->dtype == BPL_HALF) scan<__half>(stream, buffers, *d);
    else scan<__nv_bfloat16>(stream, buffers, *d);
    launch_ok();
}

void state_scan_step(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "state_scan_step: 1..128 states, channels a multiple of groups");
    if (d == nullptr || d->channels == 0 || d->tokens == 0) return;
    if (d->tokens > 65535 || d->sequences >= (1u << 31) || (buffers[8] == nullptr && d->sequences < d->tokens)) {
        set_status(BPL_ERR_ARGUMENT, "state_scan_step: at most 65535 rows, and a state for every row");
        return;
    }
    if (!all_given(buffers, {0, 1, 2, 3, 4, 10}, "state_scan_step: null buffer") ||
        (d->sequences > 0 && !all_given(buffers, {9}, "state_scan_step: null buffer")))
        return;
    StepArgs p = {};
    p.x = buffers[0]; p.delta = buffers[1]; p.A = static_cast<const float *>(buffers[2]); p.B = buffers[3]; p.C = buffers[4];
    p.D = static_cast<const float *>(buffers[5]); p.z = buffers[6]; p.bias = static_cast<const float *>(buffers[7]);
    p.slots = static_cast<const int *>(buffers[8]); p.state = static_cast<float *>(buffers[9]); p.y = buffers[10];
    p.x_stride = d->x_stride; p.delta_stride = d->delta_stride; p.z_stride = d->z_stride;
    p.B_stride = d->B_stride; p.B_group = d->B_group_stride; p.C_stride = d->C_stride; p.C_group = d->C_group_stride;
    p.rows = d->tokens; p.pool = d->sequences; p.channels = d->channels; p.per_group = d->channels / d->groups; p.n = d->state;
    p.softplus = (d->flags & BPL_SCAN_SOFTPLUS) != 0;
    p.vector = p.n % 4 == 0 && aligned16(p.state) && aligned16(p.A);
    if (d->dtype == BPL_FLOAT) step<float>(stream, p);
    else if (d->dtype == BPL_HALF) step<__half>(stream, p);
    else step<__nv_bfloat16>(stream, p);
    launch_ok();
}

}  // extern "C"
