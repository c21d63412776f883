// Linear attention with a decay for each head (no counterpart in brainpylib): the walk over whole sequences on the cores for
// 32-bit arithmetic, the gradients by the same walk (decay_attention.cuh), and the form for one new token per running sequence.
//
// The walk: a block holds 64 columns of a head's state in registers, thread (kk, vg) the rows 4 kk .. 4 kk + 3 (+ 64 m) and the columns
// 4 vg .. 4 vg + 3, and goes through the tokens one by one: three multiply-adds an element and token (as many as the same in chunks of
// 64 tokens would take), two neighbouring rows at a time, as k and q lie.  Tiles of 16 tokens are turned to floats in shared memory,
// the next one on its way in registers.  Read-outs of four tokens are summed over the 16 lanes of a column at once.  Bound by
// instructions: 140 a token and warp, 48 of them the multiply-adds (1501 tokens of 5 heads of 75 and 90 in 24 segments: 42 us a walk; rows one by
// one with their columns in pairs 57, as every k and q then had to be doubled).
//
// A single token: bound by memory, the state is read and written once (100 rows, 16 heads of 128: 42 us, 4.4 TB/s).
#include <initializer_list>
#include <type_traits>

#include "decay_attention.cuh"

namespace bpl {

SegmentPlan plan_segments(const bpl_decay_attention_descriptor &d, bool packed, uint64_t units, uint64_t wanted, uint32_t least) {
    SegmentPlan q = {d.tokens ? d.tokens : 1, 1, false};
    const uint64_t pieces = units ? wanted / units : 1;
    if (pieces <= 1 || d.tokens == 0) return q;
    if (!packed && d.sequences >= pieces) {               // whole sequences
        const uint64_t whole = (d.sequences + pieces - 1) / pieces * d.length;
        q.segment = whole < 1 || whole > d.tokens ? d.tokens : static_cast<uint32_t>(whole);
    } else {
        const uint64_t each = (d.tokens + pieces - 1) / pieces;
        q.segment = static_cast<uint32_t>(each < least ? least : (each + 63) / 64 * 64);
        q.crossing = packed || d.sequences == 0 || d.length % q.segment != 0 || d.length > q.segment;
    }
    q.segments = (d.tokens + q.segment - 1) / q.segment;
    if (q.segments <= 1) q.segments = 1, q.crossing = false;
    return q;
}

namespace {

constexpr int WALK_THREADS = 256;
constexpr uint32_t WALK_TOKENS = 16;        // of a tile
constexpr uint32_t COLUMNS = 64;            // of a block
constexpr int K_LANES = 16;                 // lanes that share a column

template<int M>
struct WalkShared {
    float k[2][WALK_TOKENS][64 * M], q[2][WALK_TOKENS][64 * M], v[2][WALK_TOKENS][COLUMNS];
};

// M: 64 M rows of the state at most; STATES: only what segments hand on.
template<typename T, int M, bool STATES>
__global__ __launch_bounds__(WALK_THREADS, M == 4 ? 1 : 2) void decay_walk_kernel(const DecayWalk p) {
    extern __shared__ __align__(16) unsigned char shared[];
    WalkShared<M> &s = *reinterpret_cast<WalkShared<M> *>(shared);
    constexpr uint32_t WIDTH = 64 * M;
    constexpr int LOADS = WALK_TOKENS * WIDTH / WALK_THREADS, V_LOADS = WALK_TOKENS * COLUMNS / WALK_THREADS;
    const uint32_t slabs = (p.v_size + COLUMNS - 1) / COLUMNS, h = blockIdx.x / slabs, c0 = blockIdx.x % slabs * COLUMNS;
    const uint32_t lane = threadIdx.x % 32, kk = lane % K_LANES, vg = threadIdx.x / K_LANES, g = blockIdx.y;
    const T *q_at = p.q.of<T>(h), *k_at = p.k.of<T>(h), *v_at = p.v.of<T>(h) + c0;
    const float a = decay_power(p.log_decay[h], 1);
    // the decay is off by up to 2^-25 of itself, which a state that lasts adds up token by token: every sixteenth one is chosen so that
    // all sixteen make the sixteenth power
    const float a16 = a > 0.5f ? static_cast<float>(exp(16.0 * static_cast<double>(p.log_decay[h]) - 15.0 * log(static_cast<double>(a)))) : a;
    pair state[2 * M][4] = {};              // rows 4 kk + 64 (i / 2) + 2 (i % 2) and the next one, columns
    const bool ragged = p.k_size != WIDTH;
    T k_next[LOADS], q_next[LOADS], v_next[V_LOADS];

    // (i: a pair of rows, o: one of them, j: a column)
    auto row_of = [&](int i, int o) { return 4 * kk + 64 * (i / 2) + 2 * (i % 2) + o; };
    auto for_states = [&](auto f) {
#pragma unroll
        for (int i = 0; i < 2 * M; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 v = split(state[i][j]);
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const uint32_t r = row_of(i, o), c = c0 + 4 * vg + j;
                    if (r < p.k_size && c < p.v_size) f(o ? v.y : v.x, r, c);
                }
            }
    };
    auto set_states = [&](auto f) {
#pragma unroll
        for (int i = 0; i < 2 * M; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float e[2];
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const uint32_t r = row_of(i, o), c = c0 + 4 * vg + j;
                    e[o] = r < p.k_size && c < p.v_size ? f(r, c) : 0.0f;
                }
                state[i][j] = make_pair(e[0], e[1]);
            }
    };
    // tokens from `t` up to `to` of the piece into registers, zeros behind them
    auto request = [&](uint32_t t, uint32_t to) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t at = threadIdx.x + i * WALK_THREADS, r = t + at / WIDTH, c = at % WIDTH;
            const bool there = r < to && c < p.k_size;
            const long long row = there ? p.seq.row(r) : 0;
            k_next[i] = there ? k_at[row * p.k.row + c] : from_float<T>(0.0f);
            if (!STATES) q_next[i] = there ? q_at[row * p.q.row + c] : from_float<T>(0.0f);
        }
#pragma unroll
        for (int i = 0; i < V_LOADS; ++i) {
            const uint32_t at = threadIdx.x + i * WALK_THREADS, r = t + at / COLUMNS, c = at % COLUMNS;
            const bool there = r < to && c0 + c < p.v_size;
            v_next[i] = there ? v_at[p.seq.row(r) * p.v.row + c] : from_float<T>(0.0f);
        }
    };
    // whether v has a number that is not finite
    auto put = [&](int buffer) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t at = threadIdx.x + i * WALK_THREADS;
            s.k[buffer][at / WIDTH][at % WIDTH] = to_float(k_next[i]);
            if (!STATES) s.q[buffer][at / WIDTH][at % WIDTH] = to_float(q_next[i]);
        }
#pragma unroll
        for (int i = 0; i < V_LOADS; ++i) {
            const uint32_t at = threadIdx.x + i * WALK_THREADS;
            const float v = to_float(v_next[i]) * p.state_scale;
            odd |= !(fabsf(v) < INFINITY);
            s.v[buffer][at / COLUMNS][at % COLUMNS] = v;
        }
        return odd && ragged;
    };
    auto write_out = [&](uint32_t row, uint32_t c, float v) {
        const size_t at = (static_cast<size_t>(row) * p.heads + h) * p.v_size + c;
        if (p.wide_out) static_cast<float *>(p.out)[at] = v;
        else static_cast<T *>(p.out)[at] = from_float<T>(v);
    };

    auto walk = [&](const Piece &piece) {
        const float *from = piece.begins ? (p.initial ? p.initial + (static_cast<size_t>(p.seq.state(piece.sequence)) * p.heads + h) * p.state_size() : nullptr)
                            : STATES ? nullptr : p.carried + (static_cast<size_t>(g - 1) * p.heads + h) * p.state_size();
        if (piece.begins) set_states([&](uint32_t r, uint32_t c) { return from ? from[p.state_at(r, c)] : 0.0f; });
        else set_states([&](uint32_t r, uint32_t c) { return from ? __ldcg(from + p.carried_at(r, c)) : 0.0f; });
        // backwards, a sequence's first state is the gradient of its last one: it has not decayed when the first token reads it
        float step = piece.begins && p.seq.backwards ? 1.0f : a;
        request(piece.from, piece.to);
        int buffer = 0;
        __syncthreads();                    // (the piece in front may still be read)
        bool careful = __syncthreads_or(put(buffer));
        // one token: state, and what it reads out; `careful`: rows that are not there stay out (zero times an infinite v is no number)
        auto token = [&](uint32_t j, float *out, auto careful_rows) {
            const float4 v4 = *reinterpret_cast<const float4 *>(&s.v[buffer][j][4 * vg]);
            const pair v[4] = {make_pair(v4.x, v4.x), make_pair(v4.y, v4.y), make_pair(v4.z, v4.z), make_pair(v4.w, v4.w)}, factor = make_pair(step, step);
            pair o[4] = {};
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const ulonglong2 k2 = *reinterpret_cast<const ulonglong2 *>(&s.k[buffer][j][4 * kk + 64 * m]);
                ulonglong2 q2 = {};
                if (!STATES) q2 = *reinterpret_cast<const ulonglong2 *>(&s.q[buffer][j][4 * kk + 64 * m]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const pair kp = i ? k2.y : k2.x, qp = i ? q2.y : q2.x;
                    const uint32_t r = row_of(2 * m + i, 0);
                    if (decltype(careful_rows)::value && r >= p.k_size) continue;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        pair &x = state[2 * m + i][c];
                        x = fma2(factor, x, mul2(kp, v[c]));
                        if (decltype(careful_rows)::value && r + 1 >= p.k_size) x = make_pair(split(x).x, 0.0f);
                        if (!STATES) o[c] = fma2(qp, x, o[c]);
                    }
                }
            }
            if (!STATES)
#pragma unroll
                for (int c = 0; c < 4; ++c) out[c] = sum2(o[c]);
        };
        for (uint32_t t0 = piece.from; t0 < piece.to; t0 += WALK_TOKENS) {
            const uint32_t n = min(WALK_TOKENS, piece.to - t0);
            if (t0 + WALK_TOKENS < piece.to) request(t0 + WALK_TOKENS, piece.to);
#pragma unroll 1
            for (uint32_t j0 = 0; j0 < n; j0 += 4) {
                float out[16] = {};         // [token][column]
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j0 + j < n) {
                        if (careful) token(j0 + j, out + 4 * j, std::true_type());
                        else token(j0 + j, out + 4 * j, std::false_type());
                        step = j0 + j == WALK_TOKENS - 2 ? a16 : a;
                    }
                if (!STATES) {
                    const float sum = sum_over_lanes<16, K_LANES>(out, kk);
                    const uint32_t j = j0 + kk / 4, c = c0 + 4 * vg + kk % 4;
                    if (j < n && c < p.v_size) write_out(p.seq.row(t0 + j), c, sum * p.out_scale);
                }
            }
            if (t0 + WALK_TOKENS < piece.to) {
                buffer ^= 1;
                careful = __syncthreads_or(put(buffer));      // (its last readers are behind the barrier of the tile before)
            }
        }
    };

    if constexpr (STATES) {
        pdl_launch_dependents();                    // (what joins the states waits before it reads them)
        Piece piece;
        if (!handed_on(p, g, piece)) return;
        walk(piece);
        float *to = p.carried + (static_cast<size_t>(g) * p.heads + h) * p.state_size();
        for_states([&](float v, uint32_t r, uint32_t c) { to[static_cast<size_t>(r) * p.v_size + c] = v; });
    } else {
        pdl_wait();                                 // for the states that segments hand on
        const uint32_t from = g * p.segment, to = g + 1 == p.segments ? p.tokens : min(p.tokens, from + p.segment);
        // rows of no sequence: the first few and the last few
        const uint32_t first = p.seq.first(), last = max(p.seq.last(), first);
        auto zeros = [&](uint32_t b, uint32_t e) {
            const uint32_t columns = min(COLUMNS, p.v_size - c0);
            for (uint32_t t = b + threadIdx.x / COLUMNS; t < e; t += WALK_THREADS / COLUMNS)
                if (threadIdx.x % COLUMNS < columns) write_out(p.seq.row(t), c0 + threadIdx.x % COLUMNS, 0.0f);
        };
        zeros(from, min(first, to));
        zeros(max(last, from), to);
        for_pieces(p, g,
            [&](const Piece &piece) {
                walk(piece);
                if (piece.ends && p.last != nullptr) {
                    float *at = p.last + (static_cast<size_t>(p.seq.state(piece.sequence)) * p.heads + h) * p.state_size();
                    for_states([&](float v, uint32_t r, uint32_t c) { at[p.state_at(r, c)] = v * (p.seq.backwards ? a : 1.0f); });
                }
            },
            [&](uint32_t sequence) {        // a sequence of no tokens leaves the state that it comes with
                if (p.last == nullptr) return;
                const size_t at = (static_cast<size_t>(p.seq.state(sequence)) * p.heads + h) * p.state_size();
                for_states([&](float, uint32_t r, uint32_t c) {
                    p.last[at + p.state_at(r, c)] = p.initial != nullptr ? p.initial[at + p.state_at(r, c)] : 0.0f;
                });
            });
    }
}

// What the segments hand on, joined in order: in[g + 1] = a^segment in[g] + own[g] where a sequence fills segment g, own[g] where it
// begins there.  A thread an element of the state.
constexpr uint32_t JOIN_THREADS = 256, JOIN_ROUND = 256;
__global__ __launch_bounds__(JOIN_THREADS) void decay_join_kernel(const DecayWalk p) {
    __shared__ uint8_t kind[JOIN_ROUND];          // of segment g: 0 nothing handed on, 1 a sequence that begins in it, 2 one that fills it
    pdl_launch_dependents();                      // (the walk behind it waits before it reads what this writes)
    const uint32_t h = blockIdx.y;
    const size_t size = p.state_size(), e = static_cast<size_t>(blockIdx.x) * JOIN_THREADS + threadIdx.x, step = p.heads * size;
    float *at = p.carried + h * size + e;
    const float a = decay_power(p.log_decay[h], p.segment);
    // (a power beyond the range makes no number of infinity, or of zero, that the decays one by one would not)
    const bool vanished = a == 0.0f && p.log_decay[h] > -INFINITY, overflowed = a == INFINITY && p.log_decay[h] < INFINITY;
    auto decayed = [&](float x) { return (vanished && !(fabsf(x) < INFINITY)) || (overflowed && x == 0.0f) ? x : a * x; };
    float in = 0.0f;
    for (uint32_t g0 = 0; g0 + 1 < p.segments; g0 += JOIN_ROUND) {
        __syncthreads();
        Piece piece;
        const uint32_t mine = g0 + threadIdx.x;
        kind[threadIdx.x] = mine + 1 < p.segments && handed_on(p, mine, piece) ? (piece.begins ? 1 : 2) : 0;
        __syncthreads();
        if (g0 == 0) pdl_wait();                  // for the states
        const uint32_t n = min(JOIN_ROUND, p.segments - 1 - g0);
        if (e >= size) continue;
        for (uint32_t i0 = 0; i0 < n; i0 += 8) {
            float own[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) own[i] = i0 + i < n && kind[i0 + i] ? __ldcg(at + (g0 + i0 + i) * step) : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i0 + i >= n || kind[i0 + i] == 0) continue;
                in = kind[i0 + i] == 2 ? decayed(in) + own[i] : own[i];
                if (kind[i0 + i] == 2) at[(g0 + i0 + i) * step] = in;
            }
        }
    }
}

// Gradients of keys and values that several heads share: the heads' own, summed in order.
template<typename T, int V>
__global__ void share_kernel(const float *from, T *to, uint64_t count, uint32_t group, uint32_t vectors) {
    pdl_wait();
    struct alignas(4 * V) In { float v[V]; };
    struct alignas(sizeof(T) * V) Out { T v[V]; };
    const In *in = reinterpret_cast<const In *>(from);
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < count; i += static_cast<uint64_t>(gridDim.x) * blockDim.x) {
        const uint64_t row = i / vectors;
        const In *at = in + row * group * vectors + (i - row * vectors);
        In sum = *at;
        for (uint32_t g = 1; g < group; ++g) {
            const In more = at[static_cast<uint64_t>(g) * vectors];
#pragma unroll
            for (int k = 0; k < V; ++k) sum.v[k] += more.v[k];
        }
        Out out;
#pragma unroll
        for (int k = 0; k < V; ++k) out.v[k] = from_float<T>(sum.v[k]);
        reinterpret_cast<Out *>(to)[i] = out;
    }
}

// ---- one token -------------------------------------------------------------------------------------------------------------
constexpr int STEP_THREADS = 256;
constexpr uint32_t STEP_COLUMNS = 32;       // of the state, to a block

struct StepArgs {
    HeadRows q, k, v;
    const float *log_decay;
    const int *slots;
    float *state;
    void *y;
    uint32_t rows, pool, heads, k_size, v_size;
    float scale;
};

__device__ __forceinline__ int slot_of(const StepArgs &p, const uint32_t row) {
    const int slot = p.slots != nullptr ? p.slots[row] : static_cast<int>(row);
    return slot < 0 ? -1 : slot >= static_cast<int>(p.pool) ? -2 : slot;
}

// A block: 32 columns of a head of a row.  V columns to a thread, all of them next to one another, so that a warp reads whole
// sectors; the rows of the state are dealt out to the thread groups, four of them on their way at once.
template<typename T, int V>
__global__ __launch_bounds__(STEP_THREADS) void decay_step_kernel(const StepArgs p) {
    constexpr uint32_t ACROSS = STEP_COLUMNS / V, DOWN = STEP_THREADS / ACROSS;
    constexpr int AHEAD = 4;
    __shared__ float sums[STEP_THREADS / 32][STEP_COLUMNS];
    const uint32_t slabs = (p.v_size + STEP_COLUMNS - 1) / STEP_COLUMNS;
    const uint32_t row = blockIdx.y, h = blockIdx.x / slabs, c = blockIdx.x % slabs * STEP_COLUMNS + threadIdx.x % ACROSS * V;
    const uint32_t down = threadIdx.x / ACROSS, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int slot = slot_of(p, row);
    float *at = p.state + (static_cast<size_t>(max(slot, 0)) * p.heads + h) * p.k_size * p.v_size + c;
    const bool there = c < p.v_size;
    const T *q = p.q.of<T>(h) + row * p.q.row, *k = p.k.of<T>(h) + row * p.k.row, *v_at = p.v.of<T>(h) + row * p.v.row + c;
    struct alignas(4 * V) Columns { float v[V]; };
    // states are on their way before it is known whether an earlier row takes them
    Columns next[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        const uint32_t r = down + i * DOWN;
        if (slot >= 0 && there && r < p.k_size) next[i] = *reinterpret_cast<const Columns *>(at + static_cast<size_t>(r) * p.v_size);
    }
    bool mine = false;
    if (p.slots != nullptr && slot >= 0)
        for (uint32_t i = threadIdx.x; i < row; i += STEP_THREADS) mine |= p.slots[i] == slot;
    if (__syncthreads_or(mine) && slot >= 0) slot = -2;
    float sum[V] = {};
    if (slot >= 0 && there) {
        const float a = decay_power(p.log_decay[h], 1);
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = to_float(v_at[j]);
        for (uint32_t r0 = down; r0 < p.k_size; r0 += AHEAD * DOWN) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const uint32_t r = r0 + i * DOWN;
                if (r >= p.k_size) continue;
                const float kr = to_float(k[r]), qr = to_float(q[r]);
                Columns x = next[i];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    x.v[j] = fmaf(a, x.v[j], kr * v[j]);
                    sum[j] = fmaf(qr, x.v[j], sum[j]);
                }
                *reinterpret_cast<Columns *>(at + static_cast<size_t>(r) * p.v_size) = x;
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const uint32_t r = r0 + (AHEAD + i) * DOWN;
                if (r < p.k_size) next[i] = *reinterpret_cast<const Columns *>(at + static_cast<size_t>(r) * p.v_size);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int o = ACROSS; o < 32; o <<= 1) sum[j] += __shfl_xor_sync(FULL_MASK, sum[j], o);
        if (lane < ACROSS) sums[warp][lane * V + j] = sum[j];
    }
    __syncthreads();
    if (threadIdx.x >= STEP_COLUMNS) return;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < STEP_THREADS / 32; ++w) total += sums[w][threadIdx.x];
    const uint32_t column = blockIdx.x % slabs * STEP_COLUMNS + threadIdx.x;
    if (column < p.v_size)
        static_cast<T *>(p.y)[(static_cast<size_t>(row) * p.heads + h) * p.v_size + column] =
            from_float<T>(slot >= 0 ? total * p.scale : slot == -1 ? 0.0f : __int_as_float(0x7fffffff));
}

// ---- launches ------------------------------------------------------------------------------------------------------------
const bpl_decay_attention_descriptor *checked(const char *opaque, size_t opaque_len, const char *what) {
    const auto *d = unpack<bpl_decay_attention_descriptor>(opaque, opaque_len);
    if (d == nullptr) return nullptr;
    if (d->dtype > BPL_BFLOAT16 || d->key < 1 || d->key > MAX_HEAD || d->value < 1 || d->value > MAX_HEAD || d->kv_heads < 1 ||
        d->heads < 1 || d->heads % d->kv_heads != 0 || d->heads > 65535 || d->tokens >= (1u << 31)) {
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

// Blocks of all heads for one segment of a walk that reads out `v_size` columns.
uint64_t walk_units(const bpl_decay_attention_descriptor &d, uint32_t v_size) {
    return static_cast<uint64_t>(d.heads) * ((v_size + COLUMNS - 1) / COLUMNS);
}
// Segments for two blocks on every SM, as many as it holds; none shorter than 64 tokens.
SegmentPlan walk_plan(const bpl_decay_attention_descriptor &d, bool packed, uint32_t v_size) {
    return plan_segments(d, packed, walk_units(d, v_size), 2ull * sm_count(), 64);
}
// On tensor cores: one block on every SM; up to 512 tokens one segment, else none shorter than 128.  A chunk of 64 tokens takes 2.2 us, a
// pass over two chunks for their states, and joining these, 15: 300 tokens of 16 heads of 128 in one segment 20.5 us, in five 28; 1024 in one 45, in
// two 50, in eight 33; 2048 in one 80, in two 77, in four 52, in eight 40.  Two blocks to an SM would wait for one another: 16,384 tokens of 80 heads of
// 64 536 us as one segment, 598 as three (8192 of 50 heads of 128, which leave a third of the SMs idle in two segments, 287, in five 251).
SegmentPlan tensor_plan(const bpl_decay_attention_descriptor &d, bool packed, uint64_t units) {
    return plan_segments(d, packed, units, sm_count(), d.tokens > 512 ? 128 : 512);
}
size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
// Scratch memory of a call: states between segments, then results that are still to be added up.  (Whether sequences are packed, and
// where operands lie, is not known where it is asked for: the largest of all plans.)
size_t carried_bytes(const bpl_decay_attention_descriptor &d, std::initializer_list<uint32_t> sizes) {
    uint32_t segments = 1;
    for (const bool packed : {true, false})
        for (const uint32_t size : sizes) {
            const uint64_t least = tensor_walk_units(d, 1, size);          // (more units, fewer segments)
            for (const SegmentPlan &q : {walk_plan(d, packed, size), tensor_plan(d, packed, least)})
                if (q.segments > segments) segments = q.segments;
        }
    return segments > 1 ? rounded(sizeof(float) * static_cast<size_t>(segments) * d.heads * d.key * d.value) : 0;
}
// of a walk with `k_size` rows to a state and `v_size` columns, whose results heads share or not
size_t wide_bytes(const bpl_decay_attention_descriptor &d, uint32_t k_size, uint32_t v_size, bool shared) {
    const uint32_t parts = d.dtype == BPL_BFLOAT16 ? tensor_walk_parts(k_size) : 1;
    return shared || parts > 1 ? rounded(sizeof(float) * static_cast<size_t>(d.tokens) * d.heads * parts * v_size) : 0;
}
size_t forward_bytes(const bpl_decay_attention_descriptor &d) { return carried_bytes(d, {d.value}) + wide_bytes(d, d.key, d.value, false); }
size_t backward_carried_bytes(const bpl_decay_attention_descriptor &d) { return carried_bytes(d, {d.key, d.value}); }
size_t backward_bytes(const bpl_decay_attention_descriptor &d) {
    const bool shared = d.heads != d.kv_heads;
    const size_t dq = wide_bytes(d, d.value, d.key, false), dk = wide_bytes(d, d.value, d.key, shared), dv = wide_bytes(d, d.key, d.value, shared);
    const size_t most = dk > dv ? dk : dv;
    return backward_carried_bytes(d) + (dq > most ? dq : most);
}

void join(cudaStream_t stream, const DecayWalk &p) {
    launch_dependent(decay_join_kernel, dim3((p.k_size * p.v_size + JOIN_THREADS - 1) / JOIN_THREADS, p.heads), dim3(JOIN_THREADS), 0, stream, p);
}

template<typename T, int M>
bool walk_sized(cudaStream_t stream, const DecayWalk &p, bool crossing) {
    constexpr unsigned bytes = sizeof(WalkShared<M>);
    const dim3 grid(p.heads * ((p.v_size + COLUMNS - 1) / COLUMNS), p.segments);
    if (!allow_shared<decay_walk_kernel<T, M, false>>(bytes) || !allow_shared<decay_walk_kernel<T, M, true>>(bytes)) {
        set_status(BPL_ERR_CUDA, "decay_attention: shared memory");
        return false;
    }
    if (crossing) {
        decay_walk_kernel<T, M, true><<<dim3(grid.x, p.segments - 1), WALK_THREADS, bytes, stream>>>(p);
        join(stream, p);
    }
    if (crossing) launch_dependent(decay_walk_kernel<T, M, false>, grid, dim3(WALK_THREADS), bytes, stream, p);
    else decay_walk_kernel<T, M, false><<<grid, WALK_THREADS, bytes, stream>>>(p);
    return true;
}

// Where walks run that are made of the same states, and in which segments.  (Operands and results are known here, where they lie too.)
struct WalkPlan : SegmentPlan {
    bool tensor;
};
template<typename T>
WalkPlan plan_walk(const bpl_decay_attention_descriptor &d, bool packed, std::initializer_list<DecayWalk> walks) {
    bool tensor = std::is_same<T, __nv_bfloat16>::value;
    uint32_t widest = 0;
    uint64_t units = 0;
    for (const DecayWalk &p : walks) {
        tensor = tensor && tensor_walk_fits(p);
        widest = p.v_size > widest ? p.v_size : widest;
        const uint64_t u = tensor_walk_units(d, p.k_size, p.v_size);
        units = u > units ? u : units;
    }
    return WalkPlan{tensor ? tensor_plan(d, packed, units) : walk_plan(d, packed, widest), tensor};
}

template<typename T>
bool walk_as_planned(cudaStream_t stream, const DecayWalk &p, const WalkPlan &plan, bool states) {
    const bool crossing = plan.crossing && states;
    if (plan.tensor) {
        if (crossing) {
            if (!tensor_walk_states(stream, p)) return false;
            join(stream, p);
        }
        return tensor_walk(stream, p, crossing);
    }
    if (p.k_size <= 64) return walk_sized<T, 1>(stream, p, crossing);
    if (p.k_size <= 128) return walk_sized<T, 2>(stream, p, crossing);
    return walk_sized<T, 4>(stream, p, crossing);
}

template<typename T>
void share(cudaStream_t stream, const float *from, void *to, uint64_t rows, uint32_t group, uint32_t size) {
    const bool vector = size % 4 == 0 && aligned16(from) && aligned16(to);
    const uint32_t vectors = vector ? size / 4 : size;
    const uint64_t count = rows * vectors, blocks = (count + 255) / 256, most = 32ull * sm_count();
    if (blocks == 0) return;
    const dim3 grid(static_cast<unsigned>(blocks < most ? blocks : most));
    if (vector) launch_dependent(share_kernel<T, 4>, grid, dim3(256), 0, stream, from, static_cast<T *>(to), count, group, vectors);
    else launch_dependent(share_kernel<T, 1>, grid, dim3(256), 0, stream, from, static_cast<T *>(to), count, group, vectors);
}

// One walk, whatever it computes, into p.out; `states`: also of what segments hand on, else that is there already.  `group` heads share a
// result; where there are several, or parts, these are in `wide` first.
template<typename T>
bool walk(cudaStream_t stream, DecayWalk p, const WalkPlan &plan, bool states, uint32_t group, float *wide) {
    void *const out = p.out;
    p.segment = plan.segment;
    p.segments = plan.segments;
    p.parts = plan.tensor ? tensor_walk_parts(p.k_size) : 1;
    p.wide_out = group * p.parts > 1;
    p.out = p.wide_out ? wide : out;
    if (!walk_as_planned<T>(stream, p, plan, states)) return false;
    if (p.wide_out) share<T>(stream, wide, out, static_cast<uint64_t>(p.tokens) * (p.heads / group), group * p.parts, p.v_size);
    return true;
}

struct Operands {
    HeadRows q, k, v;
    const float *log_decay;
    const int *indptr;
};
// (heads that lie on one another are one that all share)
HeadRows rows_of(const void *p, long long row, long long head, const bpl_decay_attention_descriptor &d, uint32_t group) {
    return HeadRows{p, row, head, head == 0 ? d.heads : group};
}
Operands operands(void **b, const bpl_decay_attention_descriptor &d) {
    const uint32_t group = d.heads / d.kv_heads;
    return Operands{rows_of(b[0], d.q_stride, d.q_head_stride, d, 1), rows_of(b[1], d.k_stride, d.k_head_stride, d, group),
                    rows_of(b[2], d.v_stride, d.v_head_stride, d, group), static_cast<const float *>(b[3]), static_cast<const int *>(b[4])};
}

DecayWalk walk_of(const Operands &o, const bpl_decay_attention_descriptor &d, void *carried, bool backwards) {
    DecayWalk p = {};
    p.log_decay = o.log_decay;
    p.carried = static_cast<float *>(carried);
    p.seq = VirtualSequences{{o.indptr, d.sequences, d.length, d.tokens}, backwards};
    p.tokens = d.tokens;
    p.heads = d.heads;
    return p;
}

template<typename T>
void forward(cudaStream_t stream, void **b, const bpl_decay_attention_descriptor &d) {
    const Operands o = operands(b, d);
    DecayWalk p = walk_of(o, d, b[8], false);
    p.q = o.q; p.k = o.k; p.v = o.v;
    p.k_size = d.key; p.v_size = d.value;
    p.initial = static_cast<const float *>(b[5]);
    p.last = static_cast<float *>(b[7]);
    p.out_scale = p.own_scale = d.scale;
    p.state_scale = 1.0f;
    float *wide = reinterpret_cast<float *>(static_cast<char *>(b[8]) + carried_bytes(d, {d.value}));
    p.out = b[6];
    walk<T>(stream, p, plan_walk<T>(d, o.indptr != nullptr, {p}), true, 1, wide);
}

template<typename T>
void backward(cudaStream_t stream, void **b, const bpl_decay_attention_descriptor &d) {
    const Operands o = operands(b, d);
    const HeadRows dy = {b[6], static_cast<long long>(d.heads) * d.value, d.value, 1};
    char *ws = static_cast<char *>(b[12]);
    float *wide = reinterpret_cast<float *>(ws + backward_carried_bytes(d));
    const bool packed = o.indptr != nullptr;
    const uint32_t group = d.heads / d.kv_heads;
    // dq: S do, the states made of v and k
    DecayWalk p = walk_of(o, d, ws, false);
    p.q = dy; p.k = o.v; p.v = o.k;
    p.k_size = d.value; p.v_size = d.key;
    p.initial = static_cast<const float *>(b[5]);
    p.transposed = true;
    p.out_scale = p.own_scale = d.scale;
    p.state_scale = 1.0f;
    p.out = b[8];
    if (!walk<T>(stream, p, plan_walk<T>(d, packed, {p}), true, 1, wide)) return;
    // dv: X^T k, X made of q and do from the last token on, and X in front of the first token is the initial state's gradient
    p = walk_of(o, d, ws, true);
    p.q = o.k; p.k = o.q; p.v = dy;
    p.k_size = d.key; p.v_size = d.value;
    p.initial = static_cast<const float *>(b[7]);
    p.out_scale = 1.0f;
    p.state_scale = p.own_scale = d.scale;
    p.last = static_cast<float *>(b[11]);
    p.out = b[10];
    // dk: X v, on the transposed state, from the same states that segments hand on
    DecayWalk r = p;
    r.q = o.v; r.k = dy; r.v = o.q;
    r.k_size = d.value; r.v_size = d.key;
    r.transposed = r.carried_turned = true;
    r.last = nullptr;
    r.out = b[9];
    const WalkPlan plan = plan_walk<T>(d, packed, {p, r});
    if (!walk<T>(stream, p, plan, true, group, wide)) return;
    walk<T>(stream, r, plan, false, group, wide);
}

template<typename F>
void with_type(uint32_t dtype, F f) {
    if (dtype == BPL_FLOAT) f(float());
    else if (dtype == BPL_HALF) f(__half());
    else f(__nv_bfloat16());
}

}  // namespace

size_t decay_attention_workspace_bytes(const char *opaque, size_t opaque_len) {
    if (opaque == nullptr || opaque_len != sizeof(bpl_decay_attention_descriptor)) return 0;
    return forward_bytes(*reinterpret_cast<const bpl_decay_attention_descriptor *>(opaque));
}
size_t decay_attention_backward_workspace_bytes(const char *opaque, size_t opaque_len) {
    if (opaque == nullptr || opaque_len != sizeof(bpl_decay_attention_descriptor)) return 0;
    return backward_bytes(*reinterpret_cast<const bpl_decay_attention_descriptor *>(opaque));
}

}  // namespace bpl

using namespace bpl;

extern "C" {

void decay_attention(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "decay_attention: heads of 1 to 256 elements, one at least and a multiple of those of k and v, fewer than 2^31 tokens");
    if (d == nullptr) return;
    if (!given(buffers, {3}, "decay_attention: null buffer") ||
        (d->tokens > 0 && !given(buffers, {0, 1, 2, 6}, "decay_attention: null buffer")) ||
        (decay_attention_workspace_bytes(opaque, opaque_len) > 0 && !given(buffers, {8}, "decay_attention: no workspace")))
        return;
    if (!sequences_fit(*d, buffers[4])) {
        set_status(BPL_ERR_ARGUMENT, "decay_attention: 2^31 sequences, or sequences and their length are not the tokens");
        return;
    }
    if (d->sequences == 0 && d->tokens == 0) return;
    with_type(d->dtype, [&](auto type) { forward<decltype(type)>(stream, buffers, *d); });
    launch_ok();
}

void decay_attention_backward(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "decay_attention_backward: heads of 1 to 256 elements, one at least and a multiple of those of k and v, fewer than 2^31 tokens");
    if (d == nullptr) return;
    if (!given(buffers, {3}, "decay_attention_backward: null buffer") ||
        (d->tokens > 0 && !given(buffers, {0, 1, 2, 6, 8, 9, 10}, "decay_attention_backward: null buffer")) ||
        (decay_attention_backward_workspace_bytes(opaque, opaque_len) > 0 && !given(buffers, {12}, "decay_attention_backward: no workspace")))
        return;
    if (!sequences_fit(*d, buffers[4])) {
        set_status(BPL_ERR_ARGUMENT, "decay_attention_backward: 2^31 sequences, or sequences and their length are not the tokens");
        return;
    }
    if (d->sequences == 0 && d->tokens == 0) return;
    with_type(d->dtype, [&](auto type) { backward<decltype(type)>(stream, buffers, *d); });
    launch_ok();
}

void decay_attention_step(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "decay_attention_step: heads of 1 to 256 elements, one at least and a multiple of those of k and v");
    if (d == nullptr || d->tokens == 0) return;
    if (d->tokens > 65535 || d->sequences >= (1u << 31) || (buffers[4] == nullptr && d->sequences < d->tokens)) {
        set_status(BPL_ERR_ARGUMENT, "decay_attention_step: at most 65535 rows, and a state for every row");
        return;
    }
    if (!given(buffers, {0, 1, 2, 3, 6}, "decay_attention_step: null buffer") ||
        (d->sequences > 0 && !given(buffers, {5}, "decay_attention_step: null buffer")))
        return;
    const Operands o = operands(buffers, *d);
    StepArgs p = {o.q, o.k, o.v, o.log_decay, o.indptr, static_cast<float *>(buffers[5]), buffers[6], d->tokens, d->sequences, d->heads, d->key,
                  d->value, d->scale};
    const dim3 grid(d->heads * ((d->value + STEP_COLUMNS - 1) / STEP_COLUMNS), d->tokens);
    with_type(d->dtype, [&](auto type) {
        using T = decltype(type);
        if (d->value % 4 == 0 && aligned16(p.state)) decay_step_kernel<T, 4><<<grid, STEP_THREADS, 0, stream>>>(p);
        else decay_step_kernel<T, 1><<<grid, STEP_THREADS, 0, stream>>>(p);
    });
    launch_ok();
}

}  // extern "C"
