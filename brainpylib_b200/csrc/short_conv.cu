// A short causal convolution of every channel with its own taps, over packed sequences (no counterpart in brainpylib):
//
//     p[t] = bias + sum_j weight[j] x[t - W + 1 + j];   y = p, or p / (1 + e^-p)
//
// its gradient, and the same for one new token per running sequence.  In front of a sequence stand the W - 1 inputs that it
// comes with, or zeros.  Bound by memory: a thread keeps the last W - 1 inputs of its neighbouring channels in registers and walks
// a run of tokens, so that an input is read once (and W - 1 more per run).  16,384 tokens of 4096 channels in 16 bits, four taps: 60 us on
// the device, 4.5 TB/s (whole calls: 63; with four rows on their way and shorter runs 68, with eight channels a thread 83).
#include <initializer_list>
#include <type_traits>

#include "sequence.cuh"

namespace bpl {
namespace {

constexpr int CONV_THREADS = 128;
constexpr uint32_t MAX_WIDTH = 8;

template<typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};
// (four elements as two pairs: an array of 16-bit elements would take a register for each)
template<typename T, int V>
using Row = std::conditional_t<V == 4 && sizeof(T) == 2, uint2, Vec<T, V>>;
template<typename T, int V>
__device__ __forceinline__ void floats_of(const Row<T, V> &raw, float (&out)[V]) {
    if constexpr (V == 4 && sizeof(T) == 2) {
        const float2 a = split(load_pair(reinterpret_cast<const T *>(&raw.x))), b = split(load_pair(reinterpret_cast<const T *>(&raw.y)));
        out[0] = a.x; out[1] = a.y; out[2] = b.x; out[3] = b.y;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = to_float(raw.v[i]);
    }
}
template<typename T, int V>
__device__ __forceinline__ void load_row(const T *at, float (&out)[V]) {
    floats_of<T, V>(*reinterpret_cast<const Row<T, V> *>(at), out);
}
template<typename T, int V>
__device__ __forceinline__ void store_row(T *at, const float (&in)[V]) {
    if constexpr (V == 4 && sizeof(T) == 2) {
        uint2 raw;
        store_pair(reinterpret_cast<T *>(&raw.x), make_float2(in[0], in[1]));
        store_pair(reinterpret_cast<T *>(&raw.y), make_float2(in[2], in[3]));
        *reinterpret_cast<uint2 *>(at) = raw;
    } else {
        Vec<T, V> r;
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = from_float<T>(in[i]);
        *reinterpret_cast<Vec<T, V> *>(at) = r;
    }
}

template<typename T>
struct ConvArgs {
    const T *x, *initial, *dy, *d_last;
    const void *weight, *bias;
    T *y, *last, *dx, *d_initial;
    void *d_weight, *d_bias;
    float *parts;                // [runs][channels][W + 1]: taps, then bias
    long long x_stride;
    Sequences seq;
    uint32_t channels, groups, run, n_runs;      // groups of V neighbouring channels; tokens of a run
    bool silu, wide, aligned;    // wide: weight and bias are float whatever T is; aligned: a thread's are at 16-byte boundaries
};

template<typename T>
__device__ __forceinline__ float parameter(const void *p, size_t i, bool wide) {
    return wide ? static_cast<const float *>(p)[i] : to_float(static_cast<const T *>(p)[i]);
}

// `count` neighbouring parameters, 16 bytes at once where their address allows it
template<typename P, int COUNT>
__device__ __forceinline__ void load_many(const P *at, float (&out)[COUNT], bool aligned) {
    constexpr int E = 16 / sizeof(P);
    if (COUNT % E == 0 && aligned) {      // (a thread's parameters begin at a multiple of COUNT)
#pragma unroll
        for (int i = 0; i + E <= COUNT; i += E) {
            const Vec<P, E> r = *reinterpret_cast<const Vec<P, E> *>(at + i);
#pragma unroll
            for (int k = 0; k < E; ++k) out[i + k] = to_float(r.v[k]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) out[i] = to_float(at[i]);
    }
}
template<typename T, int W, int V>
__device__ __forceinline__ void load_weights(const ConvArgs<T> &p, uint32_t c, float (&w)[W][V], float (&b)[V]) {
    float all[V * W];
    if (p.wide) load_many(static_cast<const float *>(p.weight) + static_cast<size_t>(c) * W, all, p.aligned);
    else load_many(static_cast<const T *>(p.weight) + static_cast<size_t>(c) * W, all, p.aligned);
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][i] = all[i * W + j];
        b[i] = 0.0f;
    }
    if (p.bias != nullptr) {
        if (p.wide) load_many(static_cast<const float *>(p.bias) + c, b, p.aligned);
        else load_many(static_cast<const T *>(p.bias) + c, b, p.aligned);
    }
}

// The W - 1 inputs in front of token t of the sequence that begins at `begin` (k = 0 the earliest).
template<typename T, int W, int V>
__device__ __forceinline__ void load_window(const ConvArgs<T> &p, uint32_t c, uint32_t s, uint32_t begin, uint32_t t,
                                            float (&window)[W][V]) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        const uint32_t back = W - 1 - k;             // the input at t - back
        if (t - begin >= back) {
            load_row<T, V>(p.x + static_cast<long long>(t - back) * p.x_stride + c, window[k]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                window[k][i] = p.initial != nullptr
                                   ? to_float(p.initial[(static_cast<size_t>(s) * p.channels + c + i) * (W - 1) + (W - 1 - (back - (t - begin)))])
                                   : 0.0f;
        }
    }
}

template<int W, int V>
__device__ __forceinline__ void push(float (&window)[W][V], const float (&x)[V]) {      // window[W - 1] is spare
#pragma unroll
    for (int k = 0; k + 2 < W; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) window[k][i] = window[k + 1][i];
    if (W > 1)
#pragma unroll
        for (int i = 0; i < V; ++i) window[W > 1 ? W - 2 : 0][i] = x[i];
}

template<typename T, int W, int V>
__global__ void __launch_bounds__(CONV_THREADS)
short_conv_kernel(const ConvArgs<T> p) {
    const uint64_t id = static_cast<uint64_t>(blockIdx.x) * CONV_THREADS + threadIdx.x;
    const uint32_t run = static_cast<uint32_t>(id / p.groups), c = static_cast<uint32_t>(id % p.groups) * V;
    if (run >= p.n_runs) return;
    const Sequences seq = p.seq;
    float w[W][V], b[V], window[W][V];
    load_weights<T, W, V>(p, c, w, b);

    const uint32_t from = run * p.run, to = min(from + p.run, seq.tokens);
    const uint32_t live_from = max(from, seq.first()), live_to = min(to, seq.last());
    uint32_t s = 0, s_end = 0;
    if (live_from < live_to) {
        s = seq.of(live_from);
        s_end = seq.end(s);
        load_window<T, W, V>(p, c, s, seq.begin(s), live_from, window);
    }
    constexpr uint32_t AHEAD = 8;                 // rows on their way at once
    auto one = [&](const float (&x)[V], float (&y)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float sum = b[i];
#pragma unroll
            for (int j = 0; j + 1 < W; ++j) sum = fmaf(w[j][i], window[j][i], sum);
            sum = fmaf(w[W - 1][i], x[i], sum);
            y[i] = p.silu ? silu(sum) : sum;
        }
        push<W, V>(window, x);
    };
    for (uint32_t t0 = from; t0 < to; t0 += AHEAD) {
        float x[V], y[V];
        T *at = p.y + static_cast<size_t>(t0) * p.channels + c;
        if (t0 >= live_from && t0 + AHEAD <= live_to && s_end > t0 + AHEAD) {        // all of one sequence that goes on
            Row<T, V> raw[AHEAD];
            const T *from_row = p.x + t0 * p.x_stride + c;
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k, from_row += p.x_stride) raw[k] = *reinterpret_cast<const Row<T, V> *>(from_row);
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k, at += p.channels) {
                floats_of<T, V>(raw[k], x);
                one(x, y);
                store_row<T, V>(at, y);
            }
            continue;
        }
#pragma unroll 1
        for (uint32_t t = t0; t < min(t0 + AHEAD, to); ++t, at += p.channels) {
            if (t < live_from || t >= live_to) {
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = 0.0f;
                store_row<T, V>(at, y);
                continue;
            }
            load_row<T, V>(p.x + t * p.x_stride + c, x);
            one(x, y);
            store_row<T, V>(at, y);
            if (t + 1 >= s_end) {
                if (p.last != nullptr) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
#pragma unroll
                        for (int j = 0; j + 1 < W; ++j)
                            p.last[(static_cast<size_t>(s) * p.channels + c + i) * (W - 1) + j] = from_float<T>(window[j][i]);
                }
                while (++s < seq.count && (s_end = seq.end(s)) <= t + 1) {}
                if (s < seq.count && t + 1 < live_to) load_window<T, W, V>(p, c, s, t + 1, t + 1, window);
                else s_end = 0xffffffffu;
            }
        }
    }
    if (p.last != nullptr)                        // sequences without a token leave the inputs they came with
        for (uint32_t q = run; q < seq.count; q += p.n_runs) {
            if (seq.end(q) > seq.begin(q)) continue;
            const size_t at = (static_cast<size_t>(q) * p.channels + c) * (W - 1);
            for (int i = 0; i < V * (W - 1); ++i) p.last[at + i] = p.initial != nullptr ? p.initial[at + i] : from_float<T>(0.0f);
        }
}

// The derivative by p of the token whose input is x and whose earlier inputs are the window's.
template<typename T, int W, int V>
__device__ __forceinline__ void slope(const ConvArgs<T> &p, const float (&w)[W][V], const float (&b)[V],
                                      const float (&window)[W][V], const float (&x)[V], const float (&dy)[V], float (&dp)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        dp[i] = dy[i];
        if (p.silu) {
            float sum = b[i];
#pragma unroll
            for (int j = 0; j + 1 < W; ++j) sum = fmaf(w[j][i], window[j][i], sum);
            sum = fmaf(w[W - 1][i], x[i], sum);
            const float sg = sigmoid(sum);
            dp[i] *= sg * fmaf(sum, 1.0f - sg, 1.0f);
        }
    }
}

// A thread walks its run and W - 1 tokens more: dx[u] is done when the last token that reads x[u] is.  Sums over tokens are left
// as one part per run.
template<typename T, int W, int V>
__global__ void __launch_bounds__(CONV_THREADS)
short_conv_backward_kernel(const ConvArgs<T> p) {
    const uint64_t id = static_cast<uint64_t>(blockIdx.x) * CONV_THREADS + threadIdx.x;
    const uint32_t run = static_cast<uint32_t>(id / p.groups), c = static_cast<uint32_t>(id % p.groups) * V;
    if (run >= p.n_runs) return;
    const Sequences seq = p.seq;
    float w[W][V], b[V], window[W][V], dw[W][V], db[V];
    load_weights<T, W, V>(p, c, w, b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][i] = 0.0f;
    }
    const uint32_t from = run * p.run, to = min(from + p.run, seq.tokens);
    const uint32_t live_from = max(from, seq.first()), live_to = min(to, seq.last());
    float zeros[V];
#pragma unroll
    for (int i = 0; i < V; ++i) zeros[i] = 0.0f;
    for (uint32_t t = from; t < to; ++t)
        if (t < live_from || t >= live_to) store_row<T, V>(p.dx + static_cast<size_t>(t) * p.channels + c, zeros);

    uint32_t a = live_from, s = live_from < live_to ? seq.of(live_from) : 0;
    while (a < live_to && s < seq.count) {
        const uint32_t begin = min(seq.begin(s), a), end = max(seq.end(s), a + 1);
        const uint32_t stop = min(live_to, end), ahead = min(stop + (W - 1), end);      // dx of [a, stop) reads up to `ahead`
        load_window<T, W, V>(p, c, s, begin, a, window);
        float dp[W][V];                           // of the last W tokens
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) dp[k][i] = 0.0f;
        constexpr uint32_t AHEAD = 4;             // rows on their way at once
        const uint32_t there = min(ahead, seq.tokens);
        for (uint32_t t0 = a; t0 < stop + (W - 1); t0 += AHEAD) {
            float x[AHEAD][V], dy[AHEAD][V];
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k)
                if (t0 + k < there) {
                    load_row<T, V>(p.x + (t0 + k) * p.x_stride + c, x[k]);
                    load_row<T, V>(p.dy + static_cast<size_t>(t0 + k) * p.channels + c, dy[k]);
                }
#pragma unroll
            for (uint32_t q = 0; q < AHEAD; ++q) {
                const uint32_t t = t0 + q;
                if (t >= stop + (W - 1)) break;
#pragma unroll
                for (int k = 0; k + 1 < W; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) dp[k][i] = dp[k + 1][i];
                if (t < there) {
                    slope<T, W, V>(p, w, b, window, x[q], dy[q], dp[W - 1]);
                    if (t < stop) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
#pragma unroll
                            for (int j = 0; j + 1 < W; ++j) dw[j][i] = fmaf(dp[W - 1][i], window[j][i], dw[j][i]);
                            dw[W - 1][i] = fmaf(dp[W - 1][i], x[q][i], dw[W - 1][i]);
                            db[i] += dp[W - 1][i];
                        }
                    }
                    push<W, V>(window, x[q]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) dp[W - 1][i] = 0.0f;
                }
                if (t >= a + (W - 1)) {
                    const uint32_t u = t - (W - 1);
                    float dx[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float sum = 0.0f;
#pragma unroll
                        for (int k = 0; k < W; ++k) sum = fmaf(w[W - 1 - k][i], dp[k][i], sum);
                        if (p.d_last != nullptr && end - u <= W - 1)
                            sum += to_float(p.d_last[(static_cast<size_t>(s) * p.channels + c + i) * (W - 1) + (W - 1 - (end - u))]);
                        dx[i] = sum;
                    }
                    store_row<T, V>(p.dx + static_cast<size_t>(u) * p.channels + c, dx);
                }
            }
        }
        a = stop;
        while (++s < seq.count && seq.end(s) <= a) {}
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float *at = p.parts + (static_cast<size_t>(run) * p.channels + c + i) * (W + 1);
#pragma unroll
        for (int j = 0; j < W; ++j) at[j] = dw[j][i];
        at[W] = db[i];
    }
}

// The gradient of the inputs that sequences come with: their first W - 1 tokens read them.
template<typename T, int W>
__global__ void __launch_bounds__(CONV_THREADS)
short_conv_initial_kernel(const ConvArgs<T> p) {
    const uint64_t id = static_cast<uint64_t>(blockIdx.x) * CONV_THREADS + threadIdx.x;
    const uint32_t s = static_cast<uint32_t>(id / p.channels), c = static_cast<uint32_t>(id % p.channels);
    if (s >= p.seq.count) return;
    const uint32_t begin = p.seq.begin(s), end = max(p.seq.end(s), begin);
    float w[W][1], b[1], window[W][1], d[W];
    load_weights<T, W, 1>(p, c, w, b);
    load_window<T, W, 1>(p, c, s, begin, begin, window);
#pragma unroll
    for (int k = 0; k < W; ++k) d[k] = 0.0f;
    const size_t at = (static_cast<size_t>(s) * p.channels + c) * (W - 1);
#pragma unroll
    for (uint32_t i = 0; i + 1 < W; ++i) {
        const uint32_t t = begin + i;
        if (t >= end) {                           // the inputs that are left behind when the sequence is short
            if (p.d_last != nullptr) d[i] += to_float(p.d_last[at + i - (end - begin)]);
            continue;
        }
        float x[1], dy[1], dp[1];
        load_row<T, 1>(p.x + t * p.x_stride + c, x);
        load_row<T, 1>(p.dy + static_cast<size_t>(t) * p.channels + c, dy);
        slope<T, W, 1>(p, w, b, window, x, dy, dp);
        push<W, 1>(window, x);
#pragma unroll
        for (uint32_t j = 0; i + j + 1 < W; ++j) d[i + j] = fmaf(w[j][0], dp[0], d[i + j]);
    }
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) p.d_initial[at + k] = from_float<T>(d[k]);
}

// Adds the parts of the runs up, 32 columns to a block, its 8 warps every 8th run; in the same order every time.
template<typename T>
__global__ void __launch_bounds__(256)
short_conv_sum_kernel(const ConvArgs<T> p, const uint32_t width) {
    __shared__ float sums[8][33];
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const size_t n = static_cast<size_t>(p.channels) * (width + 1), i = static_cast<size_t>(blockIdx.x) * 32 + lane;
    float sum = 0.0f;
    if (i < n) {
#pragma unroll 4
        for (uint32_t r = warp; r < p.n_runs; r += 8) sum += __ldcg(p.parts + r * n + i);
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || i >= n) return;
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += sums[w][lane];
    const size_t c = i / (width + 1), j = i % (width + 1);
    void *out = j < width ? p.d_weight : p.d_bias;
    if (out == nullptr) return;
    const size_t at = j < width ? c * width + j : c;
    if (p.wide) static_cast<float *>(out)[at] = sum;
    else static_cast<T *>(out)[at] = from_float<T>(sum);
}

// ---- one token per running sequence ------------------------------------------------------------------------------------
template<typename T>
struct ConvStepArgs {
    const T *x;
    const void *weight, *bias;
    const int *slots;
    T *state, *y;
    long long x_stride;
    uint32_t rows, pool, channels;
    bool silu, wide;
};

// Bound by latency: a window is read before it is known whether an earlier row takes it (what is read then is dropped, and nothing
// is written), two latencies of memory in a row instead of three (200 rows of 5120 channels: 7.4 us on the device).
template<typename T, int W>
__global__ void __launch_bounds__(CONV_THREADS)
short_conv_step_kernel(const ConvStepArgs<T> p) {
    const uint32_t row = blockIdx.y, c = blockIdx.x * CONV_THREADS + threadIdx.x;
    const int slot = p.slots != nullptr ? p.slots[row] : static_cast<int>(row);
    const bool valid = c < p.channels, inside = valid && slot >= 0 && slot < static_cast<int>(p.pool);
    T *at = p.state + (static_cast<size_t>(max(slot, 0)) * p.channels + c) * (W - 1);
    T window[W];
    float w[W], sum = 0.0f;
    if (inside) {
#pragma unroll
        for (int j = 0; j + 1 < W; ++j) window[j] = at[j];
        window[W - 1] = p.x[row * p.x_stride + c];
#pragma unroll
        for (int j = 0; j < W; ++j) w[j] = parameter<T>(p.weight, static_cast<size_t>(c) * W + j, p.wide);
        if (p.bias != nullptr) sum = parameter<T>(p.bias, c, p.wide);
    }
    bool taken = false;
    if (p.slots != nullptr) {
        for (uint32_t i = threadIdx.x; i < row; i += CONV_THREADS) taken |= p.slots[i] == slot;
        taken = __syncthreads_or(taken);
    }
    if (!valid) return;
    T *y = p.y + static_cast<size_t>(row) * p.channels + c;
    if (!inside || taken) {
        *y = from_float<T>(slot < 0 ? 0.0f : __int_as_float(0x7fffffff));
        return;
    }
#pragma unroll
    for (int j = 0; j < W; ++j) sum = fmaf(w[j], to_float(window[j]), sum);
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) at[j] = window[j + 1];
    *y = from_float<T>(p.silu ? silu(sum) : sum);
}

// ---- launches -----------------------------------------------------------------------------------------------------------
const bpl_short_conv_descriptor *checked(const char *opaque, size_t opaque_len, const char *what) {
    const auto *d = unpack<bpl_short_conv_descriptor>(opaque, opaque_len);
    if (d == nullptr) return nullptr;
    if (d->dtype > BPL_BFLOAT16 || d->width < 1 || d->width > MAX_WIDTH || d->tokens >= (1u << 31) ||
        (d->weight_dtype != BPL_FLOAT && d->weight_dtype != d->dtype)) {
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

// tokens of a run: 64 where that leaves `threads` threads to an SM (half that number, or runs of 32 or 128: the same time within 3 %),
// fewer for smaller calls
uint32_t run_tokens(uint32_t tokens, uint32_t groups, uint32_t most, uint32_t threads) {
    uint32_t run = most;
    while (run > 8 && static_cast<uint64_t>(tokens) * groups / run < static_cast<uint64_t>(threads) * sm_count()) run /= 2;
    return run;
}
// (by what the descriptor says of the rows: groups of four channels, or single ones)
uint32_t backward_run(const bpl_short_conv_descriptor &d) {
    return run_tokens(d.tokens, d.channels % 4 == 0 && d.x_stride % 4 == 0 ? d.channels / 4 : d.channels, 64, 512);
}

template<typename F>
void with_width(uint32_t width, F f) {
    switch (width) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        case 4: return f(std::integral_constant<int, 4>());
        case 5: return f(std::integral_constant<int, 5>());
        case 6: return f(std::integral_constant<int, 6>());
        case 7: return f(std::integral_constant<int, 7>());
        default: return f(std::integral_constant<int, 8>());
    }
}
template<typename F>
void with_type(uint32_t dtype, F f) {
    if (dtype == BPL_FLOAT) f(float());
    else if (dtype == BPL_HALF) f(__half());
    else f(__nv_bfloat16());
}

bool rows_aligned(std::initializer_list<const void *> rows, long long stride, uint32_t channels, size_t elem, uint32_t v) {
    for (const void *r : rows)
        if (reinterpret_cast<uintptr_t>(r) % (elem * v) != 0) return false;
    return stride % v == 0 && channels % v == 0;
}

template<typename T>
ConvArgs<T> arguments(void **b, const bpl_short_conv_descriptor &d) {
    ConvArgs<T> p = {};
    p.x = static_cast<const T *>(b[0]);
    p.weight = b[1];
    p.bias = b[2];
    p.seq = Sequences{static_cast<const int *>(b[3]), d.sequences, d.length, d.tokens};
    p.initial = static_cast<const T *>(b[4]);
    p.x_stride = d.x_stride;
    p.channels = d.channels;
    p.silu = (d.flags & BPL_CONV_SILU) != 0;
    p.wide = d.weight_dtype == BPL_FLOAT;
    p.aligned = aligned16(p.weight) && aligned16(p.bias);
    return p;
}

unsigned blocks_for(uint64_t threads, int block) { return static_cast<unsigned>((threads + block - 1) / block); }

}  // namespace

size_t short_conv_backward_workspace_bytes(const char *opaque, size_t opaque_len) {
    if (opaque == nullptr || opaque_len != sizeof(bpl_short_conv_descriptor)) return 0;
    const auto &d = *reinterpret_cast<const bpl_short_conv_descriptor *>(opaque);
    const uint32_t run = backward_run(d);
    return sizeof(float) * ((d.tokens + run - 1) / run) * static_cast<size_t>(d.channels) * (d.width + 1);
}

}  // namespace bpl

using namespace bpl;

extern "C" {

void short_conv(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "short_conv: 1..8 taps of the inputs' type or float, fewer than 2^31 tokens");
    if (d == nullptr || d->channels == 0 || (d->tokens == 0 && d->sequences == 0)) return;
    if (!given(buffers, {1}, "short_conv: null buffer") || (d->tokens > 0 && !given(buffers, {0, 5}, "short_conv: null buffer")))
        return;
    if (!sequences_fit(*d, buffers[3])) {
        set_status(BPL_ERR_ARGUMENT, "short_conv: 2^31 sequences, or sequences and their length are not the tokens");
        return;
    }
    with_type(d->dtype, [&](auto type) {
        using T = decltype(type);
        constexpr int V = 4;        // (eight of 16 bits a thread take 168 registers and a fifth more time)
        ConvArgs<T> p = arguments<T>(buffers, *d);
        p.y = static_cast<T *>(buffers[5]);
        p.last = static_cast<T *>(buffers[6]);
        const bool vector = rows_aligned({p.x, p.y}, d->x_stride, d->channels, sizeof(T), V);
        p.groups = vector ? d->channels / V : d->channels;
        p.run = run_tokens(d->tokens, p.groups, 64, 1024);
        p.n_runs = d->tokens ? (d->tokens + p.run - 1) / p.run : 1;
        with_width(d->width, [&](auto width) {
            constexpr int W = decltype(width)::value;
            const unsigned blocks = blocks_for(static_cast<uint64_t>(p.groups) * p.n_runs, CONV_THREADS);
            if (vector) short_conv_kernel<T, W, V><<<blocks, CONV_THREADS, 0, stream>>>(p);
            else short_conv_kernel<T, W, 1><<<blocks, CONV_THREADS, 0, stream>>>(p);
        });
    });
    launch_ok();
}

void short_conv_backward(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "short_conv_backward: 1..8 taps of the inputs' type or float, fewer than 2^31 tokens");
    if (d == nullptr || d->channels == 0) return;
    if (!given(buffers, {1, 8}, "short_conv_backward: null buffer") ||
        (d->tokens > 0 && !given(buffers, {0, 5, 7, 11}, "short_conv_backward: null buffer")) ||
        (buffers[2] != nullptr && !given(buffers, {9}, "short_conv_backward: null buffer")) ||
        (buffers[4] != nullptr && !given(buffers, {10}, "short_conv_backward: null buffer")))
        return;
    if (!sequences_fit(*d, buffers[3])) {
        set_status(BPL_ERR_ARGUMENT, "short_conv_backward: 2^31 sequences, or sequences and their length are not the tokens");
        return;
    }
    with_type(d->dtype, [&](auto type) {
        using T = decltype(type);
        constexpr int V = 4;
        ConvArgs<T> p = arguments<T>(buffers, *d);
        p.dy = static_cast<const T *>(buffers[5]);
        p.d_last = static_cast<const T *>(buffers[6]);
        p.dx = static_cast<T *>(buffers[7]);
        p.d_weight = buffers[8];
        p.d_bias = buffers[2] != nullptr ? buffers[9] : nullptr;
        p.d_initial = static_cast<T *>(buffers[10]);
        p.parts = static_cast<float *>(buffers[11]);
        const bool vector = rows_aligned({p.x, p.dy, p.dx}, d->x_stride, d->channels, sizeof(T), V);
        p.groups = vector ? d->channels / V : d->channels;
        p.run = backward_run(*d);
        p.n_runs = (d->tokens + p.run - 1) / p.run;
        with_width(d->width, [&](auto width) {
            constexpr int W = decltype(width)::value;
            if (p.n_runs > 0) {
                const unsigned blocks = blocks_for(static_cast<uint64_t>(p.groups) * p.n_runs, CONV_THREADS);
                if (vector) short_conv_backward_kernel<T, W, V><<<blocks, CONV_THREADS, 0, stream>>>(p);
                else short_conv_backward_kernel<T, W, 1><<<blocks, CONV_THREADS, 0, stream>>>(p);
            }
            if (W > 1 && p.initial != nullptr && d->sequences > 0)
                short_conv_initial_kernel<T, W><<<blocks_for(static_cast<uint64_t>(d->sequences) * d->channels, CONV_THREADS),
                                                  CONV_THREADS, 0, stream>>>(p);
        });
        short_conv_sum_kernel<T><<<blocks_for(static_cast<uint64_t>(d->channels) * (d->width + 1), 32), 256, 0, stream>>>(p, d->width);
    });
    launch_ok();
}

void short_conv_step(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "short_conv_step: 1..8 taps of the inputs' type or float");
    if (d == nullptr || d->channels == 0 || d->tokens == 0) return;
    if (d->tokens > 65535 || d->sequences >= (1u << 31) || (buffers[3] == nullptr && d->sequences < d->tokens)) {
        set_status(BPL_ERR_ARGUMENT, "short_conv_step: at most 65535 rows, and a state for every row");
        return;
    }
    if (!given(buffers, {0, 1, 5}, "short_conv_step: null buffer") ||
        (d->width > 1 && d->sequences > 0 && !given(buffers, {4}, "short_conv_step: null buffer")))
        return;
    with_type(d->dtype, [&](auto type) {
        using T = decltype(type);
        ConvStepArgs<T> p = {};
        p.x = static_cast<const T *>(buffers[0]); p.weight = buffers[1]; p.bias = buffers[2];
        p.slots = static_cast<const int *>(buffers[3]); p.state = static_cast<T *>(buffers[4]); p.y = static_cast<T *>(buffers[5]);
        p.x_stride = d->x_stride; p.rows = d->tokens; p.pool = d->sequences; p.channels = d->channels;
        p.silu = (d->flags & BPL_CONV_SILU) != 0; p.wide = d->weight_dtype == BPL_FLOAT;
        with_width(d->width, [&](auto width) {
            constexpr int W = decltype(width)::value;
            short_conv_step_kernel<T, W><<<dim3(blocks_for(d->channels, CONV_THREADS), d->tokens), CONV_THREADS, 0, stream>>>(p);
        });
    });
    launch_ok();
}

}  // extern "C"
