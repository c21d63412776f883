// Rows of a table that tokens name, scaled (no counterpart in brainpylib), and the gradient of the table:
//
//     y[t] = scale w[id_t];   dw[v] = scale sum_{t: id_t = v} dy[t]
//
// Bound by memory: the lookup reads the rows and writes them, the gradient reads dy once and writes the whole table.  The
// gradient uses no atomics on values, so the same call gives the same bits: tokens are sorted by (id, place), equal runs of
// sorted tokens are summed in order, and what a row has in several runs is joined in order.  32,768 tokens, 64,000 rows of 2048 in 16 bits:
// lookup 29 us, sorting 27, sums and zeros 86 to 90 (4.5 TB/s), joining 14.
#include <initializer_list>
#include <type_traits>

#include "sequence.cuh"

namespace bpl {
namespace {

template<typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

// V neighbouring elements; those of 16 bits as the words they lie in (an array of them would take a register for each)
template<typename T, int V>
using Raw = std::conditional_t<sizeof(T) == 2 && V == 8, uint4, Vec<T, V>>;
template<typename T, int V>
__device__ __forceinline__ void elements(const Raw<T, V> &raw, float (&to)[V]) {
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
__device__ __forceinline__ Raw<T, V> raw_of(const float (&from)[V]) {
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

// ---- lookup ------------------------------------------------------------------------------------------------------------
constexpr int LOOKUP_THREADS = 128;

template<typename T, typename I>
struct LookupArgs {
    const I *ids;
    const T *weight;
    T *y;
    long long weight_stride;
    uint32_t tokens, vocabulary, vectors;      // vectors: of a row
    uint32_t per_row;                          // threads that share a row: a power of two
    float scale;
};

// A thread has up to four vectors of a row on their way at once.
template<typename T, typename I, int V>
__global__ __launch_bounds__(LOOKUP_THREADS) void embedding_kernel(const LookupArgs<T, I> p) {
    using Row = Raw<T, V>;
    const uint32_t t = blockIdx.x * (LOOKUP_THREADS / p.per_row) + threadIdx.x / p.per_row, part = threadIdx.x % p.per_row;
    if (t >= p.tokens) return;
    const long long id = static_cast<long long>(__ldg(p.ids + t));
    const bool good = id >= 0 && id < static_cast<long long>(p.vocabulary);
    const Row *from = reinterpret_cast<const Row *>(p.weight + (good ? id : 0) * p.weight_stride);
    Row *to = reinterpret_cast<Row *>(p.y + static_cast<size_t>(t) * p.vectors * V);
    const float missing = id < 0 ? 0.0f : __int_as_float(0x7fffffff);
    for (uint32_t c = part; c < p.vectors; c += 4 * p.per_row) {
        Row r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (good && c + i * p.per_row < p.vectors) r[i] = from[c + i * p.per_row];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[V];
            elements<T, V>(r[i], v);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = good ? v[k] * p.scale : missing;
            r[i] = raw_of<T, V>(v);
            if (c + i * p.per_row < p.vectors) to[c + i * p.per_row] = r[i];
        }
    }
}

// ---- sorting -------------------------------------------------------------------------------------------------------------
// Stable, by digits from the lowest (least significant digit first): tokens of a block are ranked among those with the same digit
// by votes of a warp over 32 tokens at a time, by counters of the warps in front, and by the counters of all blocks.  A key is the
// id, or the vocabulary for what has no gradient, which so comes last.
constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32, SORT_ROUNDS = 4;
constexpr uint32_t SORT_TILE = SORT_THREADS * SORT_ROUNDS;      // tokens that a block ranks at once
constexpr uint32_t MAX_BITS = 11, MAX_BINS = 1u << MAX_BITS;
constexpr uint32_t MAX_SORT_BLOCKS = 64;        // (every block reads the counters of all)

struct SortPass {
    const void *ids;                       // of the first pass, else null
    const uint32_t *keys, *places;         // of the pass in front
    uint32_t *new_keys, *new_places;
    uint32_t *counts, *next_counts;        // [bins][blocks]; of the next pass, else null
    uint32_t tokens, vocabulary, shift, bits, blocks, tiles;      // tiles: of a block
    bool wide;                             // ids are of 64 bits
};

__device__ __forceinline__ uint32_t key_of(const SortPass &p, uint32_t i) {
    if (p.ids == nullptr) return __ldcg(p.keys + i);
    const long long id = p.wide ? static_cast<const long long *>(p.ids)[i] : static_cast<const int *>(p.ids)[i];
    return id >= 0 && id < static_cast<long long>(p.vocabulary) ? static_cast<uint32_t>(id) : p.vocabulary;
}

// Exclusive prefix sums of `n` counters of shared memory, by the whole block; `sums` has a word for every warp and one more.
__device__ __forceinline__ void prefix(uint32_t *counts, uint32_t n, uint32_t *sums) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, each = (n + SORT_THREADS - 1) / SORT_THREADS;
    const uint32_t from = threadIdx.x * each;
    uint32_t mine = 0;
    for (uint32_t i = from; i < min(from + each, n); ++i) mine += counts[i];
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(FULL_MASK, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    uint32_t base = upto - mine;
    for (uint32_t w = 0; w < warp; ++w) base += sums[w];
    for (uint32_t i = from; i < min(from + each, n); ++i) {
        const uint32_t c = counts[i];
        counts[i] = base;
        base += c;
    }
    __syncthreads();
}

// Counters of the first pass; those of the second are cleared.
__global__ __launch_bounds__(SORT_THREADS) void count_kernel(const SortPass p) {
    __shared__ uint32_t bins[MAX_BINS];
    const uint32_t n_bins = 1u << p.bits;
    for (uint32_t i = threadIdx.x; i < n_bins; i += SORT_THREADS) bins[i] = 0;
    __syncthreads();
    const uint32_t from = blockIdx.x * p.tiles * SORT_TILE, to = min(p.tokens, from + p.tiles * SORT_TILE);
    for (uint32_t i = from + threadIdx.x; i < to; i += SORT_THREADS) atomicAdd(&bins[(key_of(p, i) >> p.shift) & (n_bins - 1)], 1u);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n_bins; i += SORT_THREADS) {
        p.counts[static_cast<size_t>(i) * p.blocks + blockIdx.x] = bins[i];
        if (p.next_counts != nullptr) p.next_counts[static_cast<size_t>(i) * p.blocks + blockIdx.x] = 0;
    }
}

struct SortShared {
    uint16_t ranks[SORT_WARPS][MAX_BINS];     // tokens of a digit in a warp, then in the warps in front of it
    uint32_t next[MAX_BINS];                  // where the next token of a digit goes
    uint32_t sums[SORT_WARPS + 1];
};

// One tile: `key` of the tokens of this thread (round r: token 32 r + lane of its warp) to their places.  `next` moves on.
__device__ __forceinline__ void place_tile(SortShared &s, const SortPass &p, uint32_t base, uint32_t count) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, n_bins = 1u << p.bits;
    for (uint32_t i = lane; i < n_bins; i += 32) s.ranks[warp][i] = 0;
    __syncthreads();
    uint32_t key[SORT_ROUNDS], place[SORT_ROUNDS], rank[SORT_ROUNDS];
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const uint32_t i = (warp * SORT_ROUNDS + r) * 32 + lane;
        key[r] = i < count ? key_of(p, base + i) : 0u;
        place[r] = i < count && p.ids == nullptr ? __ldcg(p.places + base + i) : base + i;
    }
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const uint32_t i = (warp * SORT_ROUNDS + r) * 32 + lane;
        const bool there = i < count;
        const uint32_t digit = (key[r] >> p.shift) & (n_bins - 1);
        const uint32_t same = __match_any_sync(FULL_MASK, there ? digit : MAX_BINS);
        const uint32_t before = there ? s.ranks[warp][digit] : 0u;
        __syncwarp();
        if (there && lane == 31 - __clz(same)) s.ranks[warp][digit] = static_cast<uint16_t>(before + __popc(same));
        __syncwarp();
        rank[r] = before + __popc(same & ((1u << lane) - 1));
    }
    __syncthreads();
    // counters of a warp become those of the warps in front of it; `next` stays this tile's until all have read it
    uint32_t total[MAX_BINS / SORT_THREADS];
#pragma unroll
    for (uint32_t k = 0; k < MAX_BINS / SORT_THREADS; ++k) {
        const uint32_t b = threadIdx.x + k * SORT_THREADS;
        total[k] = 0;
        if (b >= n_bins) continue;
        uint32_t sum = 0;
        for (int w = 0; w < SORT_WARPS; ++w) {
            const uint32_t c = s.ranks[w][b];
            s.ranks[w][b] = static_cast<uint16_t>(sum);
            sum += c;
        }
        total[k] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const uint32_t i = (warp * SORT_ROUNDS + r) * 32 + lane;
        const uint32_t digit = (key[r] >> p.shift) & (n_bins - 1);
        if (i < count) {
            const uint32_t to = s.next[digit] + s.ranks[warp][digit] + rank[r];
            p.new_keys[to] = key[r];
            p.new_places[to] = place[r];
            // the next pass counts what of its digits its blocks will hold: places are known here
            if (p.next_counts != nullptr)
                atomicAdd(p.next_counts + static_cast<size_t>(key[r] >> (p.shift + p.bits) & (n_bins - 1)) * p.blocks + to / (p.tiles * SORT_TILE), 1u);
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < MAX_BINS / SORT_THREADS; ++k)
        if (threadIdx.x + k * SORT_THREADS < n_bins) s.next[threadIdx.x + k * SORT_THREADS] += total[k];
    __syncthreads();
}

__global__ __launch_bounds__(SORT_THREADS) void place_kernel(const SortPass p) {
    extern __shared__ __align__(16) unsigned char shared[];
    SortShared &s = *reinterpret_cast<SortShared *>(shared);
    pdl_wait();
    // where a block's first token of a digit goes: behind all tokens of smaller digits, and those of this one in the blocks in front
    const uint32_t n_bins = 1u << p.bits;
    uint32_t ahead[MAX_BINS / SORT_THREADS];
#pragma unroll
    for (uint32_t k = 0; k < MAX_BINS / SORT_THREADS; ++k) {
        const uint32_t i = threadIdx.x + k * SORT_THREADS;
        uint32_t mine = 0, all = 0;
        if (i < n_bins)
#pragma unroll 8
            for (uint32_t b = 0; b < p.blocks; ++b) {
                const uint32_t c = __ldcg(p.counts + static_cast<size_t>(i) * p.blocks + b);
                mine += b < blockIdx.x ? c : 0u;
                all += c;
            }
        ahead[k] = mine;
        s.next[i] = all;
    }
    __syncthreads();
    prefix(s.next, MAX_BINS, s.sums);
#pragma unroll
    for (uint32_t k = 0; k < MAX_BINS / SORT_THREADS; ++k) s.next[threadIdx.x + k * SORT_THREADS] += ahead[k];
    __syncthreads();
    const uint32_t from = blockIdx.x * p.tiles * SORT_TILE, to = min(p.tokens, from + p.tiles * SORT_TILE);
    for (uint32_t at = from; at < to; at += SORT_TILE) place_tile(s, p, at, min(SORT_TILE, to - at));
}

// All passes of up to SORT_TILE tokens, by one block; what a pass writes, the next one reads behind the barriers.
__global__ __launch_bounds__(SORT_THREADS) void sort_small_kernel(SortPass p, uint32_t *keys, uint32_t *places, uint32_t *other_keys,
                                                                  uint32_t *other_places, uint32_t passes) {
    extern __shared__ __align__(16) unsigned char shared[];
    SortShared &s = *reinterpret_cast<SortShared *>(shared);
    for (uint32_t pass = 0; pass < passes; ++pass) {
        p.shift = pass * p.bits;
        // (the last pass writes `keys` and `places`)
        const bool out = (passes - 1 - pass) % 2 == 0;
        p.new_keys = out ? keys : other_keys;
        p.new_places = out ? places : other_places;
        for (uint32_t i = threadIdx.x; i < MAX_BINS; i += SORT_THREADS) s.next[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < p.tokens; i += SORT_THREADS) atomicAdd(&s.next[(key_of(p, i) >> p.shift) & ((1u << p.bits) - 1)], 1u);
        __syncthreads();
        prefix(s.next, MAX_BINS, s.sums);
        place_tile(s, p, 0, p.tokens);
        p.ids = nullptr;
        p.keys = p.new_keys;
        p.places = p.new_places;
    }
}

// ---- sums of sorted tokens ------------------------------------------------------------------------------------------------
constexpr int SUM_THREADS = 128;
constexpr uint32_t ZERO_ROWS = 64;            // rows of the table that a block looks for

template<typename T>
struct SumArgs {
    const T *dy;
    T *dw;
    const uint32_t *keys, *places;
    float *head, *tail;          // [runs][width]: what a run has of a row that began before it, and of one that goes on behind it
    uint32_t tokens, vocabulary, width, run, runs, slabs;
    float scale;
};

template<typename T, int V>
__device__ __forceinline__ void write_row(const SumArgs<T> &p, uint32_t row, uint32_t c, const float (&sum)[V]) {
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = sum[k] * p.scale;
    *reinterpret_cast<Raw<T, V> *>(p.dw + static_cast<size_t>(row) * p.width + c) = raw_of<T, V>(v);
}
template<int V>
__device__ __forceinline__ void write_part(float *to, const float (&sum)[V]) {
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int k = 0; k < V; k += 4) *reinterpret_cast<float4 *>(to + k) = make_float4(sum[k], sum[k + 1], sum[k + 2], sum[k + 3]);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) to[k] = sum[k];
    }
}
template<int V>
__device__ __forceinline__ void read_part(const float *from, float (&part)[V]) {
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const float4 f = __ldcg(reinterpret_cast<const float4 *>(from + k));
            part[k] = f.x; part[k + 1] = f.y; part[k + 2] = f.z; part[k + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) part[k] = __ldcg(from + k);
    }
}

// Zeros into the rows of the table that no token names.
template<typename T, int V>
__device__ __forceinline__ void zero_rows(const SumArgs<T> &p, uint32_t first) {
    __shared__ bool missing[ZERO_ROWS];
    const uint32_t rows = min(ZERO_ROWS, p.vocabulary - first);
    if (threadIdx.x < rows) {
        uint32_t lo = 0, hi = p.tokens;
        const uint32_t want = first + threadIdx.x;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (__ldcg(p.keys + mid) < want) lo = mid + 1; else hi = mid;
        }
        missing[threadIdx.x] = lo >= p.tokens || __ldcg(p.keys + lo) != want;
    }
    __syncthreads();
    const float none[V] = {};
    const Raw<T, V> zero = raw_of<T, V>(none);
    for (uint32_t r = 0; r < rows; ++r) {
        if (!missing[r]) continue;
        Raw<T, V> *to = reinterpret_cast<Raw<T, V> *>(p.dw + static_cast<size_t>(first + r) * p.width);
        for (uint32_t c = threadIdx.x; c < p.width / V; c += SUM_THREADS) to[c] = zero;
    }
}

// Blocks below runs * slabs: a run of sorted tokens, V neighbouring columns a thread.  The others: zeros.
template<typename T, int V>
__global__ __launch_bounds__(SUM_THREADS) void sum_kernel(const SumArgs<T> p) {
    constexpr int AHEAD = 8;
    pdl_wait();
    const uint32_t b = blockIdx.x, summing = p.runs * p.slabs;
    if (b >= summing) return zero_rows<T, V>(p, (b - summing) * ZERO_ROWS);
    const uint32_t run = b / p.slabs, c = (b % p.slabs * SUM_THREADS + threadIdx.x) * V;
    const uint32_t from = run * p.run, to = min(p.tokens, from + p.run);
    if (c >= p.width) return;
    float sum[V] = {};
    uint32_t row = __ldcg(p.keys + from);
    bool begun_before = from > 0 && __ldcg(p.keys + from - 1) == row;
    for (uint32_t at = from; at < to && row < p.vocabulary; at += AHEAD) {
        Raw<T, V> r[AHEAD];
        uint32_t key[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            key[i] = at + i < to ? __ldcg(p.keys + at + i) : p.vocabulary;
            if (key[i] < p.vocabulary)
                r[i] = *reinterpret_cast<const Raw<T, V> *>(p.dy + static_cast<size_t>(__ldcg(p.places + at + i)) * p.width + c);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (at + i >= to) break;
            if (key[i] != row) {
                if (begun_before) write_part<V>(p.head + static_cast<size_t>(run) * p.width + c, sum);
                else write_row<T, V>(p, row, c, sum);
                begun_before = false;
                row = key[i];
                if (row >= p.vocabulary) return;          // what has no gradient comes last
#pragma unroll
                for (int k = 0; k < V; ++k) sum[k] = 0.0f;
            }
            float v[V];
            elements<T, V>(r[i], v);
#pragma unroll
            for (int k = 0; k < V; ++k) sum[k] += v[k];
        }
    }
    if (row >= p.vocabulary) return;
    const bool goes_on = to < p.tokens && __ldcg(p.keys + to) == row;
    if (begun_before) write_part<V>(p.head + static_cast<size_t>(run) * p.width + c, sum);
    else if (goes_on) write_part<V>(p.tail + static_cast<size_t>(run) * p.width + c, sum);
    else write_row<T, V>(p, row, c, sum);
}

// Rows that several runs have tokens of: the block of the run in which the row begins adds the parts in order.
template<typename T, int V>
__global__ __launch_bounds__(SUM_THREADS) void join_kernel(const SumArgs<T> p) {
    constexpr int AHEAD = 8;
    pdl_wait();
    const uint32_t run = blockIdx.x / p.slabs, c = (blockIdx.x % p.slabs * SUM_THREADS + threadIdx.x) * V;
    const uint32_t from = run * p.run, to = from + p.run;
    if (to >= p.tokens) return;
    const uint32_t row = __ldcg(p.keys + to - 1);
    if (row >= p.vocabulary || __ldcg(p.keys + to) != row) return;                      // nothing goes on
    if (from > 0 && __ldcg(p.keys + from - 1) == row) return;                           // began before: another block's
    // the runs that hold more of it: found by halves, keys being sorted
    uint32_t lo = run + 1, hi = p.runs;           // the run at `lo` begins with the row; that at `hi` does not
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (__ldcg(p.keys + mid * p.run) == row) lo = mid; else hi = mid;
    }
    if (c >= p.width) return;
    float sum[V];
    read_part<V>(p.tail + static_cast<size_t>(run) * p.width + c, sum);
    for (uint32_t r = run + 1; r < hi; r += AHEAD) {
        float part[AHEAD][V];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (r + i < hi) read_part<V>(p.head + static_cast<size_t>(r + i) * p.width + c, part[i]);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (r + i < hi) sum[k] += part[i][k];
    }
    write_row<T, V>(p, row, c, sum);
}

// ---- launches ------------------------------------------------------------------------------------------------------------
struct BackwardPlan {
    uint32_t passes, bits, blocks, tiles, run, runs;
    size_t keys, counts, parts;          // bytes of one array of words a token, of the counters, of one array of parts
    size_t bytes() const { return 4 * keys + 2 * counts + 2 * parts; }
};
BackwardPlan plan_backward(const bpl_embedding_descriptor &d) {
    BackwardPlan q = {};
    uint32_t total = 1;
    while (total < 32 && (d.vocabulary >> total) != 0) ++total;        // keys are 0 .. vocabulary
    q.passes = (total + MAX_BITS - 1) / MAX_BITS;
    q.bits = (total + q.passes - 1) / q.passes;
    const uint32_t all = (d.tokens + SORT_TILE - 1) / SORT_TILE;
    q.tiles = (all + MAX_SORT_BLOCKS - 1) / MAX_SORT_BLOCKS;
    q.blocks = q.tiles ? (all + q.tiles - 1) / q.tiles : 0;
    // Runs: a thousand of them where there are tokens enough, so that many SMs read, and parts stay few beside the tokens.
    q.run = 16;
    while (q.run < 256 && d.tokens / q.run > 1024) q.run *= 2;
    q.runs = (d.tokens + q.run - 1) / q.run;
    auto rounded = [](size_t n) { return (n + 255) / 256 * 256; };
    q.keys = rounded(sizeof(uint32_t) * static_cast<size_t>(d.tokens));
    q.counts = q.blocks > 1 ? rounded(sizeof(uint32_t) * static_cast<size_t>(q.blocks) << q.bits) : 0;
    q.parts = q.runs > 1 ? rounded(sizeof(float) * static_cast<size_t>(q.runs) * d.width) : 0;
    return q;
}

const bpl_embedding_descriptor *checked(const char *opaque, size_t opaque_len, const char *what) {
    const auto *d = unpack<bpl_embedding_descriptor>(opaque, opaque_len);
    if (d == nullptr) return nullptr;
    if (d->dtype > BPL_BFLOAT16 || d->tokens >= (1u << 31) || d->vocabulary >= (1u << 31) || d->width >= (1u << 28)) {
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

template<typename F>
void with_type(uint32_t dtype, F f) {
    if (dtype == BPL_FLOAT) f(float());
    else if (dtype == BPL_HALF) f(__half());
    else f(__nv_bfloat16());
}

template<typename T, typename I>
void lookup(cudaStream_t stream, void **b, const bpl_embedding_descriptor &d) {
    constexpr int V = 16 / sizeof(T);
    LookupArgs<T, I> p = {};
    p.ids = static_cast<const I *>(b[0]);
    p.weight = static_cast<const T *>(b[1]);
    p.y = static_cast<T *>(b[2]);
    p.weight_stride = d.weight_stride; p.tokens = d.tokens; p.vocabulary = d.vocabulary; p.scale = d.scale;
    const bool vector = d.width % V == 0 && d.weight_stride % V == 0 && aligned16(b[1]) && aligned16(b[2]);
    p.vectors = vector ? d.width / V : d.width;
    // four vectors of a row to a thread, so that a block has several rows on their way where they are short
    p.per_row = 1;
    while (p.per_row < LOOKUP_THREADS && p.per_row * 4 < p.vectors) p.per_row *= 2;
    const uint32_t rows = LOOKUP_THREADS / p.per_row, blocks = (d.tokens + rows - 1) / rows;
    if (vector) embedding_kernel<T, I, V><<<blocks, LOOKUP_THREADS, 0, stream>>>(p);
    else embedding_kernel<T, I, 1><<<blocks, LOOKUP_THREADS, 0, stream>>>(p);
}

template<typename T, int V>
void sums(cudaStream_t stream, SumArgs<T> p) {
    p.slabs = (p.width + SUM_THREADS * V - 1) / (SUM_THREADS * V);
    const uint32_t zeros = (p.vocabulary + ZERO_ROWS - 1) / ZERO_ROWS;
    launch_dependent(sum_kernel<T, V>, dim3(p.runs * p.slabs + zeros), dim3(SUM_THREADS), 0, stream, p);
    if (p.runs > 1) launch_dependent(join_kernel<T, V>, dim3(p.runs * p.slabs), dim3(SUM_THREADS), 0, stream, p);
}

bool sort(cudaStream_t stream, const bpl_embedding_descriptor &d, const BackwardPlan &q, const void *ids, uint32_t *const (&arrays)[4],
          uint32_t *counts) {
    SortPass p = {};
    p.ids = ids; p.counts = counts; p.tokens = d.tokens; p.vocabulary = d.vocabulary; p.bits = q.bits; p.blocks = q.blocks; p.tiles = q.tiles;
    p.wide = d.wide_ids != 0;
    constexpr unsigned bytes = sizeof(SortShared);
    if (q.blocks <= 1) {
        if (!allow_shared<sort_small_kernel>(bytes)) return false;
        sort_small_kernel<<<1, SORT_THREADS, bytes, stream>>>(p, arrays[0], arrays[1], arrays[2], arrays[3], q.passes);
        return true;
    }
    if (!allow_shared<place_kernel>(bytes)) return false;
    for (uint32_t pass = 0; pass < q.passes; ++pass) {
        const bool out = (q.passes - 1 - pass) % 2 == 0;
        p.shift = pass * q.bits;
        p.new_keys = arrays[out ? 0 : 2];
        p.new_places = arrays[out ? 1 : 3];
        // (passes are up to three: counters of the one behind the next take the place of this one's)
        p.counts = counts + (pass % 2) * q.counts / sizeof(uint32_t);
        p.next_counts = pass + 1 < q.passes ? counts + ((pass + 1) % 2) * q.counts / sizeof(uint32_t) : nullptr;
        if (pass == 0) count_kernel<<<q.blocks, SORT_THREADS, 0, stream>>>(p);
        else if (p.next_counts != nullptr) cudaMemsetAsync(p.next_counts, 0, q.counts, stream);
        if (pass > 0 && p.next_counts != nullptr) place_kernel<<<q.blocks, SORT_THREADS, bytes, stream>>>(p);
        else launch_dependent(place_kernel, dim3(q.blocks), dim3(SORT_THREADS), bytes, stream, p);
        p.ids = nullptr;
        p.keys = p.new_keys;
        p.places = p.new_places;
    }
    return true;
}

}  // namespace

size_t embedding_backward_workspace_bytes(const char *opaque, size_t opaque_len) {
    if (opaque == nullptr || opaque_len != sizeof(bpl_embedding_descriptor)) return 0;
    return plan_backward(*reinterpret_cast<const bpl_embedding_descriptor *>(opaque)).bytes();
}

}  // namespace bpl

using namespace bpl;

extern "C" {

void embedding(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "embedding: fewer than 2^31 tokens and rows, and 2^28 columns");
    if (d == nullptr || d->tokens == 0 || d->width == 0) return;
    if (!given(buffers, {0, 2}, "embedding: null buffer") || (d->vocabulary > 0 && !given(buffers, {1}, "embedding: null buffer"))) return;
    with_type(d->dtype, [&](auto type) {
        using T = decltype(type);
        if (d->wide_ids) lookup<T, long long>(stream, buffers, *d);
        else lookup<T, int>(stream, buffers, *d);
    });
    launch_ok();
}

void embedding_backward(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len, "embedding_backward: fewer than 2^31 tokens and rows, and 2^28 columns");
    if (d == nullptr || d->vocabulary == 0 || d->width == 0) return;
    if (!given(buffers, {2}, "embedding_backward: null buffer") ||
        (d->tokens > 0 && !given(buffers, {0, 1, 3}, "embedding_backward: null buffer")))
        return;
    if (d->tokens == 0) {
        with_type(d->dtype, [&](auto type) {
            cudaMemsetAsync(buffers[2], 0, sizeof(type) * static_cast<size_t>(d->vocabulary) * d->width, stream);
        });
        launch_ok();
        return;
    }
    const BackwardPlan q = plan_backward(*d);
    char *at = static_cast<char *>(buffers[3]);
    uint32_t *arrays[4];
    for (auto &a : arrays) {
        a = reinterpret_cast<uint32_t *>(at);
        at += q.keys;
    }
    if (!sort(stream, *d, q, buffers[0], arrays, reinterpret_cast<uint32_t *>(at))) {
        set_status(BPL_ERR_CUDA, "embedding_backward: shared memory");
        return;
    }
    at += 2 * q.counts;
    with_type(d->dtype, [&](auto type) {
        using T = decltype(type);
        constexpr int V = 16 / sizeof(T);
        SumArgs<T> p = {};
        p.dy = static_cast<const T *>(buffers[1]); p.dw = static_cast<T *>(buffers[2]);
        p.keys = arrays[0]; p.places = arrays[1];
        p.head = reinterpret_cast<float *>(at); p.tail = reinterpret_cast<float *>(at + q.parts);
        p.tokens = d->tokens; p.vocabulary = d->vocabulary; p.width = d->width; p.run = q.run; p.runs = q.runs; p.scale = d->scale;
        // (parts of sums are read and written in 16 bytes, too)
        if (d->width % V == 0 && aligned16(p.dy) && aligned16(p.dw) && aligned16(p.head)) sums<T, V>(stream, p);
        else sums<T, 1>(stream, p);
    });
    launch_ok();
}

}  // extern "C"
