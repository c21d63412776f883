// The walk of decay_attention.cuh on tensor cores, for bfloat16.  With more than 128 elements to a head of q and k, two blocks share these
// out: products of q and k, and states read out, are sums over them, so that their results add up.
//
// Tokens go by in chunks of 64.  With the columns of the chunk's tokens, S the state in front of it (turned: a row for every column of
// v), a the decay and n the tokens there are:
//
//     P = (Q K^T) . a^(i - j), j <= i          M tokens i, N tokens j              P as two numbers of 16 bits
//     O = V^T P^T + (S Q^T) . a^(i + 1)        M columns of v, N tokens i          S as two numbers of 16 bits
//     S = a^n S + U, U = (V . a^(n - 1 - j))^T K   M columns of v, N elements of k     the factor as three numbers of 16 bits
//
// Operands of products have 16 bits, 8 of them for the number.  Split into two of these, P and the state that a chunk reads lose 2^-17 of
// themselves, and the result is off by what rounding it once is off by (rounded to 16 bits each: 1.41 times that).  Three, for what goes
// into the state, keep 24 bits.
//
// S stays in registers in 32 bits and is added to with one rounding a chunk; U, what a chunk brings, is all that accumulates in tensor
// memory.  (Accumulators cut off what they cannot hold.  With S itself in them a state that forgets nothing lost 2^-24 of itself a chunk:
// 2e-5 to 4e-5 after 16,384 tokens, 3e-7 now.)
//
// A block holds 128 columns of one head of one segment.  Sixteen warps carry S from chunk to chunk and write O of the chunk in front, eight
// split V (and help out with P), two turn P, one lists the chunks and copies tiles ahead, one asks for the products.  The chain from chunk
// to chunk is: U read and added to S, S rounded (300 to 1300 clocks), products with it and into U (1300); everything else goes beside it.
// The warps that hold S take the registers that the others leave (72 for each: 150 bytes on the stack, for which the tiles leave no cache;
// 160 us instead of 138 for the prompts below, as they were with P and S rounded once).
//
// 16,384 tokens of 16 heads of 128 in seven sequences, 144.5 us: 100 for the walk, 144 blocks of 30 chunks of 4500 clocks, 2.6 TB/s, and 43
// for the states that segments hand on.  Bound by the chain and by issue slots.  A third stage for v, q or k has no room beside three terms
// of two chunks.
//
// Tiles lie in the order of memory, also in a walk backwards in time: there the powers of the decay run the other way.  Rows behind a
// chunk's last token belong to others; those of k and v are cleared, what comes of the others is not written.
//
// A number of v that is not finite would reach tokens in front of it (0 times it, in V^T P^T).  It is taken out of the chunk, and the
// column is no number from its token on.
#include <cuda.h>

#include <atomic>
#include <cstring>

#include "decay_attention.cuh"
#include "tensor_core.cuh"

namespace bpl {
namespace {

using bf16 = __nv_bfloat16;

constexpr uint32_t CHUNK = 64, COLUMNS = 128;        // tokens, columns of v
// Warps, in this order (a warp reaches the lanes of tensor memory of its place in its group of four): those that carry the state and write
// O, turn P, copy, ask for products, and split V.
constexpr int STATE_WARPS = 16, TURN_WARPS = 2, SPLIT_WARPS = 8;
constexpr int TURN_HELP = 3;                         // of the warps that split
constexpr int TENSOR_THREADS = 32 * (STATE_WARPS + TURN_WARPS + 2 + SPLIT_WARPS);
constexpr int SLOTS = 8;
constexpr uint32_t TILE = CHUNK * 128;               // bytes of 64 rows of 64 elements

// columns of tensor memory
constexpr uint32_t T_UPDATE = 0, T_ROUNDED = 128, T_REST = 64, T_SCORES = 256, T_EARLIER = 320, T_OWN = 384, T_COLUMNS = 512;

constexpr int TERMS = 3;                             // of what goes into the state

// A chunk, as the copying warp lists it for the others: its tokens lie in memory from row `row` on.
enum : uint32_t { FIRST = 1, BEGINS = 2, LEAVES = 4 };      // of its piece; of its sequence, too; the state behind it is written
struct alignas(16) Chunk {
    uint32_t row, tokens, state, flags;              // tokens: none behind the last chunk; state: of its sequence
};

// STATES: only the states that segments hand on; without q, P and O there is room for more chunks (four of each: 43 us for the pass below,
// two 54).
template<int KP, bool STATES>
struct TensorShared {
    static constexpr uint32_t HALVES = KP / 64;
    static constexpr int HEADS_AHEAD = STATES ? 4 : 2, VALUES_AHEAD = HEADS_AHEAD;      // chunks of q and k, and of v
    static constexpr uint32_t KEYS = STATES ? 0 : TILE, RUN = KEYS + TILE;              // tile of k of a run, from one run to the next
    // for each run of 64 elements of a head the tile of q, then that of k
    unsigned char heads[HEADS_AHEAD][HALVES * RUN];
    unsigned char values[VALUES_AHEAD][2 * TILE];
    unsigned char terms[2][TERMS][2 * TILE];
    unsigned char scores[2][STATES ? 16 : TILE];     // P rounded, and what that leaves of it
    unsigned char out[STATES ? 1 : STATE_WARPS][8 * 64];      // O of 8 tokens and 32 columns, a token to 64 bytes
    float power[CHUNK + 1];                          // of the decay
    alignas(16) float within[16];                    // a^(15 - e) times the scale of P, or backwards a^e
    float lead[CHUNK + 16];                          // a^(i - 15)
    alignas(8) float ahead[CHUNK];                   // what token i of a whole chunk reads of the state in front of it
    Chunk chunks[SLOTS];
    uint8_t poison[SLOTS][COLUMNS];                  // the first token that the walk meets in a chunk whose v is not finite, by column
    uint64_t heads_full[HEADS_AHEAD], heads_empty[HEADS_AHEAD], values_full[VALUES_AHEAD], values_empty[VALUES_AHEAD];
    uint64_t listed, scored, turned, decayed, split[2], spent[2], stated, read_out[2], drained;
    uint32_t tensor, failed;
};

struct Maps {
    CUtensorMap q, k, v;
};

// Registers of a thread: of the warps that hold the state, of the others.  (Multiples of 8, together no more than the launch gives.)
constexpr int STATE_REGISTERS = 88, OTHER_REGISTERS = 48, LAUNCH_REGISTERS = 65536 / TENSOR_THREADS / 8 * 8;
static_assert(32 * STATE_WARPS * STATE_REGISTERS + (TENSOR_THREADS - 32 * STATE_WARPS) * OTHER_REGISTERS <= TENSOR_THREADS * LAUNCH_REGISTERS, "registers");
static_assert(STATE_WARPS % 4 == 0 && TENSOR_THREADS % 128 == 0, "whole groups of four warps change their registers");

// The chunks of a segment, piece by piece.
struct Chunks {
    const DecayWalk &p;
    uint32_t to, next_sequence, at;
    bool whole;                   // all pieces, else only the one that is handed on
    bool inside;
    Piece piece;

    __device__ __forceinline__ Chunks(const DecayWalk &walk, uint32_t g, bool all) : p(walk), whole(all), inside(false) {
        const uint32_t from = g * p.segment;
        to = g + 1 == p.segments ? p.tokens : min(p.tokens, from + p.segment);
        next_sequence = 0;
        at = 0;
        if (!all) {
            inside = handed_on(p, g, piece);
            at = inside ? piece.from : 0;
            return;
        }
        uint32_t begin, which;
        if (from > 0 && p.seq.crosses(from, begin, which)) {
            const uint32_t end = p.seq.at(which + 1);
            piece = Piece{from, min(end, to), which, false, end <= to};
            inside = true;
            at = from;
        }
        next_sequence = p.seq.beginning(from);
    }
    __device__ __forceinline__ bool next(Chunk &c) {
        c = Chunk{};
        if (!inside) {
            if (!whole) return false;
            for (; next_sequence < p.seq.seq.count; ++next_sequence) {
                const uint32_t b = p.seq.at(next_sequence), e = p.seq.at(next_sequence + 1);
                if (b >= to) return false;
                if (e <= b) continue;
                piece = Piece{b, min(e, to), next_sequence, true, e <= to};
                inside = true;
                at = b;
                ++next_sequence;
                break;
            }
            if (!inside) return false;
        }
        c.flags = at == piece.from ? (piece.begins ? FIRST | BEGINS : FIRST) : 0;
        c.tokens = min(CHUNK, piece.to - at);
        c.row = p.seq.backwards ? p.seq.seq.tokens - at - c.tokens : at;
        c.state = p.seq.state(piece.sequence);
        at += c.tokens;
        inside = at < piece.to;
        if (!inside && (!whole || (piece.ends && p.last != nullptr))) c.flags |= LEAVES;
        return true;
    }
};

__device__ uint32_t failures;     // blocks whose waits ran out

// A wait for a barrier must not fall two arrivals behind: every wait below is for an arrival that the next one of the same barrier waits
// for in turn.  Waits end: after a second at the latest, and then in all warps.  (Time that the kernels in front take does not count:
// some warps wait for those.)
constexpr long long MOST_CLOCKS = 2000000000;
__device__ __forceinline__ bool wait_long(uint64_t *b, uint32_t parity, const DecayWalk &p, volatile uint32_t *failed) {
    pdl_wait();
    const long long began = clock64();
    while (!barrier_passed(b, parity)) {
        if (*failed || clock64() - began > p.patience) {
            *failed = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool wait(uint64_t *b, uint32_t parity, const DecayWalk &p, volatile uint32_t *failed) {
    return barrier_passed(b, parity) || wait_long(b, parity, p, failed);
}
// by a whole warp, which goes on together
__device__ __forceinline__ bool wait_warp(uint64_t *b, uint32_t parity, const DecayWalk &p, volatile uint32_t *failed) {
    return __all_sync(FULL_MASK, wait(b, parity, p, failed));
}

__device__ __forceinline__ uint32_t pack(float a, float b) {       // a in the low half
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return reinterpret_cast<const uint32_t &>(v);
}
__device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// Two numbers as sums of two of 16 bits each: 2^-17 of them is lost.
__device__ __forceinline__ void pack_twice(float a, float b, uint32_t &rounded, uint32_t &rest) {
    rounded = pack(a, b);
    const float2 r = split(fma2(make_pair(low(rounded), high(rounded)), make_pair(-1.0f, -1.0f), make_pair(a, b)));
    rest = pack(r.x, r.y);
}

// table[at] becomes at most `value`
__device__ void lower(uint8_t *table, uint32_t at, uint32_t value) {
    uint32_t *word = reinterpret_cast<uint32_t *>(table + at / 4 * 4);
    const uint32_t shift = at % 4 * 8;
    uint32_t seen = *word;
    while ((seen >> shift & 255) > value) {
        const uint32_t was = atomicCAS(word, seen, (seen & ~(255u << shift)) | value << shift);
        if (was == seen) break;
        seen = was;
    }
}

// P: row i by lane i of a warp that reaches the lanes of that row, 16 columns at a time.  a^(i - j) is a^(i - j0 - 15) of the row times
// a^(15 - e) of the column j0 + e (backwards a^(j0 - i) a^e), where the first cannot leave the range; else powers are looked up.
// What is not counted is left out, not multiplied by zero.  The blocks of 32 rows and 32 columns on the diagonal go to two warps
// each, those beside it to one; the warps that split V help out.
template<int KP, bool STATES>
__device__ __forceinline__ bool turn(TensorShared<KP, STATES> &s, const DecayWalk &p, uint32_t n, uint32_t tokens, uint32_t from, uint32_t to) {
    const bool backwards = p.seq.backwards;
    const float own_scale = p.own_scale;
    // (The power of the column and the scale first, 2^-30 to 1 times the scale: what that power makes smaller that of the row makes larger
    // again, so that nothing is infinite on the way that is not in the end.  Products of tokens from 2^-90 on, and scales, keep their bits.)
    const bool steep = !(s.power[1] >= 0.25f && s.power[1] <= 1.0f) || fabsf(own_scale) < 0x1p-90f;
    const uint32_t lane = threadIdx.x % 32, first = threadIdx.x / 32 % 4 * 32, i = first + lane, tensor = s.tensor, lanes = first << 16;
    // (the scores of a chunk come behind the products that read the P of the chunk before)
    if (!wait_warp(&s.scored, n & 1, p, &s.failed)) return false;
    tensor_fence_after();
#pragma unroll 1
    for (uint32_t j0 = from; j0 < to; j0 += 16) {
        uint32_t x[16];
        tensor_load_16(tensor + lanes + T_SCORES + j0, x);
        const int d = static_cast<int>(i) - static_cast<int>(j0), count = static_cast<int>(tokens) - static_cast<int>(j0);
        const float row = s.lead[max(0, (backwards ? 15 - d : d))];
        tensor_wait_loads();
        if (steep) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                x[e] = __float_as_uint(__uint_as_float(x[e]) * (s.power[min(63, max(0, backwards ? e - d : d - e))] * own_scale));
        } else {
            const pair lead = make_pair(row, row);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(s.within + 2 * e);
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const float2 v = split(mul2(mul2(make_pair(__uint_as_float(x[2 * (e + o)]), __uint_as_float(x[2 * (e + o) + 1])), o == 0 ? w.x : w.y),
                                                lead));
                    x[2 * (e + o)] = __float_as_uint(v.x);
                    x[2 * (e + o) + 1] = __float_as_uint(v.y);
                }
            }
        }
        if (backwards) {
            if (j0 < first + 31 || count < 16) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (e < d || e >= count) x[e] = 0;
            }
        } else if (j0 + 15 > first) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (e > d) x[e] = 0;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t rounded[4], rest[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) pack_twice(__uint_as_float(x[8 * half + 2 * e]), __uint_as_float(x[8 * half + 2 * e + 1]), rounded[e], rest[e]);
            *reinterpret_cast<uint4 *>(s.scores[0] + swizzled(i, j0 / 8 + half)) = make_uint4(rounded[0], rounded[1], rounded[2], rounded[3]);
            *reinterpret_cast<uint4 *>(s.scores[1] + swizzled(i, j0 / 8 + half)) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
        }
    }
    fence_shared_for_tensor();
    tensor_fence_before();
    barrier_arrive(&s.turned);
    return true;
}

template<int KP, bool STATES>
__global__ __launch_bounds__(TENSOR_THREADS, 1) void decay_tensor_kernel(const DecayWalk p, const __grid_constant__ Maps maps) {
    extern __shared__ __align__(1024) unsigned char shared[];
    using Shared = TensorShared<KP, STATES>;
    Shared &s = *reinterpret_cast<Shared *>(shared);
    constexpr uint32_t HALVES = Shared::HALVES, KEYS = Shared::KEYS, RUN = Shared::RUN;
    constexpr int HEADS_AHEAD = Shared::HEADS_AHEAD, VALUES_AHEAD = Shared::VALUES_AHEAD;
    const uint32_t slabs = (p.v_size + COLUMNS - 1) / COLUMNS, unit = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    const uint32_t h = unit / slabs, c0 = unit % slabs * COLUMNS, g = blockIdx.y;
    const uint32_t k0 = part * 128, k_size = min(p.k_size - k0, 128u);           // rows of the state of this block
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const bool backwards = p.seq.backwards;
    if (STATES) pdl_launch_dependents();             // (what joins the states waits before it reads them)

    if (threadIdx.x <= CHUNK) s.power[threadIdx.x] = decay_power(p.log_decay[h], threadIdx.x);
    if (threadIdx.x < SLOTS * COLUMNS / 4) reinterpret_cast<uint32_t *>(s.poison)[threadIdx.x] = CHUNK * 0x01010101u;
    if (threadIdx.x == 0) {
        for (int i = 0; i < HEADS_AHEAD; ++i) {
            barrier_init(&s.heads_full[i], 1);
            barrier_init(&s.heads_empty[i], 1);
        }
        for (int i = 0; i < VALUES_AHEAD; ++i) {
            barrier_init(&s.values_full[i], 1);
            barrier_init(&s.values_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            barrier_init(&s.split[i], 32 * SPLIT_WARPS);
            barrier_init(&s.spent[i], 1);
            barrier_init(&s.read_out[i], 1);
        }
        barrier_init(&s.listed, 1);
        barrier_init(&s.scored, 1);
        barrier_init(&s.turned, 32 * (TURN_WARPS + TURN_HELP));
        barrier_init(&s.decayed, 32 * STATE_WARPS);
        barrier_init(&s.stated, 1);
        barrier_init(&s.drained, 1);
        s.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 0) tensor_alloc(&s.tensor, T_COLUMNS);
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tensor = s.tensor, lanes = (warp % 4 * 32) << 16;
    if (threadIdx.x < CHUNK + 16)
        s.lead[threadIdx.x] = static_cast<float>(exp(static_cast<double>(p.log_decay[h]) * (static_cast<int>(threadIdx.x) - 15)));
    if (threadIdx.x < CHUNK) s.ahead[threadIdx.x] = s.power[backwards ? CHUNK - threadIdx.x : threadIdx.x + 1] * p.out_scale;
    // what of P is never counted
    for (uint32_t i = threadIdx.x; i < sizeof(s.scores) / 16; i += TENSOR_THREADS) reinterpret_cast<uint4 *>(s.scores[0])[i] = make_uint4(0, 0, 0, 0);
    fence_shared_for_tensor();
    if (threadIdx.x < 16) s.within[threadIdx.x] = s.power[backwards ? threadIdx.x : 15 - threadIdx.x] * p.own_scale;
    __syncthreads();
    volatile uint32_t *failed = &s.failed;

    // A sequence's first state backwards is the gradient of its last one, and has not decayed when the first token reads it.
    auto late_by = [&](const Chunk &c) { return backwards && (c.flags & BEGINS) ? 1u : 0u; };
    // Chunk n + 1 is listed before the copies of chunk n are asked for: who has seen one of the barriers behind these may read it.
    auto first_chunk = [&](Chunk &c) {
        c.tokens = 0;
        if (wait_warp(&s.listed, 0, p, failed)) c = s.chunks[0];
    };
    auto next_chunk = [&](uint32_t n, Chunk &c) { c = s.chunks[(n + 1) % SLOTS]; };

    if (warp < STATE_WARPS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(STATE_REGISTERS));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(OTHER_REGISTERS));
    if (warp < STATE_WARPS) {
        constexpr uint32_t OWN = KP * 4 / STATE_WARPS;        // columns of the state (elements of k) of a thread
        const uint32_t column = threadIdx.x % 128, quarter = threadIdx.x / 128, i0 = quarter * OWN;
        const bool mine = c0 + column < p.v_size;
        // O of chunk n, 16 tokens and 32 columns to a warp: fragments of 8 tokens turned by way of shared memory
        const uint32_t columns = c0 + warp % 4 * 32 < p.v_size ? min(32u, p.v_size - c0 - warp % 4 * 32) : 0u;
        // S Q^T of a chunk, which makes room for that of the next one: fragments of 8 tokens, or 16 tokens of the thread's column
        auto load_earlier = [&](uint32_t (&earlier)[16]) {
            const uint32_t from = tensor + lanes + T_EARLIER + 16 * quarter;
            if (p.wide_out) {
                tensor_load_16(from, earlier);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) tensor_load_fragment(from + (i % 2 * 16 << 16) + i / 2 * 8, earlier + 4 * i);
            }
            tensor_wait_loads();
        };
        auto read_out = [&](uint32_t n, uint32_t row, uint32_t tokens, uint32_t late, const uint32_t (&earlier)[16]) {
            if (!wait_warp(&s.read_out[n & 1], n / 2 & 1, p, failed)) return false;
            tensor_fence_after();
            const size_t step = static_cast<size_t>(p.heads) * p.parts * p.v_size;
            const size_t at = row * step + (h * p.parts + part) * p.v_size + c0 + warp % 4 * 32;
            const uint32_t from = tensor + lanes + T_OWN + (n & 1) * CHUNK;
            // token i reads the state decayed i + 1 times, less `late`; backwards, i counts from the other end
            const float *factor = s.power + (backwards ? tokens - late : 1 - late);
            const int way = backwards ? -1 : 1;
            const bool plain = tokens == CHUNK && late == 0, poisoned = __any_sync(FULL_MASK, s.poison[n % SLOTS][warp % 4 * 32 + lane] < CHUNK);
            auto spoilt = [&](uint32_t i, uint32_t c) { return poisoned && (backwards ? tokens - 1 - i : i) >= s.poison[n % SLOTS][warp % 4 * 32 + c]; };
            if (!p.wide_out) {
                unsigned char *staged = s.out[warp];
                auto place = [](uint32_t i, uint32_t piece) { return i * 64 + ((piece ^ (i >> 1 & 3)) << 4); };
#pragma unroll
                for (uint32_t group = 0; group < 2; ++group) {
                    const uint32_t t0 = 16 * quarter + 8 * group;
                    uint32_t own[2][4], packed[4];
#pragma unroll
                    for (uint32_t side = 0; side < 2; ++side) tensor_load_fragment(from + (side * 16 << 16) + t0, own[side]);
                    const int i = static_cast<int>(t0 + 2 * (lane % 4)), last = static_cast<int>(tokens) - 1;
                    pair f;                          // (behind the last token: any power will do)
                    if (plain) f = *reinterpret_cast<const pair *>(s.ahead + i);
                    else f = make_pair(factor[way * min(i, last)] * p.out_scale, factor[way * min(i + 1, last)] * p.out_scale);
                    tensor_wait_loads();
#pragma unroll
                    for (uint32_t m = 0; m < 4; ++m) {
                        const uint32_t side = m / 2, r = m % 2 * 2;
                        const uint32_t *e = earlier + 8 * group + 4 * side + r;
                        float2 o = split(fma2(make_pair(__uint_as_float(e[0]), __uint_as_float(e[1])), f,
                                              make_pair(__uint_as_float(own[side][r]), __uint_as_float(own[side][r + 1]))));
                        if (poisoned) {
                            if (spoilt(i, 8 * m + lane / 4)) o.x = __int_as_float(0x7fffffff);
                            if (spoilt(i + 1, 8 * m + lane / 4)) o.y = __int_as_float(0x7fffffff);
                        }
                        packed[m] = pack(o.x, o.y);
                    }
                    store_turned(shared_address(staged + place(lane % 8, lane / 8)), packed[0], packed[1], packed[2], packed[3]);
                    __syncwarp();
                    const uint32_t token = t0 + lane / 4;
                    if (token < tokens && lane % 4 * 8 < columns)
                        *reinterpret_cast<uint4 *>(static_cast<bf16 *>(p.out) + at + token * step + lane % 4 * 8) =
                            *reinterpret_cast<const uint4 *>(staged + place(lane / 4, lane % 4));
                    __syncwarp();
                }
            } else {
                uint32_t own[16];
                tensor_load_16(from + 16 * quarter, own);
                tensor_wait_loads();
                float *to = static_cast<float *>(p.out) + at + lane + 16 * quarter * step;
#pragma unroll
                for (uint32_t k = 0; k < 16; ++k) {
                    const uint32_t i = 16 * quarter + k;
                    if (i < tokens && lane < columns) {
                        const float o = fmaf(__uint_as_float(earlier[k]), factor[way * static_cast<int>(i)] * p.out_scale, __uint_as_float(own[k]));
                        *to = spoilt(i, lane) ? __int_as_float(0x7fffffff) : o;
                    }
                    to += step;
                }
            }
            tensor_fence_before();
            return true;
        };
        // S: elements i0 .. i0 + OWN - 1 of k of the thread's column, in pairs
        pair state[OWN / 2] = {};
        // (to the next element of k in global memory, and from there to the thread's)
        auto down = [&](bool turned) { return turned ? size_t(1) : size_t(p.v_size); };
        auto to_mine = [&](bool turned) { return (k0 + i0) * down(turned) + (c0 + column) * (turned ? size_t(p.k_size) : size_t(1)); };
        if (!STATES) pdl_wait();                     // for the states that segments hand on
        Chunk c;
        first_chunk(c);
        uint32_t row = 0, tokens = 0, late = 0;      // of the chunk in front
        float *end = nullptr;                        // where the state behind it goes, if it does
        bool infinite = false;                       // whether the piece came with numbers that are
        for (uint32_t n = 0;; ++n) {
            uint32_t earlier[16];
            if (n > 0) {                             // a S and what the chunk in front brings, which the products have left
                if (!wait_warp(&s.stated, (n - 1) & 1, p, failed)) break;
                tensor_fence_after();
                next_chunk(n - 1, c);
                const float a = s.power[tokens - late];
                const pair decay = make_pair(a, a);
#pragma unroll
                for (uint32_t k = 0; k < OWN; k += 16) {
                    uint32_t x[16];
                    tensor_load_16(tensor + lanes + T_UPDATE + i0 + k, x);
                    tensor_wait_loads();
#pragma unroll
                    for (uint32_t e = 0; e < 16; e += 2)
                        state[(k + e) / 2] = fma2(state[(k + e) / 2], decay, make_pair(__uint_as_float(x[e]), __uint_as_float(x[e + 1])));
                }
                if (!STATES) load_earlier(earlier);
                if (end != nullptr) {
                    const bool turned = !STATES && p.transposed;
                    const float factor = !STATES && backwards ? s.power[1] : 1.0f;
                    float *at = end + to_mine(turned);
#pragma unroll
                    for (uint32_t e = 0; e < OWN; ++e) {
                        const float2 v = split(state[e / 2]);
                        if (mine && i0 + e < k_size) *at = (e % 2 ? v.y : v.x) * factor;
                        at += down(turned);
                    }
                }
            }
            if (c.tokens > 0) {
                if (c.flags & FIRST) {
                    const bool turned = c.flags & BEGINS ? p.transposed : p.carried_turned;
                    const float *at = nullptr;
                    if (c.flags & BEGINS) {
                        if (p.initial != nullptr) at = p.initial + (static_cast<size_t>(c.state) * p.heads + h) * p.state_size();
                    } else if (!STATES) {
                        at = p.carried + (static_cast<size_t>(g - 1) * p.heads + h) * p.state_size();
                    }
                    infinite = false;
                    if (at == nullptr) {
#pragma unroll
                        for (uint32_t e = 0; e < OWN / 2; ++e) state[e] = 0;
                    } else {
                        at += to_mine(turned);
#pragma unroll
                        for (uint32_t e = 0; e < OWN; e += 2) {
                            const float even = mine && i0 + e < k_size ? __ldcg(at) : 0.0f;
                            at += down(turned);
                            const float odd = mine && i0 + e + 1 < k_size ? __ldcg(at) : 0.0f;
                            at += down(turned);
                            infinite |= !(fabsf(even) < INFINITY) || !(fabsf(odd) < INFINITY);
                            state[e / 2] = make_pair(even, odd);
                        }
                    }
                }
                if (!STATES) {
#pragma unroll
                    for (uint32_t k = 0; k < OWN; k += 16) {
                        uint32_t rounded[8], rest[8];
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e) {
                            const float2 v = split(state[k / 2 + e]);
                            pack_twice(v.x, v.y, rounded[e], rest[e]);
                        }
                        if (infinite)                // (infinity less itself is no number)
#pragma unroll
                            for (uint32_t e = 0; e < 8; ++e) {
                                if ((rounded[e] & 0x7fffu) == 0x7f80u) rest[e] &= 0xffff0000u;
                                if ((rounded[e] & 0x7fff0000u) == 0x7f800000u) rest[e] &= 0xffffu;
                            }
                        tensor_store_8(tensor + lanes + T_ROUNDED + (i0 + k) / 2, rounded);
                        tensor_store_8(tensor + lanes + T_ROUNDED + T_REST + (i0 + k) / 2, rest);
                    }
                    tensor_wait_stores();
                }
                tensor_fence_before();
                barrier_arrive(&s.decayed);
            }
            // (O of the chunk in front stands until the products behind the next one of these)
            if (!STATES && n > 0 && !read_out(n - 1, row, tokens, late, earlier)) break;
            if (c.tokens == 0) break;
            row = c.row;
            tokens = c.tokens;
            late = late_by(c);
            end = !(c.flags & LEAVES) ? nullptr
                  : STATES            ? p.carried + (static_cast<size_t>(g) * p.heads + h) * p.state_size()
                                      : p.last + (static_cast<size_t>(c.state) * p.heads + h) * p.state_size();
        }
    } else if (warp < STATE_WARPS + TURN_WARPS) {
        if constexpr (!STATES) {
            // (row 0 or 32 on) a quarter of the diagonal, or the block beside it
            const bool beside = backwards == (warp % 4 == 0);
            const uint32_t from = backwards ? 32 : 0;
            Chunk c;
            first_chunk(c);
            for (uint32_t n = 0; c.tokens > 0; ++n) {
                if (!turn(s, p, n, c.tokens, from, from + (beside ? 32 : 16))) break;
                next_chunk(n, c);
            }
        }
    } else if (warp == STATE_WARPS + TURN_WARPS) {
        if (lane == 0 && p.patience > 0) {
            prefetch_map(&maps.k);
            prefetch_map(&maps.v);
            if (!STATES) prefetch_map(&maps.q);
            Chunks it(p, g, !STATES);
            Chunk c, after;
            it.next(c);
            s.chunks[0] = c;
            barrier_arrive(&s.listed);
            uint32_t m = 0, n = 0;
            for (; c.tokens > 0; c = after) {
                it.next(after);
                s.chunks[(n + 1) % SLOTS] = after;   // (in the place of one that all are done with)
                uint32_t stage = n % HEADS_AHEAD, at = shared_address(s.heads[stage]);
                if (n >= HEADS_AHEAD && !wait(&s.heads_empty[stage], (n / HEADS_AHEAD - 1) & 1, p, failed)) break;
                uint64_t *full = &s.heads_full[stage];
                barrier_expect(full, HALVES * RUN);
#pragma unroll
                for (uint32_t half = 0; half < HALVES; ++half) {
                    if (!STATES) copy_box(at + half * RUN, &maps.q, k0 + 64 * half, h / p.q.group, c.row, full);
                    copy_box(at + half * RUN + KEYS, &maps.k, k0 + 64 * half, h / p.k.group, c.row, full);
                }
                ++n;
                stage = m % VALUES_AHEAD;
                at = shared_address(s.values[stage]);
                if (m >= VALUES_AHEAD && !wait(&s.values_empty[stage], (m / VALUES_AHEAD - 1) & 1, p, failed)) break;
                full = &s.values_full[stage];
                barrier_expect(full, 2 * TILE);
                copy_box(at, &maps.v, c0, h / p.v.group, c.row, full);
                copy_box(at + TILE, &maps.v, c0 + 64, h / p.v.group, c.row, full);
                ++m;
            }
            // copies on their way end before the block does, also where another warp gave up
            auto ended = [&](uint64_t *b, uint32_t parity) {
                const long long since = clock64();
                while (!barrier_passed(b, parity) && clock64() - since < MOST_CLOCKS) {}
            };
            for (uint32_t i = n > HEADS_AHEAD ? n - HEADS_AHEAD : 0; i < n; ++i) ended(&s.heads_full[i % HEADS_AHEAD], i / HEADS_AHEAD & 1);
            for (uint32_t i = m > VALUES_AHEAD ? m - VALUES_AHEAD : 0; i < m; ++i) ended(&s.values_full[i % VALUES_AHEAD], i / VALUES_AHEAD & 1);
        }
    } else if (warp >= STATE_WARPS + TURN_WARPS + 2) {
        // V times the decays, as numbers of 16 bits, in 32 parts of eight rows and four pieces of 16 bytes each: lane (j, q) has of part
        // 4 r + k, in row 8 r + j, piece q or q + 4 of tile k / 2 (rows with an odd number the other way round: eight lanes reach all banks).
        const uint32_t tid = threadIdx.x - 32 * (STATE_WARPS + TURN_WARPS + 2), q = lane % 4;
        const pair minus = make_pair(-1.0f, -1.0f), zero = make_pair(0.0f, 0.0f);
        // Warps 0 and 1 (and, of the half that has the block beside the diagonal, 4 or 5) turn 16 columns of the diagonal, a chunk behind.
        const uint32_t helper = warp - (STATE_WARPS + TURN_WARPS + 2), help_row = warp % 4;
        const bool helps = !STATES && (backwards ? helper == 0 || helper == 1 || helper == 4 : helper == 0 || helper == 1 || helper == 5);
        // forwards: rows 0: columns 16; rows 32: 32 and 48.  backwards: rows 32: 48; rows 0: 0 and 16
        const uint32_t help_from = backwards ? (help_row == 1 ? 48 : helper == 4 ? 16 : 0) : (help_row == 0 ? 16 : helper == 5 ? 48 : 32);
        // Four parts to a warp.  Where there is P to turn, two or three to those that help, the rest by what else their schedulers have to do:
        // 3, 2, 5, 5, 5, 3, 5 and 4 forwards; backwards the fifth and the sixth change places.  (Four to each: 146 us instead of 144.5 of the
        // prompts above, 22.5 instead of 20.5 of 300 tokens.)  The first part of every warp, in bytes:
        const uint64_t begins = STATES ? 0x1c1814100c080400ull : backwards ? 0x1c17120f0a050300ull : 0x1c17140f0a050300ull;
        const uint32_t first_part = begins >> 8 * helper & 255, last_part = helper + 1 < SPLIT_WARPS ? begins >> 8 * (helper + 1) & 255 : 32;
        Chunk c;
        first_chunk(c);
        uint32_t before = 0;                         // tokens of the chunk before
        for (uint32_t n = 0;; ++n) {
            if (helps && n > 0 && !turn(s, p, n - 1, before, help_from, help_from + 16)) break;
            if (c.tokens == 0) break;
            if (!wait_warp(&s.values_full[n % VALUES_AHEAD], n / VALUES_AHEAD & 1, p, failed) || (n >= 2 && !wait_warp(&s.spent[n & 1], (n / 2 - 1) & 1, p, failed))) break;
            if (!STATES && tid < COLUMNS) s.poison[(n + SLOTS / 2) % SLOTS][tid] = CHUNK;
            unsigned char *from = s.values[n % VALUES_AHEAD], *to = s.terms[n & 1][0];
#pragma unroll 1
            for (uint32_t share = first_part; share < last_part; ++share) {
                const uint32_t j = share / 4 * 8 + lane / 4, half = share % 4 / 2, piece = q + 4 * ((share ^ j) & 1);
                const uint32_t at = half * TILE + swizzled(j, piece);
                const bool there = j < c.tokens;
                const float w = there ? s.power[backwards ? j : c.tokens - 1 - j] * p.state_scale : 0.0f;
                const pair weight = make_pair(w, w);
                pair odd = zero;                     // no number once an element is infinite or none
                uint4 raw = *reinterpret_cast<const uint4 *>(from + at);
                if (!there) *reinterpret_cast<uint4 *>(from + at) = raw = make_uint4(0, 0, 0, 0);
                const uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
                uint32_t t[TERMS][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const pair v = make_pair(low(x[e]), high(x[e]));
                    if (!STATES) odd = fma2(v, zero, odd);
                    pair rest = mul2(v, weight);
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) {
                        const float2 r = split(rest);
                        t[m][e] = pack(r.x, r.y);
                        if (m + 1 < TERMS) rest = fma2(make_pair(low(t[m][e]), high(t[m][e])), minus, rest);
                    }
                }
#pragma unroll
                for (int m = 0; m < TERMS; ++m) *reinterpret_cast<uint4 *>(to + m * 2 * TILE + at) = make_uint4(t[m][0], t[m][1], t[m][2], t[m][3]);
                if (!STATES && sum2(odd) != 0.0f)
#pragma unroll 1
                    for (uint32_t e = 0; e < 8; ++e) {
                        uint16_t *v = reinterpret_cast<uint16_t *>(from + at) + e;
                        if ((*v & 0x7f80) == 0x7f80) {
                            *v = 0;
                            lower(s.poison[n % SLOTS], half * 64 + piece * 8 + e, backwards ? c.tokens - 1 - j : j);
                        }
                    }
            }
            if (c.tokens < CHUNK) {                  // (and of k)
                if (!wait_warp(&s.heads_full[n % HEADS_AHEAD], n / HEADS_AHEAD & 1, p, failed)) break;
                if (tid / 4 >= c.tokens)
                    for (uint32_t k = 0; k < KP / 32; ++k)
                        *reinterpret_cast<uint4 *>(s.heads[n % HEADS_AHEAD] + KEYS + k / 2 * RUN + swizzled(tid / 4, q + 4 * (k & 1))) = make_uint4(0, 0, 0, 0);
            }
            fence_shared_for_tensor();
            barrier_arrive(&s.split[n & 1]);
            before = c.tokens;
            next_chunk(n, c);
        }
    } else {
        const uint32_t chosen = elect_lane(), tensor = __shfl_sync(FULL_MASK, s.tensor, 0);
        Chunk c;
        first_chunk(c);
        auto score = [&](uint32_t n) {              // P: rows of q (and, unused, of k) by rows of k
            const uint32_t at = operand(shared_address(s.heads[n % HEADS_AHEAD]));
#pragma unroll
            for (uint32_t k = 0; k < KP / 16; ++k) {
                const uint32_t from = at + (k / 4 * RUN + k % 4 * 32) / 16;
                multiply(tensor + T_SCORES, from, from + KEYS / 16, product_of(CHUNK, false, false), k > 0, chosen);
            }
            products_arrive(&s.scored, chosen);
        };
        bool more = c.tokens > 0, good = !more || wait_warp(&s.heads_full[0], 0, p, failed);
        if (!STATES && more && good) {
            tensor_fence_after();
            score(0);
        }
        uint32_t n = 0;
        for (; more && good; ++n) {
            const uint32_t stage = shared_address(s.heads[n % HEADS_AHEAD]);
            if (!(good = wait_warp(&s.split[n & 1], n / 2 & 1, p, failed) && wait_warp(&s.decayed, n & 1, p, failed))) break;
            tensor_fence_after();
            const uint32_t keys = operand(stage + KEYS, RUN), terms = operand(shared_address(s.terms[n & 1]), TILE), queries = operand(stage);
            if constexpr (!STATES) {                // (in front of the state's: once those are done, this state is read out)
#pragma unroll
                for (uint32_t m = 0; m < 2; ++m)
#pragma unroll
                    for (uint32_t k = 0; k < KP / 16; ++k)
                        multiply_from_tensor(tensor + T_EARLIER, tensor + T_ROUNDED + m * T_REST + 8 * k,
                                             queries + (k / 4 * RUN + k % 4 * 32) / 16, product_of(CHUNK, false, false), m + k > 0, chosen);
            }
#pragma unroll
            for (uint32_t m = 0; m < TERMS; ++m)
#pragma unroll
                for (uint32_t k = 0; k < CHUNK / 16; ++k)
                    multiply(tensor + T_UPDATE, terms + (m * 2 * TILE + k * 2048) / 16, keys + k * 2048 / 16, product_of(KP, true, true), m + k > 0, chosen);
            products_arrive(&s.stated, chosen);
            products_arrive(&s.spent[n & 1], chosen);
            products_arrive(&s.heads_empty[n % HEADS_AHEAD], chosen);
            if constexpr (STATES) {
                products_arrive(&s.values_empty[n % VALUES_AHEAD], chosen);
            } else {
                const uint32_t values = operand(shared_address(s.values[n % VALUES_AHEAD]), TILE), scores = operand(shared_address(s.scores[0]));
                if (!(good = wait_warp(&s.turned, n & 1, p, failed))) break;
                tensor_fence_after();
#pragma unroll
                for (uint32_t m = 0; m < 2; ++m)
#pragma unroll
                    for (uint32_t k = 0; k < CHUNK / 16; ++k)
                        multiply(tensor + T_OWN + (n & 1) * CHUNK, values + k * 2048 / 16, scores + (m * TILE + k * 32) / 16, product_of(CHUNK, true, false), m + k > 0, chosen);
                products_arrive(&s.read_out[n & 1], chosen);
                products_arrive(&s.values_empty[n % VALUES_AHEAD], chosen);
            }
            next_chunk(n, c);
            more = c.tokens > 0;
            if (more) {                             // (every copy is waited for, so that none is on its way when the block ends)
                if (!(good = wait_warp(&s.heads_full[(n + 1) % HEADS_AHEAD], (n + 1) / HEADS_AHEAD & 1, p, failed))) break;
                tensor_fence_after();
                if (!STATES) score(n + 1);
            }
        }
        // the last arrival of all: none comes when the block has ended
        if (good && n > 0) good = wait_warp(&s.values_empty[(n - 1) % VALUES_AHEAD], (n - 1) / VALUES_AHEAD & 1, p, failed);
        if (!good) {                                // products on their way end before tensor memory is given back
            *failed = 1;
            products_arrive(&s.drained, chosen);
            const long long began = clock64();
            while (!barrier_passed(&s.drained, 0) && clock64() - began < MOST_CLOCKS) {}
        }
    }
    __syncwarp();
    if (warp < STATE_WARPS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(LAUNCH_REGISTERS));
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(LAUNCH_REGISTERS));
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (warp == 0) tensor_free(tensor, T_COLUMNS);
    if (s.failed && threadIdx.x == 0) atomicAdd(&failures, 1u);

    // what the block was to write, where it gave up: no numbers
    const uint32_t columns = min(COLUMNS, p.v_size - c0);
    auto spoil = [&](float *to, bool turned) {
        for (uint32_t i = threadIdx.x; i < k_size * columns; i += TENSOR_THREADS) {
            const uint32_t r = k0 + i / columns, c = c0 + i % columns;
            to[turned ? static_cast<size_t>(c) * p.k_size + r : static_cast<size_t>(r) * p.v_size + c] = __int_as_float(0x7fffffff);
        }
    };
    if (STATES && s.failed) spoil(p.carried + (static_cast<size_t>(g) * p.heads + h) * p.state_size(), false);

    if constexpr (!STATES) {
        const uint32_t from = g * p.segment, to = g + 1 == p.segments ? p.tokens : min(p.tokens, from + p.segment);
        const uint32_t first = p.seq.first(), last = max(p.seq.last(), first);
        if (s.failed && p.last != nullptr)
            for_pieces(p, g, [&](const Piece &piece) {
                if (piece.ends) spoil(p.last + (static_cast<size_t>(p.seq.state(piece.sequence)) * p.heads + h) * p.state_size(), p.transposed);
            }, [](uint32_t) {});
        auto fill = [&](uint32_t b, uint32_t e, float v) {
            static_assert(TENSOR_THREADS % COLUMNS == 0, "a row of threads for a token");
            for (uint32_t t = b + threadIdx.x / COLUMNS; t < e; t += TENSOR_THREADS / COLUMNS) {
                if (threadIdx.x % COLUMNS >= columns) continue;
                const size_t at = ((static_cast<size_t>(p.seq.row(t)) * p.heads + h) * p.parts + part) * p.v_size + c0 + threadIdx.x % COLUMNS;
                if (p.wide_out) static_cast<float *>(p.out)[at] = v;
                else static_cast<bf16 *>(p.out)[at] = __float2bfloat16_rn(v);
            }
        };
        if (s.failed) fill(from, to, __int_as_float(0x7fffffff));
        // rows of no sequence: the first few and the last few
        fill(from, min(first, to), 0.0f);
        fill(max(last, from), to, 0.0f);
        // a sequence of no tokens leaves the state that it comes with
        if (p.last != nullptr)
            for (uint32_t q = p.seq.beginning(from); q < p.seq.seq.count; ++q) {
                const uint32_t b = p.seq.at(q), e = p.seq.at(q + 1);
                if (b >= to && g + 1 != p.segments) break;
                if (e > b) continue;
                const size_t at = (static_cast<size_t>(p.seq.state(q)) * p.heads + h) * p.state_size();
                for (uint32_t i = threadIdx.x; i < k_size * columns; i += TENSOR_THREADS) {
                    const size_t x = at + p.state_at(k0 + i / columns, c0 + i % columns);
                    p.last[x] = p.initial != nullptr ? p.initial[x] : 0.0f;
                }
            }
    }
}

using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                            const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encoder() {
    static const Encode found = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult result;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &result) == cudaSuccess && result == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<Encode>(f) : nullptr;
    }();
    return found;
}

// An operand as (elements of a head, heads, tokens), in boxes of 64 elements of 64 tokens of one head.
bool map_of(CUtensorMap *map, const HeadRows &r, const DecayWalk &p, uint32_t size) {
    const uint32_t heads = p.heads / r.group;
    const cuuint64_t sizes[3] = {size, heads, p.tokens};
    // (what there is only one of has no distance)
    const cuuint64_t strides[2] = {heads > 1 ? static_cast<cuuint64_t>(r.head) * 2 : 256, p.tokens > 1 ? static_cast<cuuint64_t>(r.row) * 2 : 256};
    const cuuint32_t box[3] = {64, 1, CHUNK}, steps[3] = {1, 1, 1};
    const Encode encode = encoder();
    return encode != nullptr &&
           encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(r.p), sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

std::atomic<long long> patience{MOST_CLOCKS};        // in clocks; what tests change

template<int KP, bool STATES>
bool launch(cudaStream_t stream, DecayWalk p, uint32_t segments, bool behind_join) {
    constexpr unsigned bytes = sizeof(TensorShared<KP, STATES>);
    static_assert(bytes <= 227 * 1024, "shared memory of a block");
    if (!allow_shared<decay_tensor_kernel<KP, STATES>>(bytes)) {
        set_status(BPL_ERR_CUDA, "decay_attention: shared memory");
        return false;
    }
    p.patience = patience.load(std::memory_order_relaxed);
    Maps maps;
    if (p.tokens == 0) {
        std::memset(&maps, 0, sizeof(maps));                // (nothing is copied)
    } else if (!map_of(&maps.q, p.q, p, p.k_size) || !map_of(&maps.k, p.k, p, p.k_size) || !map_of(&maps.v, p.v, p, p.v_size)) {
        set_status(BPL_ERR_CUDA, "decay_attention: tensor maps");
        return false;
    }
    const dim3 grid(p.heads * ((p.v_size + COLUMNS - 1) / COLUMNS) * p.parts, segments);
    if (behind_join) launch_dependent(decay_tensor_kernel<KP, STATES>, grid, dim3(TENSOR_THREADS), bytes, stream, p, maps);
    else decay_tensor_kernel<KP, STATES><<<grid, TENSOR_THREADS, bytes, stream>>>(p, maps);
    return true;
}

}  // namespace

uint64_t tensor_walk_units(const bpl_decay_attention_descriptor &d, uint32_t k_size, uint32_t v_size) {
    return static_cast<uint64_t>(d.heads) * ((v_size + COLUMNS - 1) / COLUMNS) * tensor_walk_parts(k_size);
}

bool tensor_walk_fits(const DecayWalk &p) {
    bool ok = p.k_size % 8 == 0 && p.v_size % 8 == 0 && aligned16(p.out);
    for (const HeadRows *r : {&p.q, &p.k, &p.v}) {
        ok &= aligned16(r->p);
        if (p.tokens > 1) ok &= r->row > 0 && r->row % 8 == 0 && r->row < (1ll << 38);
        if (p.heads > r->group) ok &= r->head > 0 && r->head % 8 == 0 && r->head < (1ll << 38);
    }
    return ok;
}

namespace {
template<bool STATES>
bool launch_sized(cudaStream_t stream, const DecayWalk &p, uint32_t segments, bool behind_join) {
    return p.k_size <= 64 ? launch<64, STATES>(stream, p, segments, behind_join) : launch<128, STATES>(stream, p, segments, behind_join);
}
}  // namespace

bool tensor_walk_states(cudaStream_t stream, const DecayWalk &p) { return launch_sized<true>(stream, p, p.segments - 1, false); }
bool tensor_walk(cudaStream_t stream, const DecayWalk &p, bool behind_join) { return launch_sized<false>(stream, p, p.segments, behind_join); }

}  // namespace bpl

extern "C" {

uint32_t bpl_tensor_walk_failures(void) {
    uint32_t n = 0;
    return cudaMemcpyFromSymbol(&n, bpl::failures, sizeof(n)) == cudaSuccess ? n : 0xffffffffu;
}

void bpl_tensor_walk_patience_for_tests(int64_t clocks) { bpl::patience = clocks < 0 || clocks > bpl::MOST_CLOCKS ? bpl::MOST_CLOCKS : clocks; }

}  // extern "C"
