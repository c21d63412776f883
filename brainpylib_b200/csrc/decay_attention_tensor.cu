// The walk of decay_attention.cuh on tensor cores, for bfloat16 with up to 128 elements to a head of q and k.
//
// Tokens go by in chunks of 64.  With the columns of the chunk's tokens, S the state in front of it (turned: a row for every column of
// v), a the decay and n the tokens there are:
//
//     P = (Q K^T) . a^(i - j), j <= i          M tokens i, N tokens j          rounded to 16 bits
//     O = V^T P^T + (S Q^T) . a^(i + 1)        M columns of v, N tokens i      S as two numbers of 16 bits
//     S = a^n S + (V . a^(n - 1 - j))^T K      M columns of v, N elements of k the factor as three numbers of 16 bits
//
// S stays in tensor memory in 32 bits.  Three terms keep all 24 bits of what goes into it, so that it is as good as one of 32-bit
// arithmetic; what a chunk reads out is rounded to 16 bits in the end, where P's rounding and the two terms of S (16 bits) do not show.
//
// A block holds 128 columns of one head of one segment: four warps turn P and write O, eight carry S from chunk to chunk and split V,
// two copy (a stage each), one thread asks for the products.  The chain from chunk to chunk is: products into S, S read,
// decayed, written back; everything else goes beside it.
//
// A number of v that is not finite would reach tokens in front of it (0 times it, in V^T P^T).  It is taken out of the chunk, and the
// column is no number from its token on.
#include <algorithm>

#include "decay_attention.cuh"
#include "tensor_core.cuh"

namespace bpl {
namespace {

using bf16 = __nv_bfloat16;

constexpr uint32_t CHUNK = 64, COLUMNS = 128;        // tokens, columns of v
constexpr int READ_WARPS = 4, STATE_WARPS = 8, COPY_WARPS = 2;
constexpr int TENSOR_THREADS = 32 * (READ_WARPS + STATE_WARPS + COPY_WARPS + 1);
constexpr int STAGES = 2, TERMS = 3, SLOTS = 8, COPIERS = 32 * COPY_WARPS / STAGES;      // (copiers: of a stage)
constexpr uint32_t TILE = CHUNK * 128;               // bytes of 64 rows of 64 elements

// columns of tensor memory
constexpr uint32_t T_STATE = 0, T_HIGH = 128, T_LOW = 192, T_SCORES = 256, T_OWN = 320, T_EARLIER = 384, T_COLUMNS = 512;

template<int KP>
struct TensorShared {
    static constexpr uint32_t HALVES = KP / 64, STAGE = (2 * HALVES + 2) * TILE;
    // a stage: for each run of 64 elements of a head the tile of q, then that of k; then the two tiles of v
    unsigned char stage[STAGES][STAGE];
    unsigned char scores[2][TILE];
    unsigned char terms[2][TERMS][2 * TILE];
    float power[CHUNK + 1], own[CHUNK];              // powers of the decay; times the scale of P
    uint32_t poison[SLOTS][COLUMNS];                 // the first token of a chunk whose v is not finite, by column
    uint64_t full[STAGES], empty[STAGES], scored, turned, decayed, split[2], ready, stated, earlier, read_out, written, drained;
    uint32_t tensor, failed;
};

struct Chunk {
    uint32_t from, tokens;        // virtual
    bool first, last;             // of its piece
};

// The chunks of a segment, piece by piece; every thread goes through them by itself.
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
        c.first = at == piece.from;
        c.from = at;
        c.tokens = min(CHUNK, piece.to - at);
        at += c.tokens;
        c.last = at >= piece.to;
        inside = !c.last;
        return true;
    }
};

__device__ uint32_t failures;     // blocks whose waits ran out

// Waits end: after a second at the latest, and then in all warps.
__device__ __forceinline__ uint64_t nanoseconds() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
__device__ __noinline__ bool wait_long(uint64_t *b, uint32_t parity, volatile uint32_t *failed) {
    const uint64_t began = nanoseconds();
    while (!barrier_passed(b, parity)) {
        if (*failed || nanoseconds() - began > 1000000000ull) {
            *failed = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool wait(uint64_t *b, uint32_t parity, volatile uint32_t *failed) {
    if (barrier_passed(b, parity) || barrier_passed(b, parity)) return true;
    return wait_long(b, parity, failed);
}
// by a whole warp, which goes on together
__device__ __forceinline__ bool wait_warp(uint64_t *b, uint32_t parity, volatile uint32_t *failed) {
    return __all_sync(FULL_MASK, wait(b, parity, failed));
}

__device__ __forceinline__ uint32_t pack(float a, float b) {       // a in the low half
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return reinterpret_cast<const uint32_t &>(v);
}
__device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

template<int KP, bool STATES>
__global__ __launch_bounds__(TENSOR_THREADS, 1) void decay_tensor_kernel(const DecayWalk p) {
    extern __shared__ __align__(1024) unsigned char shared[];
    using Shared = TensorShared<KP>;
    Shared &s = *reinterpret_cast<Shared *>(shared);
    constexpr uint32_t HALVES = Shared::HALVES, V_AT = 2 * HALVES * TILE;
    const uint32_t slabs = (p.v_size + COLUMNS - 1) / COLUMNS, h = blockIdx.x / slabs, c0 = blockIdx.x % slabs * COLUMNS, g = blockIdx.y;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const bool backwards = p.seq.backwards;

    if (threadIdx.x <= CHUNK) s.power[threadIdx.x] = decay_power(p.log_decay[h], threadIdx.x);
    for (uint32_t i = threadIdx.x; i < SLOTS * COLUMNS; i += TENSOR_THREADS) s.poison[i / COLUMNS][i % COLUMNS] = CHUNK;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            barrier_init(&s.full[i], COPIERS);
            barrier_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) barrier_init(&s.split[i], 32 * STATE_WARPS);
        barrier_init(&s.scored, 1);
        barrier_init(&s.turned, 64);
        barrier_init(&s.decayed, 32 * STATE_WARPS);
        barrier_init(&s.ready, 32 * STATE_WARPS);
        barrier_init(&s.stated, 1);
        barrier_init(&s.earlier, 1);
        barrier_init(&s.read_out, 1);
        barrier_init(&s.written, 32 * READ_WARPS);
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
    if (threadIdx.x < CHUNK) s.own[threadIdx.x] = s.power[threadIdx.x] * p.own_scale;
    __syncthreads();
    volatile uint32_t *failed = &s.failed;

    // A sequence's first state backwards is the gradient of its last one, and has not decayed when the first token reads it.
    auto shift = [&](const Chunks &it, const Chunk &c) { return backwards && c.first && it.piece.begins ? 1u : 0u; };

    if (warp < READ_WARPS) {
        if constexpr (!STATES) {
            Chunks it(p, g, true);
            Chunk now, next;
            bool more = it.next(now);
            uint32_t shift_now = more ? shift(it, now) : 0;
            // P of chunk n: row i by thread i
            auto turn = [&](uint32_t n) {
                if (warp >= 2) return true;
                if (!wait_warp(&s.scored, n & 1, failed)) return false;
                tensor_fence_after();
                const uint32_t i = threadIdx.x;
                unsigned char *to = s.scores[n & 1];
#pragma unroll
                for (uint32_t part = 0; part < 4; ++part) {
                    uint32_t x[16], y[8];
                    tensor_load_16(tensor + lanes + T_SCORES + 16 * part, x);
                    tensor_wait_loads();
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint32_t j = 16 * part + 2 * k;
                        const float a = j <= i ? __uint_as_float(x[2 * k]) * s.own[i - min(j, i)] : 0.0f;
                        const float b = j + 1 <= i ? __uint_as_float(x[2 * k + 1]) * s.own[i - min(j + 1, i)] : 0.0f;
                        y[k] = pack(a, b);
                    }
                    *reinterpret_cast<uint4 *>(to + swizzled(i, 2 * part)) = make_uint4(y[0], y[1], y[2], y[3]);
                    *reinterpret_cast<uint4 *>(to + swizzled(i, 2 * part + 1)) = make_uint4(y[4], y[5], y[6], y[7]);
                }
                fence_shared_for_tensor();
                tensor_fence_before();
                barrier_arrive(&s.turned);
                return true;
            };
            const uint32_t column = threadIdx.x;
            const bool mine = c0 + column < p.v_size;
            bool good = !more || turn(0);
            for (uint32_t n = 0; more && good; ++n) {
                const bool another = it.next(next);
                const uint32_t shift_next = another ? shift(it, next) : 0;
                if (another && !(good = turn(n + 1))) break;
                if (!(good = wait_warp(&s.read_out, n & 1, failed))) break;
                tensor_fence_after();
                const uint32_t poison = s.poison[n % SLOTS][column];
                const long long step = static_cast<long long>(p.heads) * p.v_size * (backwards ? -1 : 1);
                long long at = (static_cast<long long>(p.seq.row(now.from)) * p.heads + h) * p.v_size + c0 + column;
#pragma unroll
                for (uint32_t part = 0; part < 4; ++part) {
                    uint32_t own[16], earlier[16];
                    tensor_load_16(tensor + lanes + T_OWN + 16 * part, own);
                    tensor_load_16(tensor + lanes + T_EARLIER + 16 * part, earlier);
                    tensor_wait_loads();
                    if (part == 3) {
                        tensor_fence_before();
                        barrier_arrive(&s.written);
                    }
#pragma unroll
                    for (uint32_t k = 0; k < 16; ++k) {
                        const uint32_t i = 16 * part + k;
                        if (i < now.tokens && mine) {
                            float o = fmaf(__uint_as_float(earlier[k]), s.power[i + 1 - shift_now] * p.out_scale, __uint_as_float(own[k]));
                            if (i >= poison) o = __int_as_float(0x7fffffff);
                            if (p.wide_out) static_cast<float *>(p.out)[at] = o;
                            else static_cast<bf16 *>(p.out)[at] = __float2bfloat16_rn(o);
                        }
                        at += step;
                    }
                }
                now = next;
                shift_now = shift_next;
                more = another;
            }
        }
    } else if (warp < READ_WARPS + STATE_WARPS) {
        constexpr uint32_t OWN = KP / 2;             // columns of the state (elements of k) of a thread
        const uint32_t tid = threadIdx.x - 32 * READ_WARPS, half = tid / 128, column = tid % 128, i0 = half * OWN;
        const bool mine = c0 + column < p.v_size;
        Chunks it(p, g, !STATES);
        Chunk now, next;
        bool more = it.next(now);
        // V of chunk n times the decays, as three numbers of 16 bits: thread (j, quarter of the columns)
        auto split = [&](uint32_t n, const Chunk &c) {
            if (!wait_warp(&s.full[n % STAGES], n / STAGES & 1, failed)) return false;
            const uint32_t j = tid / 4, q = tid % 4;
            unsigned char *from = s.stage[n % STAGES] + V_AT + q / 2 * TILE, *to = s.terms[n & 1][0] + q / 2 * TILE;
            const float w = j < c.tokens ? s.power[c.tokens - 1 - j] * p.state_scale : 0.0f;
            if (tid < COLUMNS) s.poison[(n + SLOTS / 2) % SLOTS][tid] = CHUNK;
            uint32_t odd = 0;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t at = swizzled(j, q % 2 * 4 + k);
                const uint4 raw = *reinterpret_cast<const uint4 *>(from + at);
                const uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
                uint32_t t[TERMS][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    odd |= ((x[e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;       // exponents of ones
                    float a = low(x[e]) * w, b = high(x[e]) * w;
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) {
                        t[m][e] = pack(a, b);
                        a -= low(t[m][e]);
                        b -= high(t[m][e]);
                    }
                }
#pragma unroll
                for (int m = 0; m < TERMS; ++m)
                    *reinterpret_cast<uint4 *>(to + m * 2 * TILE + at) = make_uint4(t[m][0], t[m][1], t[m][2], t[m][3]);
            }
            if (!STATES && odd != 0)
                for (uint32_t e = 0; e < 32; ++e) {
                    uint16_t *v = reinterpret_cast<uint16_t *>(from + swizzled(j, q % 2 * 4 + e / 8)) + e % 8;
                    if ((*v & 0x7f80) == 0x7f80) {
                        *v = 0;
                        atomicMin(&s.poison[n % SLOTS][q * 32 + e], j);
                    }
                }
            fence_shared_for_tensor();
            barrier_arrive(&s.split[n & 1]);
            return true;
        };
        auto for_elements = [&](auto f) {            // of the state, as it lies in global memory
#pragma unroll 8
            for (uint32_t k = 0; k < OWN; ++k)
                if (mine && i0 + k < p.k_size) f(k, i0 + k, c0 + column);
        };
        bool good = !more || split(0, now);
        for (uint32_t n = 0; more && good; ++n) {
            const Piece piece = it.piece;
            const uint32_t shift_now = shift(it, now);
            if (n > 0 && !(good = wait_warp(&s.stated, (n - 1) & 1, failed))) break;
            tensor_fence_after();
            uint32_t x[OWN];
            if (now.first) {
#pragma unroll
                for (uint32_t k = 0; k < OWN; ++k) x[k] = 0;
                if (piece.begins ? p.initial != nullptr : !STATES) {
                    const float *from = piece.begins ? p.initial + (static_cast<size_t>(p.seq.state(piece.sequence)) * p.heads + h) * p.state_size()
                                                     : p.carried + (static_cast<size_t>(g - 1) * p.heads + h) * p.state_size();
                    const size_t down = piece.begins && p.transposed ? 1 : p.v_size, across = piece.begins && p.transposed ? p.k_size : 1;
#pragma unroll
                    for (uint32_t k = 0; k < OWN; ++k)
                        if (mine && i0 + k < p.k_size) x[k] = __float_as_uint(__ldcg(from + (i0 + k) * down + (c0 + column) * across));
                }
            } else {
#pragma unroll
                for (uint32_t k = 0; k < OWN; k += 16) tensor_load_16(tensor + lanes + T_STATE + i0 + k, x + k);
                tensor_wait_loads();
            }
            const float a = s.power[now.tokens - shift_now];
#pragma unroll
            for (uint32_t k = 0; k < OWN; k += 16) {
                uint32_t y[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(x[k + e]) * a);
                tensor_store_16(tensor + lanes + T_STATE + i0 + k, y);
            }
            tensor_wait_stores();
            tensor_fence_before();
            barrier_arrive(&s.decayed);
            if constexpr (!STATES) {
                if (n > 0 && !(good = wait_warp(&s.earlier, (n - 1) & 1, failed))) break;
                tensor_fence_after();
#pragma unroll
                for (uint32_t k = 0; k < OWN; k += 32) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float u = __uint_as_float(x[k + 2 * e]), v = __uint_as_float(x[k + 2 * e + 1]);
                        hi[e] = pack(u, v);
                        lo[e] = pack(u - low(hi[e]), v - high(hi[e]));
                    }
                    tensor_store_16(tensor + lanes + T_HIGH + (i0 + k) / 2, hi);
                    tensor_store_16(tensor + lanes + T_LOW + (i0 + k) / 2, lo);
                }
                tensor_wait_stores();
                tensor_fence_before();
                barrier_arrive(&s.ready);
            }
            const bool another = it.next(next);
            if (another && !(good = split(n + 1, next))) break;
            if (now.last && (STATES || (piece.ends && p.last != nullptr))) {
                if (!(good = wait_warp(&s.stated, n & 1, failed))) break;
                tensor_fence_after();
                float *to = STATES ? p.carried + (static_cast<size_t>(g) * p.heads + h) * p.state_size()
                                   : p.last + (static_cast<size_t>(p.seq.state(piece.sequence)) * p.heads + h) * p.state_size();
                const size_t down = !STATES && p.transposed ? 1 : p.v_size, across = !STATES && p.transposed ? p.k_size : 1;
                const float end = !STATES && backwards ? s.power[1] : 1.0f;
#pragma unroll
                for (uint32_t k = 0; k < OWN; k += 16) {
                    tensor_load_16(tensor + lanes + T_STATE + i0 + k, x + k);
                    tensor_wait_loads();
#pragma unroll
                    for (uint32_t e = 0; e < 16; ++e)
                        if (mine && i0 + k + e < p.k_size) to[(i0 + k + e) * down + (c0 + column) * across] = __uint_as_float(x[k + e]) * end;
                }
                tensor_fence_before();
            }
            now = next;
            more = another;
        }
    } else if (warp < READ_WARPS + STATE_WARPS + COPY_WARPS) {
        // two groups of threads, each with a stage of its own: chunks 0, 2, 4, ... and 1, 3, 5, ...
        const uint32_t tid = threadIdx.x - 32 * (READ_WARPS + STATE_WARPS), group = tid / COPIERS, me = tid % COPIERS;
        unsigned char *stage = s.stage[group];
        const uint32_t stage_at = shared_address(stage);
        Chunks it(p, g, !STATES);
        Chunk c;
        auto rows = [&](const HeadRows &from, uint32_t at, uint32_t distance, uint32_t size, uint32_t offset, auto pieces) {
            constexpr uint32_t PIECES = decltype(pieces)::value, TOGETHER = COPIERS / PIECES;        // 16-byte pieces of a row; rows at once
            const uint32_t piece = me % PIECES, r0 = me / PIECES;
            const bool column = offset + piece * 8 < size;
            const bf16 *base = from.of<bf16>(h);
            const bf16 *row = base + (column ? offset + piece * 8 : 0);
            const uint32_t to = stage_at + at + piece / 8 * distance;
#pragma unroll 8
            for (uint32_t r = r0; r < CHUNK; r += TOGETHER) {
                const bool there = column && r < c.tokens;
                copy_16_or_zeros(to + swizzled(r, piece % 8), there ? row + static_cast<long long>(p.seq.row(c.from + r)) * from.row : base, there);
            }
        };
        for (uint32_t n = 0; it.next(c); ++n) {
            if (n % STAGES != group) continue;
            if (n >= STAGES && !wait_warp(&s.empty[group], (n / STAGES - 1) & 1, failed)) break;
            rows(p.k, TILE, 2 * TILE, p.k_size, 0, std::integral_constant<uint32_t, KP / 8>());
            rows(p.v, V_AT, TILE, p.v_size, c0, std::integral_constant<uint32_t, COLUMNS / 8>());
            if (!STATES) rows(p.q, 0, 2 * TILE, p.k_size, 0, std::integral_constant<uint32_t, KP / 8>());
            copies_wait_all();
            fence_shared_for_tensor();
            barrier_arrive(&s.full[group]);
        }
        copies_wait_all();
    } else if (lane == 0) {
        Chunks it(p, g, !STATES);
        Chunk c;
        auto score = [&](uint32_t n) {              // P: rows of q (and, unused, of k) by rows of k
            const uint32_t at = shared_address(s.stage[n % STAGES]);
#pragma unroll
            for (uint32_t k = 0; k < KP / 16; ++k) {
                const uint32_t from = at + k / 4 * 2 * TILE + k % 4 * 32;
                multiply(tensor + T_SCORES, operand(from, 1024), operand(from + TILE, 1024), product_of(CHUNK, false, false), k > 0);
            }
            products_arrive(&s.scored);
        };
        bool more = it.next(c), good = !more || wait(&s.full[0], 0, failed);
        if (!STATES && more && good) {
            tensor_fence_after();
            score(0);
        }
        for (uint32_t n = 0; more && good; ++n) {
            const uint32_t at = shared_address(s.stage[n % STAGES]);
            if (!(good = wait(&s.decayed, n & 1, failed) && wait(&s.split[n & 1], n / 2 & 1, failed))) break;
            tensor_fence_after();
#pragma unroll
            for (uint32_t m = 0; m < TERMS; ++m) {
                const uint32_t v = shared_address(s.terms[n & 1][m]);
#pragma unroll
                for (uint32_t k = 0; k < CHUNK / 16; ++k)
                    multiply(tensor + T_STATE, operand(v + k * 2048, 1024, TILE), operand(at + TILE + k * 2048, 1024, 2 * TILE),
                             product_of(KP, true, true), true);
            }
            products_arrive(&s.stated);
            if constexpr (STATES) {
                products_arrive(&s.empty[n % STAGES]);
            } else {
                if (!(good = wait(&s.ready, n & 1, failed) && (n == 0 || wait(&s.written, (n - 1) & 1, failed)))) break;
                tensor_fence_after();
#pragma unroll
                for (uint32_t m = 0; m < 2; ++m)
#pragma unroll
                    for (uint32_t k = 0; k < KP / 16; ++k)
                        multiply_from_tensor(tensor + T_EARLIER, tensor + (m == 0 ? T_HIGH : T_LOW) + 8 * k,
                                             operand(at + k / 4 * 2 * TILE + k % 4 * 32, 1024), product_of(CHUNK, false, false), m + k > 0);
                products_arrive(&s.earlier);
                if (!(good = wait(&s.turned, n & 1, failed))) break;
                tensor_fence_after();
                const uint32_t scores = shared_address(s.scores[n & 1]);
#pragma unroll
                for (uint32_t k = 0; k < CHUNK / 16; ++k)
                    multiply(tensor + T_OWN, operand(at + V_AT + k * 2048, 1024, TILE), operand(scores + k * 32, 1024),
                             product_of(CHUNK, true, false), k > 0);
                products_arrive(&s.read_out);
                products_arrive(&s.empty[n % STAGES]);
            }
            more = it.next(c);
            if (more && !STATES) {
                if (!(good = wait(&s.full[(n + 1) % STAGES], (n + 1) / STAGES & 1, failed))) break;
                tensor_fence_after();
                score(n + 1);
            }
        }
        if (!good) {                                // products on their way end before tensor memory is given back
            *failed = 1;
            products_arrive(&s.drained);
            const uint64_t began = nanoseconds();
            while (!barrier_passed(&s.drained, 0) && nanoseconds() - began < 1000000000ull) {}
        }
    }
    __syncwarp();
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (warp == 0) tensor_free(tensor, T_COLUMNS);
    if (s.failed && threadIdx.x == 0) atomicAdd(&failures, 1u);

    if constexpr (!STATES) {
        const uint32_t from = g * p.segment, to = g + 1 == p.segments ? p.tokens : min(p.tokens, from + p.segment);
        const uint32_t first = p.seq.first(), last = max(p.seq.last(), first), columns = min(COLUMNS, p.v_size - c0);
        auto fill = [&](uint32_t b, uint32_t e, float v) {
            for (uint32_t t = b + threadIdx.x / COLUMNS; t < e; t += TENSOR_THREADS / COLUMNS) {
                if (threadIdx.x % COLUMNS >= columns || threadIdx.x / COLUMNS >= TENSOR_THREADS / COLUMNS) continue;
                const size_t at = (static_cast<size_t>(p.seq.row(t)) * p.heads + h) * p.v_size + c0 + threadIdx.x % COLUMNS;
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
                for (uint32_t i = threadIdx.x; i < p.k_size * columns; i += TENSOR_THREADS) {
                    const size_t x = at + p.state_at(i / columns, c0 + i % columns);
                    p.last[x] = p.initial != nullptr ? p.initial[x] : 0.0f;
                }
            }
    }
}

template<int KP, bool STATES>
bool launch(cudaStream_t stream, const DecayWalk &p, uint32_t segments) {
    constexpr unsigned bytes = sizeof(TensorShared<KP>);
    static_assert(bytes <= 227 * 1024, "shared memory of a block");
    if (!allow_shared<decay_tensor_kernel<KP, STATES>>(bytes)) {
        set_status(BPL_ERR_CUDA, "decay_attention: shared memory");
        return false;
    }
    decay_tensor_kernel<KP, STATES><<<dim3(p.heads * ((p.v_size + COLUMNS - 1) / COLUMNS), segments), TENSOR_THREADS, bytes, stream>>>(p);
    return true;
}

}  // namespace

uint64_t tensor_walk_units(const bpl_decay_attention_descriptor &d, uint32_t v_size) {
    return static_cast<uint64_t>(d.heads) * ((v_size + COLUMNS - 1) / COLUMNS);
}

bool tensor_walk_fits(const DecayWalk &p) {
    bool ok = p.k_size <= 128 && p.k_size % 8 == 0 && p.v_size % 8 == 0;
    for (const HeadRows *r : {&p.q, &p.k, &p.v})
        ok &= aligned16(r->p) && r->row % 8 == 0 && (p.heads <= r->group || r->head % 8 == 0);
    return ok;
}

bool tensor_walk_states(cudaStream_t stream, const DecayWalk &p) {
    return p.k_size <= 64 ? launch<64, true>(stream, p, p.segments - 1) : launch<128, true>(stream, p, p.segments - 1);
}
bool tensor_walk(cudaStream_t stream, const DecayWalk &p) {
    return p.k_size <= 64 ? launch<64, false>(stream, p, p.segments) : launch<128, false>(stream, p, p.segments);
}

}  // namespace bpl

extern "C" uint32_t bpl_tensor_walk_failures(void) {
    uint32_t n = 0;
    return cudaMemcpyFromSymbol(&n, bpl::failures, sizeof(n)) == cudaSuccess ? n : 0xffffffffu;
}
