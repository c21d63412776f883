// Linear attention with a decay for each head over packed sequences: what its kernels share.
//
//     S[t] = a S[t - 1] + k[t] v[t]^T;   o[t] = scale S[t]^T q[t],   a = exp(log_decay) of the head
//
// One walk computes this and, with its operands exchanged, every gradient (X: the gradient of a state by all later outputs):
//
//     dq = walk(do, v, k)                      on the transposed state: S[t] do[t]
//     dv = walk backwards in time (k, q, do):  X^T k
//     dk = walk backwards in time (v, do, q):  X v, on the transposed state
//
// A walk goes through virtual tokens: token t itself, or the t-th from the end.  Tokens are cut into segments that are walked at
// once.  A walk over all segments but the last first makes the state that each hands on, from nothing but its own tokens; these are
// joined in order, and the walk proper starts every segment from the state of the one in front.
#ifndef BPL_CSRC_DECAY_ATTENTION_CUH_
#define BPL_CSRC_DECAY_ATTENTION_CUH_

#include "sequence.cuh"

namespace bpl {

constexpr uint32_t MAX_HEAD = 256;          // elements of a head

// Head h of token t: at p + t row + (h / group) head.
struct HeadRows {
    const void *p;
    long long row, head;
    uint32_t group;
    template<typename T>
    __device__ __forceinline__ const T *of(uint32_t h) const {
        return static_cast<const T *>(p) + static_cast<long long>(h / group) * head;
    }
};

// Packed sequences in virtual order.
struct VirtualSequences {
    Sequences seq;
    bool backwards;

    __device__ __forceinline__ uint32_t at(uint32_t i) const { return backwards ? seq.tokens - seq.at(seq.count - i) : seq.at(i); }
    __device__ __forceinline__ uint32_t row(uint32_t t) const { return backwards ? seq.tokens - 1 - t : t; }
    __device__ __forceinline__ uint32_t state(uint32_t s) const { return backwards ? seq.count - 1 - s : s; }
    __device__ __forceinline__ uint32_t first() const { return seq.count ? at(0) : 0u; }
    __device__ __forceinline__ uint32_t last() const { return seq.count ? at(seq.count) : 0u; }
    // the first sequence that begins at or behind t, or count
    __device__ __forceinline__ uint32_t beginning(uint32_t t) const {
        uint32_t lo = 0, hi = seq.count;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (at(mid) < t) lo = mid + 1; else hi = mid;
        }
        return lo;
    }
    // whether a sequence goes on from token t - 1 to token t; where it begins
    __device__ __forceinline__ bool crosses(uint32_t t, uint32_t &begin, uint32_t &which) const {
        const uint32_t s = beginning(t);
        if (s == 0) return false;
        which = s - 1;
        begin = at(which);
        return begin < t && at(s) > t;
    }
};

struct DecayWalk {
    HeadRows q, k, v;
    void *out;                    // [tokens][heads][parts][v_size], dense
    const float *log_decay;
    const float *initial;         // [sequences][heads][k_size][v_size], or of v_size and k_size where `transposed`
    float *last;                  // like `initial`
    float *carried;               // [segments][heads][k_size][v_size]: what segment g hands on
    VirtualSequences seq;
    uint32_t tokens, heads, k_size, v_size, segment, segments;
    uint32_t parts;               // walks that share the rows of a state out (128 to each), their results to be added; 1 or 2
    float out_scale, state_scale; // of what is read out, and of what goes into the state
    float own_scale;              // of a token's products with the tokens of its chunk (out_scale state_scale)
    bool transposed, wide_out;    // wide_out: results are float whatever T is
    bool carried_turned;          // `carried` is of [v_size][k_size]: another walk's, on the transposed state
    long long patience;           // on tensor cores: clocks after which a wait for a barrier is given up; 0: nothing is copied, for tests

    __device__ __forceinline__ size_t state_at(uint32_t i, uint32_t j) const {
        return transposed ? static_cast<size_t>(j) * k_size + i : static_cast<size_t>(i) * v_size + j;
    }
    __device__ __forceinline__ size_t carried_at(uint32_t i, uint32_t j) const {
        return carried_turned ? static_cast<size_t>(j) * k_size + i : static_cast<size_t>(i) * v_size + j;
    }
    __device__ __forceinline__ size_t state_size() const { return static_cast<size_t>(k_size) * v_size; }
};

// Part of a sequence that lies in one segment.
struct Piece {
    uint32_t from, to;            // virtual tokens
    uint32_t sequence;
    bool begins, ends;            // whether the sequence does, in it
};

// Calls f(piece) for the pieces of segment g in order, and empty(sequence) for the sequences without tokens that lie there.
template<typename F, typename G>
__device__ __forceinline__ void for_pieces(const DecayWalk &p, uint32_t g, F f, G empty) {
    const uint32_t from = g * p.segment, to = g + 1 == p.segments ? p.tokens : min(p.tokens, from + p.segment);
    uint32_t begin, which;
    if (from > 0 && p.seq.crosses(from, begin, which)) {
        const uint32_t end = p.seq.at(which + 1);
        f(Piece{from, min(end, to), which, false, end <= to});
    }
    for (uint32_t s = p.seq.beginning(from); s < p.seq.seq.count; ++s) {
        const uint32_t b = p.seq.at(s), e = p.seq.at(s + 1);
        if (b >= to && g + 1 != p.segments) break;
        if (e <= b) empty(s);
        else if (b < to) f(Piece{b, min(e, to), s, true, e <= to});
    }
}

// The piece that segment g hands on to the next one, if any does.
__device__ __forceinline__ bool handed_on(const DecayWalk &p, uint32_t g, Piece &piece) {
    const uint32_t from = g * p.segment, to = from + p.segment;
    if (g + 1 >= p.segments || to >= p.tokens) return false;
    uint32_t begin, which;
    if (!p.seq.crosses(to, begin, which)) return false;
    piece = Piece{max(begin, from), to, which, begin >= from, false};
    return true;
}

// decay^n of the head, in 64 bits until the end (a decay of zero to the power of zero is one)
__device__ __forceinline__ float decay_power(float log_decay, uint32_t n) {
    return n == 0 ? 1.0f : static_cast<float>(exp(static_cast<double>(log_decay) * n));
}

// How tokens are cut into segments: `units` blocks walk each of them.
struct SegmentPlan {
    uint32_t segment, segments;
    bool crossing;                // whether a sequence may lie in several
};
SegmentPlan plan_segments(const bpl_decay_attention_descriptor &d, bool packed, uint64_t units, uint64_t wanted, uint32_t least);

// The walk on tensor cores (decay_attention_tensor.cu): whether it takes these operands (bfloat16), blocks of all heads for a segment, the
// states that segments hand on, and the walk proper.
bool tensor_walk_fits(const DecayWalk &p);
uint64_t tensor_walk_units(const bpl_decay_attention_descriptor &d, uint32_t k_size, uint32_t v_size);
inline uint32_t tensor_walk_parts(uint32_t k_size) { return k_size > 128 ? 2 : 1; }
bool tensor_walk_states(cudaStream_t stream, const DecayWalk &p);
bool tensor_walk(cudaStream_t stream, const DecayWalk &p, bool behind_join);      // behind_join: starts while states are joined

}  // namespace bpl

#endif  // BPL_CSRC_DECAY_ATTENTION_CUH_
