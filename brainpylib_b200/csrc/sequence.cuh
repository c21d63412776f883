// Device helpers shared by the operators over whole sequences (state_scan*.cu, short_conv.cu): element types, exponentials,
// packed pairs of floats, and which sequence a token belongs to.
#ifndef BPL_CSRC_SEQUENCE_CUH_
#define BPL_CSRC_SEQUENCE_CUH_

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "abi.h"
#include "common.cuh"

namespace bpl {

// ---- element types: read as float, rounded to nearest once when written ----------------------------------------------
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template<typename T> __device__ __forceinline__ T from_float(float v);
template<> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template<> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template<> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---- exponentials ----------------------------------------------------------------------------------------------------
constexpr float LOG2_E = 1.44269504088896340736f;
constexpr float LN_2 = 0.69314718055994530942f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// log(1 + u) / u on [0, 1], a polynomial fitted to the smallest relative error there (3e-8)
__device__ __forceinline__ float log1p_over(float u) {
    float p = 0.005232692696154118f;
    p = fmaf(p, u, -0.029505232349038124f);
    p = fmaf(p, u, 0.07822594046592712f);
    p = fmaf(p, u, -0.13663244247436523f);
    p = fmaf(p, u, 0.19106006622314453f);
    p = fmaf(p, u, -0.2484298199415207f);
    p = fmaf(p, u, 0.3331909775733948f);
    p = fmaf(p, u, -0.4999949336051941f);
    return fmaf(p, u, 0.9999999403953552f);
}
// log(1 + e^v): max(v, 0) + log(1 + e^-|v|), so that a far negative v keeps its relative precision
__device__ __forceinline__ float softplus(float v) {
    const float u = ex2(-fabsf(v) * LOG2_E);
    return fmaf(u, log1p_over(u), fmaxf(v, 0.0f));
}
// 1 / (1 + e^-v): a far negative v makes e^-v infinite and the result 0
__device__ __forceinline__ float sigmoid(float v) { return rcp(1.0f + ex2(v * -LOG2_E)); }
__device__ __forceinline__ float silu(float v) { return v * sigmoid(v); }

// ---- pairs of floats in one 64-bit register pair: one instruction does both ---------------------------------------------
using pair = unsigned long long;
__device__ __forceinline__ pair make_pair(float a, float b) {
    pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 split(pair p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ pair mul2(pair a, pair b) {
    pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ pair fma2(pair a, pair b, pair c) {
    pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ pair add2(pair a, pair b) {
    pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float sum2(pair p) {
    const float2 v = split(p);
    return v.x + v.y;
}
__device__ __forceinline__ pair ex2_pair(pair p) {
    const float2 v = split(p);
    return make_pair(ex2(v.x), ex2(v.y));
}

// The decay 2^(time * rate2).  ex2.approx gives slow decays (exponents of -0.001 to -0.25) 0.1 to 0.4 * 2^-24 too low on average,
// and a state that lasts a thousand tokens adds that up: 2^-24 * 300.  The exponent is raised by what brings the mean error to
// +0.1 * 2^-24 for exponents between -0.003 and 0 and to -0.1 to -0.3 up to -0.1; far ones swallow it.  An exponent of zero still
// gives 1.
constexpr float DECAY_SHIFT = 1.8e-8f;
__device__ __forceinline__ float decay(float time, float rate2) { return ex2(fmaf(time, rate2, DECAY_SHIFT)); }
__device__ __forceinline__ pair decay_pair(pair time, pair rate2) {
    return ex2_pair(fma2(time, rate2, make_pair(DECAY_SHIFT, DECAY_SHIFT)));
}

// log(1 + e^v) of two values, as softplus()
__device__ __forceinline__ pair softplus_pair(pair v) {
    const float2 a = split(v);
    const float2 t = split(mul2(make_pair(fabsf(a.x), fabsf(a.y)), make_pair(LOG2_E, LOG2_E)));
    const pair u = make_pair(ex2(-t.x), ex2(-t.y));
    pair q = make_pair(0.005232692696154118f, 0.005232692696154118f);
    auto next = [&](float c) { q = fma2(q, u, make_pair(c, c)); };
    next(-0.029505232349038124f);
    next(0.07822594046592712f);
    next(-0.13663244247436523f);
    next(0.19106006622314453f);
    next(-0.2484298199415207f);
    next(0.3331909775733948f);
    next(-0.4999949336051941f);
    next(0.9999999403953552f);
    return fma2(u, q, make_pair(fmaxf(a.x, 0.0f), fmaxf(a.y, 0.0f)));
}

// ---- sequences -------------------------------------------------------------------------------------------------------
// Sequence s holds the tokens indptr[s] .. indptr[s + 1] - 1 (without an indptr: every sequence holds `length` tokens).
// Whatever the array says, a begin or end is a number between 0 and the number of tokens.
struct Sequences {
    const int *indptr;
    uint32_t count, length, tokens;

    __device__ __forceinline__ uint32_t at(uint32_t i) const {
        if (indptr == nullptr) return i * length;
        const int v = __ldg(indptr + i);
        return v < 0 ? 0u : min(static_cast<uint32_t>(v), tokens);
    }
    __device__ __forceinline__ uint32_t begin(uint32_t s) const { return at(s); }
    __device__ __forceinline__ uint32_t end(uint32_t s) const { return at(s + 1); }
    // tokens outside [first(), last()) belong to no sequence
    __device__ __forceinline__ uint32_t first() const { return count ? at(0) : 0u; }
    __device__ __forceinline__ uint32_t last() const { return count ? at(count) : 0u; }
    // the last sequence that begins at or before t (count > 0): the one that holds t, if any does
    __device__ __forceinline__ uint32_t of(uint32_t t) const {
        if (indptr == nullptr) return length ? min(t / length, count - 1) : count - 1;
        uint32_t lo = 0, hi = count;          // at(lo) <= t (or lo = 0), at(hi) > t (or hi = count)
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (at(mid) <= t) lo = mid; else hi = mid;
        }
        return lo;
    }
};

// Whether a descriptor's sequences are its tokens: without an indptr, sequences of `length` tokens each; the kernels go by all three.
template<typename D>
inline bool sequences_fit(const D &d, const void *indptr) {
    return d.sequences < (1u << 31) && (indptr != nullptr || static_cast<uint64_t>(d.sequences) * d.length == d.tokens);
}

// ---- copies into shared memory that run by themselves --------------------------------------------------------------------
template<int BYTES>
__device__ __forceinline__ void copy_async(void *to, const void *from) {
    const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(at), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(at), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template<int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// Two neighbouring elements as a pair of floats, and back.
__device__ __forceinline__ pair load_pair(const float *p) { return *reinterpret_cast<const pair *>(p); }
__device__ __forceinline__ pair load_pair(const __half *p) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(p));
    return make_pair(v.x, v.y);
}
__device__ __forceinline__ pair load_pair(const __nv_bfloat16 *p) {
    const uint32_t v = *reinterpret_cast<const uint32_t *>(p);
    return make_pair(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ void store_pair(float *p, float2 v) { *reinterpret_cast<float2 *>(p) = v; }
__device__ __forceinline__ void store_pair(__half *p, float2 v) { *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(v.x, v.y); }
__device__ __forceinline__ void store_pair(__nv_bfloat16 *p, float2 v) {
    *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(v.x, v.y);
}

// Sums the `K` values of a lane over the `LANES` neighbouring lanes it shares a channel with; lane i of them is left with the
// sum of value i % K.  A lane hands over half of its values at each step, so K sums cost K - 1 shuffles, not K log2(LANES).
template<int K, int LANES>
__device__ __forceinline__ float sum_over_lanes(float (&v)[K], const int part) {
    static_assert(LANES % K == 0 && (K & (K - 1)) == 0, "powers of two");
#pragma unroll
    for (int m = K / 2; m > 0; m >>= 1) {
        const bool upper = (part & m) != 0;
#pragma unroll
        for (int i = 0; i < m; ++i) {
            const float give = upper ? v[i] : v[i + m], keep = upper ? v[i + m] : v[i];
            v[i] = keep + __shfl_xor_sync(FULL_MASK, give, m);
        }
    }
#pragma unroll
    for (int m = K; m < LANES; m <<= 1) v[0] += __shfl_xor_sync(FULL_MASK, v[0], m);
    return v[0];
}

// The same sum of a single value, in the same order, for all lanes.
template<int K, int LANES>
__device__ __forceinline__ float sum_over_lanes(float v) {
#pragma unroll
    for (int m = K / 2; m > 0; m >>= 1) v += __shfl_xor_sync(FULL_MASK, v, m);
#pragma unroll
    for (int m = K; m < LANES; m <<= 1) v += __shfl_xor_sync(FULL_MASK, v, m);
    return v;
}

}  // namespace bpl

#endif  // BPL_CSRC_SEQUENCE_CUH_
