// The norm over all gradients of a training step, and clipping (no counterpart in brainpylib):
//
//     N = (sum of g^2)^(1/2) or max |g| over all tensors;  g = g * min(1, m / (N + 1e-6))
//
// Bound by memory: the gradients are read for the norm and once more for the result, backwards, so that what was read last is
// still in L2 (600 million elements of 16 bits in 390 tensors: 722 us, 5.0 TB/s on two reads and one write).  The tensors' addresses
// travel as kernel arguments (no table in device memory: a call can be captured and needs no copy), a thousand to a launch.  A block's
// share of the chunks, and the order of all sums, depend on the sizes alone.
#include <algorithm>
#include <cstring>
#include <new>
#include <type_traits>
#include <vector>

#include "sequence.cuh"

namespace bpl {
namespace {

constexpr int CLIP_THREADS = 256;
constexpr uint32_t CHUNK_BYTES = 16384;
constexpr int BLOCKS_PER_SM = 8;

struct Entry {
    const void *in;
    void *out;
    unsigned long long count;       // elements
    uint32_t chunk, dtype;          // first chunk of the tensor
};
template<int MAX>
struct Table {
    Entry entry[MAX];
    uint32_t tensors, chunks;
};
constexpr int TABLE_SMALL = 24, TABLE_MEDIUM = 160, TABLE_LARGE = 1000;      // 32 bytes each; arguments end at 32,764 bytes
static_assert(sizeof(Table<TABLE_LARGE>) + 64 <= 32764, "kernel arguments");

__host__ __device__ constexpr uint32_t bytes_of(uint32_t dtype) { return dtype == BPL_DOUBLE ? 8u : dtype == BPL_FLOAT ? 4u : 2u; }

template<int MAX>
__device__ __forceinline__ uint32_t tensor_of(const Table<MAX> &t, uint32_t chunk) {
    uint32_t lo = 0, hi = t.tensors;
#pragma unroll 1
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (t.entry[mid].chunk <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

// The elements of a 32-bit word of a packet: one float, or two of 16 bits (doubles are taken as two words).
template<typename T>
__device__ __forceinline__ float2 of_word(uint32_t w) {
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w), 0.0f);
    else if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template<typename T>
__device__ __forceinline__ uint32_t to_word(float2 f) {
    if constexpr (sizeof(T) == 4) {
        return __float_as_uint(f.x);
    } else if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(f.x, f.y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
__device__ __forceinline__ double double_of(uint32_t low, uint32_t high) { return __hiloint2double(static_cast<int>(high), static_cast<int>(low)); }
__device__ __forceinline__ double wide(double v) { return v; }
template<typename T> __device__ __forceinline__ double wide(T v) { return static_cast<double>(to_float(v)); }

// Out of line, and from memory: it is called for packets of zeros, of far values and of no numbers, and would take the registers
// that loads need.
template<typename T>
__device__ __noinline__ double squares_in_64_bits(const T *at) {
    double sum = 0.0;
#pragma unroll 1
    for (uint32_t i = 0; i < 16 / sizeof(T); ++i) sum = fma(wide(at[i]), wide(at[i]), sum);
    return sum;
}

struct SumOfSquares {
    double sum = 0.0;
    __device__ __forceinline__ void one(double v) { sum = fma(v, v, sum); }
    // Squares of a packet (which lies at `at`): of doubles in 64 bits; of up to eight smaller elements in 32 bits, at most 8 roundings of
    // 2^-24 on a sum of one sign, where none of them can have left the range, else in 64.  (Widened one by one, every element would take
    // a conversion.)
    template<typename T>
    __device__ __forceinline__ void add(const uint4 p, const T *at) {
        if constexpr (sizeof(T) < 8) {
            float s = 0.0f;
            const auto word = [&s](uint32_t w) {
                const float2 f = of_word<T>(w);
                s = fmaf(f.x, f.x, s);
                if (sizeof(T) == 2) s = fmaf(f.y, f.y, s);
            };
            word(p.x);
            word(p.y);
            word(p.z);
            word(p.w);
            if (s > 1e-28f && s < 1e38f) sum += static_cast<double>(s);
            else sum += squares_in_64_bits(at);
        } else {
            one(double_of(p.x, p.y));
            one(double_of(p.z, p.w));
        }
    }
    __device__ __forceinline__ void join(double other) { sum += other; }
    __device__ __forceinline__ double value() const { return sum; }
};
struct LargestMagnitude {
    double most = 0.0;
    __device__ __forceinline__ void join(double v) { most = v > most || v != v ? v : most; }    // no number stays none
    __device__ __forceinline__ void one(double v) { join(fabs(v)); }
    template<typename T>
    __device__ __forceinline__ void add(const uint4 p, const T *) {
        if constexpr (sizeof(T) < 8) {
            float m = 0.0f;
            const auto larger = [&m](float f) { m = fabsf(f) > m || f != f ? fabsf(f) : m; };
            const auto word = [&larger](uint32_t w) {
                const float2 f = of_word<T>(w);
                larger(f.x);
                if (sizeof(T) == 2) larger(f.y);
            };
            word(p.x);
            word(p.y);
            word(p.z);
            word(p.w);
            join(static_cast<double>(m));
        } else {
            one(double_of(p.x, p.y));
            one(double_of(p.z, p.w));
        }
    }
    __device__ __forceinline__ double value() const { return most; }
};

template<typename Norm>
__device__ __forceinline__ double block_join(Norm n, double *shared) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n.join(__shfl_xor_sync(FULL_MASK, n.value(), o));
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = n.value();
    __syncthreads();
    Norm all;
    for (int w = 0; w < CLIP_THREADS / 32; ++w) all.join(shared[w]);
    __syncthreads();
    return all.value();
}

// A chunk of a tensor as bytes: up to the next 16-byte boundary element by element, then 16 bytes at a time, four of them on their
// way whatever the type is, then element by element again.
constexpr uint32_t AHEAD = CHUNK_BYTES / 16 / CLIP_THREADS;
static_assert(AHEAD == 4, "a chunk is four packets a thread");

struct Chunk {
    const char *in;
    char *out;
    uint32_t bytes, head, packets, tail, dtype;       // head and tail: bytes in front of, offset behind the packets
    template<int MAX>
    __device__ __forceinline__ Chunk(const Table<MAX> &t, uint32_t c) {
        const Entry &e = t.entry[tensor_of(t, c)];
        const unsigned long long from = static_cast<unsigned long long>(c - e.chunk) * CHUNK_BYTES;
        dtype = e.dtype;
        in = static_cast<const char *>(e.in) + from;
        out = static_cast<char *>(e.out) + from;
        bytes = static_cast<uint32_t>(min(static_cast<unsigned long long>(CHUNK_BYTES), e.count * bytes_of(dtype) - from));
        const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(in) & 15u);
        head = min(bytes, odd ? 16u - odd : 0u);
        packets = (bytes - head) / 16;
        tail = head + packets * 16;
    }
    __device__ __forceinline__ void no_packets() {
        head = bytes;
        packets = 0;
        tail = bytes;
    }
    __device__ __forceinline__ void load(uint4 (&v)[AHEAD]) const {
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k)
            if (threadIdx.x + k * CLIP_THREADS < packets) v[k] = reinterpret_cast<const uint4 *>(in + head)[threadIdx.x + k * CLIP_THREADS];
    }
    // f(element number) of the elements in front of and behind the packets
    template<typename F>
    __device__ __forceinline__ void rest(uint32_t size, F f) const {
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i * size < head; i += CLIP_THREADS) f(i);
#pragma unroll 1
        for (uint32_t i = tail / size + threadIdx.x; i * size < bytes; i += CLIP_THREADS) f(i);
    }
};

template<typename T, typename Norm>
__device__ __forceinline__ void norm_of(const Chunk &c, const uint4 (&v)[AHEAD], Norm &n) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; ++k)
        if (threadIdx.x + k * CLIP_THREADS < c.packets) n.add(v[k], reinterpret_cast<const T *>(c.in + c.head) + (threadIdx.x + k * CLIP_THREADS) * V);
    c.rest(sizeof(T), [&](uint32_t i) { n.one(wide(reinterpret_cast<const T *>(c.in)[i])); });
}

template<typename Norm, int MAX>
__global__ void __launch_bounds__(CLIP_THREADS, 4)
gradient_norm_kernel(const __grid_constant__ Table<MAX> t, double *parts) {
    __shared__ double shared[CLIP_THREADS / 32];
    pdl_launch_dependents();
    Norm n;
#pragma unroll 1
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Chunk chunk(t, c);
        uint4 v[AHEAD];
        chunk.load(v);
        if (chunk.dtype == BPL_FLOAT) norm_of<float>(chunk, v, n);
        else if (chunk.dtype == BPL_HALF) norm_of<__half>(chunk, v, n);
        else if (chunk.dtype == BPL_BFLOAT16) norm_of<__nv_bfloat16>(chunk, v, n);
        else norm_of<double>(chunk, v, n);
    }
    const double all = block_join(n, shared);
    if (threadIdx.x == 0) parts[blockIdx.x] = all;
}

// The norm from the parts, in every block for itself (a few hundred numbers) and in the same order.
template<typename Norm>
__device__ __forceinline__ double total_norm(const double *parts, uint32_t n_parts, bool root, double *shared) {
    Norm n;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < n_parts; i += CLIP_THREADS) n.join(__ldcg(parts + i));
    const double all = block_join(n, shared);
    return root ? sqrt(all) : all;
}

// A factor below the normal numbers of 32 bits would lose bits there, and the products (of gradients whose norm is beyond 10^38) with it:
// then they are taken in 64 bits, element by element, and rounded once.
constexpr double LEAST_FACTOR = 1.1754943508222875e-38;

template<typename T>
__device__ __forceinline__ T scaled(T v, double s) {
    if constexpr (sizeof(T) == 8) return v * s;
    else return from_float<T>(s > 0.0 && s < LEAST_FACTOR ? static_cast<float>(to_float(v) * s) : to_float(v) * static_cast<float>(s));
}

template<typename T>
__device__ __forceinline__ void scale(const Chunk &c, const uint4 (&v)[AHEAD], const double s) {
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; ++k)
        if (threadIdx.x + k * CLIP_THREADS < c.packets) {
            uint4 r;
            if constexpr (sizeof(T) == 8) {
                const double a = double_of(v[k].x, v[k].y) * s, b = double_of(v[k].z, v[k].w) * s;
                r = make_uint4(__double2loint(a), __double2hiint(a), __double2loint(b), __double2hiint(b));
            } else {
                const auto word = [s](uint32_t w) {
                    const float2 f = of_word<T>(w);
                    return to_word<T>(make_float2(f.x * static_cast<float>(s), f.y * static_cast<float>(s)));
                };
                r = make_uint4(word(v[k].x), word(v[k].y), word(v[k].z), word(v[k].w));
            }
            reinterpret_cast<uint4 *>(c.out + c.head)[threadIdx.x + k * CLIP_THREADS] = r;
        }
    c.rest(sizeof(T), [&](uint32_t i) { reinterpret_cast<T *>(c.out)[i] = scaled(reinterpret_cast<const T *>(c.in)[i], s); });
}

template<typename Norm, int MAX>
__global__ void __launch_bounds__(CLIP_THREADS, 4)
clip_kernel(const __grid_constant__ Table<MAX> t, const double *parts, const uint32_t n_parts, const bool root,
            const double max_norm, void *norm_out, const uint32_t norm_dtype, const bool in_place) {
    __shared__ double shared[CLIP_THREADS / 32];
    pdl_wait();                             // for the parts
    const double norm = total_norm<Norm>(parts, n_parts, root, shared);
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out != nullptr) {
        if (norm_dtype == BPL_DOUBLE) *static_cast<double *>(norm_out) = norm;
        else *static_cast<float *>(norm_out) = static_cast<float>(norm);
    }
    double s = max_norm / (norm + 1e-6);
    if (s >= 1.0) {
        if (in_place) return;               // nothing to clip
        s = 1.0;
    }
#pragma unroll 1
    for (uint32_t i = blockIdx.x; i < t.chunks; i += gridDim.x) {
        Chunk chunk(t, t.chunks - 1 - i);
        if (((reinterpret_cast<uintptr_t>(chunk.in) ^ reinterpret_cast<uintptr_t>(chunk.out)) & 15u) != 0 || (s > 0.0 && s < LEAST_FACTOR))
            chunk.no_packets();
        uint4 v[AHEAD];
        chunk.load(v);
        if (chunk.dtype == BPL_FLOAT) scale<float>(chunk, v, s);
        else if (chunk.dtype == BPL_HALF) scale<__half>(chunk, v, s);
        else if (chunk.dtype == BPL_BFLOAT16) scale<__nv_bfloat16>(chunk, v, s);
        else scale<double>(chunk, v, s);
    }
}

template<typename Norm>
__global__ void __launch_bounds__(CLIP_THREADS)
norm_only_kernel(const double *parts, const uint32_t n_parts, const bool root, void *norm_out, const uint32_t norm_dtype) {
    __shared__ double shared[CLIP_THREADS / 32];
    const double norm = total_norm<Norm>(parts, n_parts, root, shared);
    if (threadIdx.x == 0) {
        if (norm_dtype == BPL_DOUBLE) *static_cast<double *>(norm_out) = norm;
        else *static_cast<float *>(norm_out) = static_cast<float>(norm);
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------------
struct Call {
    const bpl_clip_descriptor *d;
    const bpl_clip_tensor *tensor;
    void **buffers;
    uint32_t count, tables, n_parts;
};

uint32_t chunks_of(const bpl_clip_tensor &t) {
    const uint64_t per = CHUNK_BYTES / bytes_of(t.dtype);
    return static_cast<uint32_t>((t.elements + per - 1) / per);
}
uint32_t blocks_of(uint32_t chunks) {
    const uint32_t most = static_cast<uint32_t>(BLOCKS_PER_SM * sm_count());
    return chunks < most ? (chunks ? chunks : 1) : most;
}

template<int MAX>
void fill(const Call &c, uint32_t first, uint32_t count, bool write, Table<MAX> &t) {
    t.tensors = 0;
    t.chunks = 0;
    for (uint32_t i = first; i < first + count; ++i) {
        if (c.tensor[i].elements == 0) continue;
        t.entry[t.tensors++] = Entry{c.buffers[i], write ? c.buffers[c.count + i] : nullptr, c.tensor[i].elements, t.chunks, c.tensor[i].dtype};
        t.chunks += chunks_of(c.tensor[i]);
    }
}

template<typename Norm, int MAX>
void launch(cudaStream_t stream, const Call &c, void *norm_out, double *parts) {
    const bool root = c.d->norm_type == 2, write = (c.d->flags & BPL_CLIP_WRITE) != 0, in_place = (c.d->flags & BPL_CLIP_IN_PLACE) != 0;
    Table<MAX> t;
    uint32_t at = 0;
    for (uint32_t i = 0; i < c.tables; ++i) {
        const uint32_t first = i * MAX, count = c.count - first < MAX ? c.count - first : MAX;
        fill(c, first, count, write, t);
        const uint32_t blocks = blocks_of(t.chunks);
        gradient_norm_kernel<Norm, MAX><<<blocks, CLIP_THREADS, 0, stream>>>(t, parts + at);
        at += blocks;
    }
    if (!write) {
        norm_only_kernel<Norm><<<1, CLIP_THREADS, 0, stream>>>(parts, at, root, norm_out, c.d->norm_dtype);
        return;
    }
    for (uint32_t i = c.tables; i-- > 0;) {
        const uint32_t first = i * MAX, count = c.count - first < MAX ? c.count - first : MAX;
        if (c.tables > 1) fill(c, first, count, write, t);
        // (a kernel that starts early waits for the one in front of it alone: behind several it is launched the ordinary way)
        if (c.tables == 1)
            launch_dependent(clip_kernel<Norm, MAX>, dim3(blocks_of(t.chunks)), dim3(CLIP_THREADS), 0, stream, t, static_cast<const double *>(parts),
                             at, root, c.d->max_norm, norm_out, c.d->norm_dtype, in_place);
        else
            clip_kernel<Norm, MAX><<<blocks_of(t.chunks), CLIP_THREADS, 0, stream>>>(
                t, parts, at, root, c.d->max_norm, i == 0 ? norm_out : nullptr, c.d->norm_dtype, in_place);
    }
}

uint32_t table_for(uint32_t count) { return count <= TABLE_SMALL ? TABLE_SMALL : count <= TABLE_MEDIUM ? TABLE_MEDIUM : TABLE_LARGE; }

const bpl_clip_descriptor *checked(const char *opaque, size_t opaque_len) {
    if (opaque == nullptr || opaque_len < sizeof(bpl_clip_descriptor)) return nullptr;
    const auto *d = reinterpret_cast<const bpl_clip_descriptor *>(opaque);
    return opaque_len == sizeof(bpl_clip_descriptor) + static_cast<size_t>(d->tensors) * sizeof(bpl_clip_tensor) ? d : nullptr;
}

// Whether something that is written overlaps anything else (a gradient and its own result in place are one).
bool overlap(const Call &c) {
    struct Range {
        uintptr_t from, to;
        bool written;
    };
    std::vector<Range> r;
    r.reserve(2 * c.count);
    for (uint32_t i = 0; i < c.count; ++i) {
        const size_t bytes = c.tensor[i].elements * bytes_of(c.tensor[i].dtype);
        if (bytes == 0) continue;
        const auto in = reinterpret_cast<uintptr_t>(c.buffers[i]), out = reinterpret_cast<uintptr_t>(c.buffers[c.count + i]);
        r.push_back({out, out + bytes, true});
        if (in != out) r.push_back({in, in + bytes, false});
    }
    const auto before = [](const Range &a, const Range &b) { return a.from < b.from; };
    if (!std::is_sorted(r.begin(), r.end(), before)) std::sort(r.begin(), r.end(), before);
    uintptr_t read_to = 0, written_to = 0;
    for (const Range &x : r) {
        if (x.from < written_to || (x.written && x.from < read_to)) return true;
        uintptr_t &end = x.written ? written_to : read_to;
        end = std::max(end, x.to);
    }
    return false;
}

}  // namespace

size_t clip_gradients_workspace_bytes(const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len);
    if (d == nullptr) return 0;
    const uint32_t tables = (d->tensors + TABLE_LARGE - 1) / TABLE_LARGE;
    return sizeof(double) * BLOCKS_PER_SM * static_cast<size_t>(sm_count()) * (tables ? tables : 1);
}

}  // namespace bpl

using namespace bpl;

extern "C" void clip_gradients(bpl_stream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
    const auto *d = checked(opaque, opaque_len);
    if (d == nullptr) {
        set_status(BPL_ERR_OPAQUE_SIZE, "Invalid opaque object size");
        return;
    }
    Call c{d, reinterpret_cast<const bpl_clip_tensor *>(opaque + sizeof(bpl_clip_descriptor)), buffers, d->tensors, 0, 0};
    const bool write = (d->flags & BPL_CLIP_WRITE) != 0;
    void *norm_out = buffers[2 * c.count], *parts = buffers[2 * c.count + 1];
    bool good = norm_out != nullptr && parts != nullptr && (d->norm_type == 2 || d->norm_type == 0) && d->max_norm >= 0.0 &&
                (d->norm_dtype == BPL_FLOAT || d->norm_dtype == BPL_DOUBLE);
    uint64_t chunks = 0;
    for (uint32_t i = 0; good && i < c.count; ++i) {
        const bpl_clip_tensor &t = c.tensor[i];
        good = t.dtype <= BPL_DOUBLE && t.elements < (1ull << 40) &&
               (t.elements == 0 || (buffers[i] != nullptr && (!write || buffers[c.count + i] != nullptr)));
        if (good && write && (d->flags & BPL_CLIP_IN_PLACE) != 0) good = buffers[i] == buffers[c.count + i];
        if (good) chunks += (t.elements * bytes_of(t.dtype) + CHUNK_BYTES - 1) / CHUNK_BYTES;
    }
    if (!good || chunks >= (1ull << 32)) {
        set_status(BPL_ERR_ARGUMENT, "clip_gradients: null buffer, unknown type or norm, or a tensor beyond 2^40 elements");
        return;
    }
    try {
        if (write && overlap(c)) {
            set_status(BPL_ERR_ARGUMENT, "clip_gradients: results share memory with one another or with other gradients");
            return;
        }
    } catch (const std::bad_alloc &) {
        set_status(BPL_ERR_ARGUMENT, "clip_gradients: no host memory");
        return;
    }
    const uint32_t max = table_for(c.count);
    c.tables = c.count ? (c.count + max - 1) / max : 1;
    double *p = static_cast<double *>(parts);
    if (d->norm_type == 2) {
        if (max == TABLE_SMALL) launch<SumOfSquares, TABLE_SMALL>(stream, c, norm_out, p);
        else if (max == TABLE_MEDIUM) launch<SumOfSquares, TABLE_MEDIUM>(stream, c, norm_out, p);
        else launch<SumOfSquares, TABLE_LARGE>(stream, c, norm_out, p);
    } else {
        if (max == TABLE_SMALL) launch<LargestMagnitude, TABLE_SMALL>(stream, c, norm_out, p);
        else if (max == TABLE_MEDIUM) launch<LargestMagnitude, TABLE_MEDIUM>(stream, c, norm_out, p);
        else launch<LargestMagnitude, TABLE_LARGE>(stream, c, norm_out, p);
    }
    launch_ok();
}
