// The norm over all gradients of a training step, and clipping (no counterpart in brainpylib):
//
//     N = (sum of g^2)^(1/2) or max |g| over all tensors;  g = g * min(1, m / (N + 1e-6))
//
// Bound by memory: the gradients are read for the norm and once more for the result, backwards, so that what was read last is
// still in L2.  The tensors' addresses travel as kernel arguments (no table in device memory: a call can be captured and needs
// no copy), a thousand to a launch.  A block's share of the chunks, and the order of all sums, depend on the sizes alone.
#include <algorithm>
#include <cstring>
#include <new>
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
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (t.entry[mid].chunk <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

template<typename T, int V>
struct alignas(sizeof(T) * V) Packet {
    T v[V];
};
__device__ __forceinline__ double wide(double v) { return v; }
template<typename T> __device__ __forceinline__ double wide(T v) { return static_cast<double>(to_float(v)); }

// (out of line: it is rarely called, and would take the registers that loads need)
template<typename T, int V>
__device__ __noinline__ double squares_in_64_bits(const Packet<T, V> p) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) sum = fma(wide(p.v[i]), wide(p.v[i]), sum);
    return sum;
}

struct SumOfSquares {
    double sum = 0.0;
    __device__ __forceinline__ void one(double v) { sum = fma(v, v, sum); }
    // Squares of a few values in 32 bits where none of them can have left the range, else in 64.
    template<typename T, int V>
    __device__ __forceinline__ void add(const Packet<T, V> &p) {
        if constexpr (sizeof(T) < 8) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) s = fmaf(to_float(p.v[i]), to_float(p.v[i]), s);
            sum += s > 1e-28f && s < 1e38f ? static_cast<double>(s) : squares_in_64_bits(p);
        } else {
            sum += squares_in_64_bits(p);
        }
    }
    __device__ __forceinline__ void join(double other) { sum += other; }
    __device__ __forceinline__ double value() const { return sum; }
};
struct LargestMagnitude {
    double most = 0.0;
    __device__ __forceinline__ void join(double v) { most = v > most || v != v ? v : most; }    // no number stays none
    __device__ __forceinline__ void one(double v) { join(fabs(v)); }
    template<typename T, int V>
    __device__ __forceinline__ void add(const Packet<T, V> &p) {
        if constexpr (sizeof(T) < 8) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float f = fabsf(to_float(p.v[i]));
                m = f > m || f != f ? f : m;
            }
            join(static_cast<double>(m));
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) one(wide(p.v[i]));
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

// `count` elements (a chunk's at most): up to the next 16-byte boundary one by one, then 16 bytes at a time, four of them on their
// way.
constexpr uint32_t AHEAD = CHUNK_BYTES / 16 / CLIP_THREADS;
static_assert(AHEAD == 4, "a chunk is four packets a thread");

template<typename T, typename Norm>
__device__ __forceinline__ void norm_of(const T *p, const uint32_t count, Norm &n) {
    constexpr uint32_t V = 16 / sizeof(T);
    const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T);
    const uint32_t head = min(count, odd ? V - odd : 0u), packets = (count - head) / V, tail = head + packets * V;
    const uint4 *body = reinterpret_cast<const uint4 *>(p + head);
    uint4 v[AHEAD];
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; ++k)
        if (threadIdx.x + k * CLIP_THREADS < packets) v[k] = body[threadIdx.x + k * CLIP_THREADS];
    for (uint32_t i = threadIdx.x; i < head; i += CLIP_THREADS) n.one(wide(p[i]));
    for (uint32_t i = tail + threadIdx.x; i < count; i += CLIP_THREADS) n.one(wide(p[i]));
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; ++k)
        if (threadIdx.x + k * CLIP_THREADS < packets) n.add(*reinterpret_cast<const Packet<T, V> *>(&v[k]));
}

template<typename Norm, int MAX>
__global__ void __launch_bounds__(CLIP_THREADS, 4)
gradient_norm_kernel(const __grid_constant__ Table<MAX> t, double *parts) {
    __shared__ double shared[CLIP_THREADS / 32];
    pdl_launch_dependents();
    Norm n;
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Entry &e = t.entry[tensor_of(t, c)];
        const unsigned long long per = CHUNK_BYTES / bytes_of(e.dtype), from = (c - e.chunk) * per;
        const uint32_t count = static_cast<uint32_t>(min(per, e.count - from));
        if (e.dtype == BPL_FLOAT) norm_of(static_cast<const float *>(e.in) + from, count, n);
        else if (e.dtype == BPL_HALF) norm_of(static_cast<const __half *>(e.in) + from, count, n);
        else if (e.dtype == BPL_BFLOAT16) norm_of(static_cast<const __nv_bfloat16 *>(e.in) + from, count, n);
        else norm_of(static_cast<const double *>(e.in) + from, count, n);
    }
    const double all = block_join(n, shared);
    if (threadIdx.x == 0) parts[blockIdx.x] = all;
}

// The norm from the parts, in every block for itself (a few hundred numbers) and in the same order.
template<typename Norm>
__device__ __forceinline__ double total_norm(const double *parts, uint32_t n_parts, bool root, double *shared) {
    Norm n;
    for (uint32_t i = threadIdx.x; i < n_parts; i += CLIP_THREADS) n.join(__ldcg(parts + i));
    const double all = block_join(n, shared);
    return root ? sqrt(all) : all;
}

template<typename T>
__device__ __forceinline__ T scaled(T v, double s) {
    if constexpr (sizeof(T) == 8) return v * s;
    else return from_float<T>(to_float(v) * static_cast<float>(s));
}

template<typename T>
__device__ __forceinline__ void scale(const T *in, T *out, const uint32_t count, const double s) {
    constexpr uint32_t V = 16 / sizeof(T);
    const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(in) & 15u) / sizeof(T);
    const bool together = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    const uint32_t head = together ? min(count, odd ? V - odd : 0u) : count, packets = (count - head) / V, tail = head + packets * V;
    const uint4 *from = reinterpret_cast<const uint4 *>(in + head);
    uint4 *to = reinterpret_cast<uint4 *>(out + head), v[AHEAD];
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; ++k)
        if (threadIdx.x + k * CLIP_THREADS < packets) v[k] = from[threadIdx.x + k * CLIP_THREADS];
    for (uint32_t i = threadIdx.x; i < head; i += CLIP_THREADS) out[i] = scaled(in[i], s);
    for (uint32_t i = tail + threadIdx.x; i < count; i += CLIP_THREADS) out[i] = scaled(in[i], s);
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; ++k)
        if (threadIdx.x + k * CLIP_THREADS < packets) {
            Packet<T, V> &e = *reinterpret_cast<Packet<T, V> *>(&v[k]);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) e.v[j] = scaled(e.v[j], s);
            to[threadIdx.x + k * CLIP_THREADS] = v[k];
        }
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
    for (uint32_t i = blockIdx.x; i < t.chunks; i += gridDim.x) {
        const uint32_t c = t.chunks - 1 - i;
        const Entry &e = t.entry[tensor_of(t, c)];
        const unsigned long long per = CHUNK_BYTES / bytes_of(e.dtype), from = (c - e.chunk) * per;
        const uint32_t count = static_cast<uint32_t>(min(per, e.count - from));
        if (e.dtype == BPL_FLOAT) scale(static_cast<const float *>(e.in) + from, static_cast<float *>(e.out) + from, count, s);
        else if (e.dtype == BPL_HALF) scale(static_cast<const __half *>(e.in) + from, static_cast<__half *>(e.out) + from, count, s);
        else if (e.dtype == BPL_BFLOAT16) scale(static_cast<const __nv_bfloat16 *>(e.in) + from, static_cast<__nv_bfloat16 *>(e.out) + from, count, s);
        else scale(static_cast<const double *>(e.in) + from, static_cast<double *>(e.out) + from, count, s);
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
