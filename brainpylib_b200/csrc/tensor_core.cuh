// Fifth-generation tensor cores (sm_100a): descriptors of operands in shared memory, products, accumulators in tensor memory, barriers
// in shared memory.  One CTA, M = 128, operands of 16 bits, sums of 32.
#ifndef BPL_CSRC_TENSOR_CORE_CUH_
#define BPL_CSRC_TENSOR_CORE_CUH_

#include <cstdint>

namespace bpl {

__device__ __forceinline__ uint32_t shared_address(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---- barriers ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void barrier_init(uint64_t *b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(shared_address(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(shared_address(b)) : "memory");
}
// Sleeps until the barrier passes, or for up to a millisecond: warps that look again and again take the slots of those that work.
__device__ __forceinline__ bool barrier_passed(uint64_t *b, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000000;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(shared_address(b)), "r"(parity) : "memory");
    return done != 0;
}

// What threads wrote to shared memory, before the tensor cores read it (the writer's side).
__device__ __forceinline__ void fence_shared_for_tensor() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory -------------------------------------------------------------------------------------------------------
// 128 lanes of 512 columns of 32 bits; a warp reaches the 32 lanes of its place in its group of four.
__device__ __forceinline__ void tensor_alloc(uint32_t *address, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(shared_address(address)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tensor_free(uint32_t address, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(address), "r"(columns) : "memory");
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tensor_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 neighbouring columns of a warp's 32 lanes
__device__ __forceinline__ void tensor_load_16(uint32_t address, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(address) : "memory");
}
__device__ __forceinline__ void tensor_store_8(uint32_t address, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 :: "r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// 16 lanes (of the warp's 32 from `address` on) by 8 neighbouring columns, as a fragment: lane l has rows l / 4 (twice) and l / 4 + 8 (twice),
// columns 2 (l % 4) and the next one.
__device__ __forceinline__ void tensor_load_fragment(uint32_t address, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(address) : "memory");
}
// Four 8 x 8 matrices of 16 bits from fragments to shared memory, turned: lane l gives the address of column l % 8 of matrix l / 8.
__device__ __forceinline__ void store_turned(uint32_t address, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                 :: "r"(address), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// ---- products --------------------------------------------------------------------------------------------------------------
// An operand in shared memory lies in rows of 128 bytes, eight of them to 1024 aligned bytes, groups of eight one behind the other,
// 16-byte piece c of row r at place c ^ (r % 8).  Rows along M or N: the contraction along the 128 bytes.  Rows along the contraction:
// M or N along the 128 bytes, in runs of 64 elements, `wide` bytes from one to the next.  The lower word of a descriptor is what
// changes: addresses can be added to it in units of 16 bytes.
constexpr uint32_t OPERAND_HIGH = 1024 / 16 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t operand(uint32_t address, uint32_t wide = 16) { return (address & 0x3ffff) >> 4 | (wide / 16) << 16; }
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

// kind::f16, bfloat16 operands, 32-bit sums, M = 128; *_rows: the operand's rows lie along the contraction
__host__ __device__ constexpr uint32_t product_of(uint32_t n, bool a_rows, bool b_rows) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (a_rows ? 1u << 15 : 0u) | (b_rows ? 1u << 16 : 0u) | (n >> 3) << 17 | (128u >> 4) << 24;
}
// Called by a whole warp, so that operands stay in uniform registers; the lane that elect_lane() has chosen asks for the product.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t chosen;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
    return chosen;
}
__device__ __forceinline__ void multiply(uint32_t to, uint32_t a, uint32_t b, uint32_t what, bool add, uint32_t chosen) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 q, %6, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
                 :: "r"(to), "r"(a), "r"(b), "r"(what), "r"(add ? 1u : 0u), "r"(OPERAND_HIGH), "r"(chosen) : "memory");
}
// a in tensor memory: 16 elements of the contraction in 8 columns
__device__ __forceinline__ void multiply_from_tensor(uint32_t to, uint32_t a, uint32_t b, uint32_t what, bool add, uint32_t chosen) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 q, %6, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
                 :: "r"(to), "r"(a), "r"(b), "r"(what), "r"(add ? 1u : 0u), "r"(OPERAND_HIGH), "r"(chosen) : "memory");
}
// `b` is arrived at once all products that the chosen lane has asked for so far are done
__device__ __forceinline__ void products_arrive(uint64_t *b, uint32_t chosen) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" :: "r"(shared_address(b)), "r"(chosen) : "memory");
}

// ---- tiles of global memory ------------------------------------------------------------------------------------------------
// Announces `bytes` of copies to a barrier, and arrives at it.
__device__ __forceinline__ void barrier_expect(uint64_t *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(shared_address(b)), "r"(bytes) : "memory");
}
// The box of a map at (x, y, z) into shared memory; zeros where it reaches out of the tensor.
__device__ __forceinline__ void copy_box(uint32_t to, const void *map, uint32_t x, uint32_t y, uint32_t z, uint64_t *b) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(to), "l"(map), "r"(x), "r"(y), "r"(z), "r"(shared_address(b)) : "memory");
}
__device__ __forceinline__ void prefetch_map(const void *map) { asm volatile("prefetch.tensormap [%0];" :: "l"(map) : "memory"); }

}  // namespace bpl

#endif  // BPL_CSRC_TENSOR_CORE_CUH_
