// tcgen05.cuh -- the sm_100a instructions that the dense kernels are built from, one function each: shared-memory barriers,
// tensor memory, matrix products on the fifth-generation tensor cores, clusters.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

__device__ __forceinline__ uint32_t cafe_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void cafe_bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void cafe_bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// CLUSTER: for what the other block of a pair tells through this barrier about tensor memory.  Tensor memory is ordered by the tcgen05
// fences on both sides (cafe_tc_before, cafe_tc_after) around the arrival and the wait, which therefore need no order of their own,
// only the cluster's scope.
template <bool CLUSTER = false> __device__ __forceinline__ bool cafe_bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    if constexpr (CLUSTER)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    else asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// Waits for the phase of `parity` to end, but not for good: after about a second, or when another wait of the block has run
// out (*bail), it gives up and says so.
template <bool CLUSTER> static __device__ __noinline__ bool cafe_bar_wait_on(uint32_t bar, uint32_t parity, volatile int* bail) {
    for (int i = 0; !cafe_bar_try<CLUSTER>(bar, parity); ++i) {
        if (i > (1 << 20) || ((i & 255) == 255 && *bail)) { *bail = 1; return false; }
    }
    return true;
}
template <bool CLUSTER = false> __device__ __forceinline__ bool cafe_bar_wait(uint32_t bar, uint32_t parity, volatile int* bail) {
    return cafe_bar_try<CLUSTER>(bar, parity) || cafe_bar_wait_on<CLUSTER>(bar, parity, bail);
}

// Launches that follow one another closely: the next kernel of the stream may start once all blocks of this one have, and does what
// does not depend on it; nothing that another kernel wrote is read, and nothing is written, before the wait, which ends when all
// kernels before this one are done.
__device__ __forceinline__ void cafe_next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void cafe_wait_for_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// One lane of the warp, all of whose lanes are here.  Copies, products and commits go inside a branch on it: what the instructions
// take then stays in uniform registers.  (A lane-0 predicate on every instruction cost 45 cycles each: 1410 cycles for the twelve
// products of 64 cycles of a turn, 910 with one branch around them.)
__device__ __forceinline__ bool cafe_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p;
}
__device__ __forceinline__ void cafe_fence_barrier_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
// this thread's writes to shared memory become visible to the tensor cores' reads
__device__ __forceinline__ void cafe_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void cafe_tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void cafe_tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// tensor memory: `cols` (a power of two from 32) columns of 128 lanes x 32 bits; the address is written to shared memory
__device__ __forceinline__ void cafe_tm_alloc(uint32_t to, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void cafe_tm_free(uint32_t at, uint32_t cols) { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols) : "memory"); }
__device__ __forceinline__ void cafe_tm_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 16 columns of the warp's 32 lanes: lane l gets its row's 16 values
__device__ __forceinline__ void cafe_tm_load16(uint32_t at, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}

// D[128 x N] (+)= A[128 x 16] B[N x 16]^T, operands in shared memory (descriptors), D in tensor memory
__device__ __forceinline__ void cafe_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add) : "memory");
}
// the barrier's next arrival: when all products issued so far by this lane are done
__device__ __forceinline__ void cafe_mma_commit(uint32_t bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"); }

// Rows of ROWB = 64 or 128 bytes, K contiguous, one behind the other; the 16-byte pieces of a row are exchanged by
// cafe_swizzle.  Eight rows are a unit.
template <int ROWB> __device__ __forceinline__ uint64_t cafe_operand(uint32_t at) {
    static_assert(ROWB == 64 || ROWB == 128, "row bytes");
    return (uint64_t)((at & 0x3ffffu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(ROWB * 8 / 16) << 32 | (uint64_t)1 << 46 | (uint64_t)(ROWB == 128 ? 2 : 4) << 61;
}
template <int ROWB> __device__ __forceinline__ uint32_t cafe_swizzle(int row, int piece) {
    return (uint32_t)(row * ROWB + ((piece ^ (ROWB == 128 ? row & 7 : (row >> 1) & 3)) << 4));
}
// kind::f16, fp32 sums: A and B both fp16 (0) or both bf16 (1), both K-major
__host__ __device__ constexpr uint32_t cafe_mma_instr(int type, int M, int N) {
    return 1u << 4 | (uint32_t)type << 7 | (uint32_t)type << 10 | (uint32_t)(N >> 3) << 17 | (uint32_t)(M >> 4) << 24;
}

// ---- pairs of blocks: a cluster of two whose tensor cores work on one tile.  D[256 x N] (+)= A[256 x 16] B[N x 16]^T: block 0 has
// rows 0 to 127 of A and D and the first half of B's rows, block 1 the rest; block 0 issues.
__device__ __forceinline__ void cafe_tm_alloc2(uint32_t to, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void cafe_tm_free2(uint32_t at, uint32_t cols) { asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols) : "memory"); }
__device__ __forceinline__ void cafe_mma2(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add) : "memory");
}
// the next arrival of the barrier at this place in both blocks
__device__ __forceinline__ void cafe_mma_commit2(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}

// An arrival at another block's barrier that tells of tensor memory having been read (cafe_bar_try's CLUSTER says what orders it; a
// release of the cluster's scope costs a fence each time: one for every box took 16384x1024x4096 in bf16 from 106 to 240 us).
__device__ __forceinline__ void cafe_bar_arrive_at(uint32_t cluster_bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory"); }

__device__ __forceinline__ uint32_t cafe_cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cafe_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cafe_cluster_map(uint32_t at, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 cafe_cluster_load4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float cafe_cluster_load(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// a barrier's next phase also waits for `bytes` of copies
__device__ __forceinline__ void cafe_bar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
// a box of a tensor (three axes, the innermost first) into shared memory; what lies outside the tensor becomes zero
__device__ __forceinline__ void cafe_box_load(uint32_t to, const void* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// The same into this block's shared memory, completing on a barrier of either block of a pair (an address in the cluster)
__device__ __forceinline__ void cafe_box_load2(uint32_t to, const void* map, int x, int y, int z, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(z), "r"(cluster_bar) : "memory");
}
// The operand whose other index is contiguous: panels of 64 of them (128 bytes, pieces exchanged as above) x k, eight k a unit;
// `panel` bytes from one panel to the next.
__device__ __forceinline__ uint64_t cafe_operand_mn(uint32_t at, uint32_t panel) {
    return (uint64_t)((at & 0x3ffffu) >> 4) | (uint64_t)(panel >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
