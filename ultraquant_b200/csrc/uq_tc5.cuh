// Fifth-generation tensor cores (tcgen05) and tensor memory: the few
// instructions that the 4-bit products use, with bounded waits.
#pragma once
#include "uq_tma.cuh"

namespace uq {
namespace tc5 {

#if defined(__CUDACC__)

__device__ __forceinline__ unsigned smem_addr(const void *p) { return unsigned(__cvta_generic_to_shared(p)); }

// Everything here works on pairs of CTAs (cta_group::2): one product of M = 256
// takes 128 rows of A from each CTA and half of B's N columns from each, and
// leaves 128 rows of D in each, so that every byte of B crosses from L2 once for
// 256 rows.

// ---- the cluster -----------------------------------------------------------------
__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The first CTA's address of a place in shared memory (for mbarrier arrivals).
__device__ __forceinline__ unsigned leader_addr(unsigned addr) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Warp number, the same in all lanes in a way that the compiler sees: a product's
// operands are uniform registers, and in code that it takes for divergent every
// one of them is fetched by a loop over lanes (115 cycles a product).
__device__ __forceinline__ int warp_id() { return __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0); }
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect() {
    unsigned r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// ---- tensor memory -----------------------------------------------------------
template <int COLS> __device__ __forceinline__ void tmem_alloc(unsigned dst) {   // one whole warp of each CTA
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(dst), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
template <int COLS> __device__ __forceinline__ void tmem_free(unsigned addr) {   // the warps that allocated
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(addr), "n"(COLS));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: register j of lane i is (lane i, column j).
__device__ __forceinline__ void ld32(unsigned addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
                   "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                   "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr) : "memory");
}
__device__ __forceinline__ void st32(unsigned addr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                    "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
                    "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
                    "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}

// ---- products ------------------------------------------------------------------
// Instruction descriptor of kind::f16: float32 sums, both operands of one type,
// M = 256, n a multiple of 32.  `amn`, `bmn`: the operand's M (N) index is the contiguous one.
__device__ __forceinline__ constexpr uint32_t idesc_f16(bool bf16, int n, bool amn, bool bmn) {
    return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(amn) << 15) | (uint32_t(bmn) << 16) |
           (uint32_t(n >> 3) << 17) | (uint32_t(256 >> 4) << 24);
}
// Shared-memory descriptor with the 128-byte swizzle.  Contraction index
// contiguous: rows of 128 bytes, 8 rows (1024 bytes) apart by `stride`.  M / N
// index contiguous: lines of 64 values, one line per contraction index, 8 lines
// apart by `stride`, the next 64 values `lead` bytes on.
__device__ __forceinline__ uint64_t desc128(unsigned addr, unsigned lead, unsigned stride) {
    return uint64_t((addr >> 4) & 0x3fff) | (uint64_t(lead >> 4) << 16) | (uint64_t(stride >> 4) << 32) | (uint64_t(1) << 46) |
           (uint64_t(2) << 61);
}
// D (tensor memory) (+)= A B, one instruction of 16 contraction steps; A in
// tensor memory or in shared memory.
__device__ __forceinline__ void mma_ts(unsigned d, unsigned a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
}
__device__ __forceinline__ void mma_ss(unsigned d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
}
// Arrives on the mbarrier at this place in both CTAs once every product issued so
// far by this thread is done.
__device__ __forceinline__ void commit(unsigned mbar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 :: "r"(mbar), "h"((unsigned short)3) : "memory");
}

// ---- waits ---------------------------------------------------------------------
__device__ __forceinline__ bool mbar_test(unsigned addr, unsigned parity) {
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ void mbar_arrive(unsigned addr) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(addr) : "memory");
}

// At a barrier of either CTA.  What it announces is read by the tensor cores, not
// by the waiting thread: tensor memory (after fence_before) or shared memory
// (after fence.proxy.async), complete in the CTA that wrote it.  So the default,
// block-scope order is enough; release.cluster here and acquire.cluster at every
// wait halved the rate of all three products.
__device__ __forceinline__ void mbar_arrive_remote(unsigned cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}

// A block's waits, each by a whole warp and at most LIMIT_MS long: the first that
// gives up sets *gave_up (shared memory), at which every other wait of the
// block gives up too, and *flag (global memory), which the host reads.
template <unsigned LIMIT_MS> __device__ __noinline__ bool wait_slow(unsigned addr, unsigned parity, volatile int *gave_up, int *flag) {
    unsigned long long t0, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    for (;;) {
        for (int i = 0; i < 64; ++i)
            if (mbar_test(addr, parity)) return true;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (*gave_up || now - t0 > LIMIT_MS * 1000000ull) {
            *gave_up = 1;
            atomicExch(flag, 1);
            return false;
        }
    }
}
template <unsigned LIMIT_MS> struct WaiterFor {
    volatile int *gave_up;
    int *flag;
    bool fail = false;
    __device__ __forceinline__ bool wait(unsigned addr, unsigned parity) {
        if (fail) return false;
        bool ok = mbar_test(addr, parity);
        if (!__all_sync(0xffffffffu, ok)) {
            if (!ok) ok = wait_slow<LIMIT_MS>(addr, parity, gave_up, flag);
            fail = !__all_sync(0xffffffffu, ok);
        }
        return !fail;
    }
    // For copies and products that are in flight when a role stops: at most 2 s, whatever the others do.
    static __device__ __noinline__ void drain(unsigned addr, unsigned parity) {
        unsigned long long t0, now;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
        do {
            if (mbar_test(addr, parity)) return;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        } while (now - t0 < 2000000000ull);
    }
};
using Waiter = WaiterFor<2000>;

#endif  // __CUDACC__

// Tiled 2-D map, zero fill.  `inner` of dims[0] elements of `type`, box of
// `b0` x `b1`; base and row stride multiples of 16 bytes.
inline bool encode2d(CUtensorMap *m, CUtensorMapDataType type, const void *base, uint64_t d0, uint64_t d1, uint64_t stride, uint32_t b0,
                     uint32_t b1, CUtensorMapSwizzle swizzle) {
    const tma::EncodeTiled fn = tma::encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {d0, d1}, strides[1] = {stride};
    const cuuint32_t box[2] = {b0, b1}, one[2] = {1, 1};
    return fn(m, type, 2, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tc5
}  // namespace uq
