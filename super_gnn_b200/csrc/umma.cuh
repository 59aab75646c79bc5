// Thin wrappers of the sm_100a instructions the tensor-core kernels here are written with: mbarriers with bounded waits,
// tiled TMA loads, tensor memory, tcgen05 matrix products; and the tensor maps on the host side.
//
// Waits are bounded: one that is not answered within two seconds gives up, the block's roles leave their loops, what
// is in flight is waited for (again with the bound), the tensor memory is freed, and a word in global memory says so.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace sgnn {

// ---- host side ----
// A row-major matrix (or a stack of `planes` of them) of 16-bit elements as a tensor map with 128-byte swizzled boxes
// of 64 columns x `box_rows` rows.  `cols` is what may be read: columns and rows beyond the extents read as zero.
int umma_tensor_map(CUtensorMap *map, const void *base, bool bf16, int64_t cols, int64_t rows, int64_t ld, int planes,
                    int64_t plane_stride, int box_rows);

// A matrix of elements of 1, 2 or 4 bytes as boxes of `box_cols` x `box_rows` that lie in shared memory row after row
int raw_tensor_map(CUtensorMap *map, const void *base, int elem_bytes, int64_t cols, int64_t rows, int64_t ld, int box_cols, int box_rows);

// Results that leave a warp as 32 rows of `box_cols` columns (128 or 64 bytes a row, swizzled as wide)
enum class StoreType { kF32, kBf16, kF16 };
int umma_store_map(CUtensorMap *map, void *base, StoreType type, int64_t cols, int64_t rows, int64_t ld, int planes,
                   int64_t plane_stride, int box_cols);

#ifdef __CUDACC__

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint64_t *bar, unsigned count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t *bar, unsigned bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *bar, unsigned parity)
{
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint64_t now_ns()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

constexpr uint64_t kWaitNs = 2000000000ull;

// Waits for the phase; false when another role gave up (*gone) or when the bound has passed, which sets *gone.
__device__ __forceinline__ bool bar_wait(uint64_t *bar, unsigned parity, volatile int *gone)
{
    if (bar_try(bar, parity)) return true;
    const uint64_t until = now_ns() + kWaitNs;
    for (int i = 0; i < (1 << 28); ++i) {
        if (bar_try(bar, parity)) return true;
        if (*gone) return false;
        if (now_ns() > until) break;
    }
    *gone = 1;
    return false;
}

// Fills that buffer s of a ring has had once `used` of them have been dealt over the buffers in turn; the last one of them completes
// the phase of parity (fills - 1) & 1 of the buffer's barrier
__host__ __device__ constexpr unsigned ring_fills(unsigned used, unsigned s, unsigned buffers)
{
    return used > s ? (used - 1 - s) / buffers + 1 : 0;
}

// Waits for what is in flight after a role gave up: the bound alone, whatever the others say.
__device__ __forceinline__ void bar_drain(uint64_t *bar, unsigned parity)
{
    const uint64_t until = now_ns() + kWaitNs / 8;
    for (int i = 0; i < (1 << 28) && now_ns() < until; ++i)
        if (bar_try(bar, parity)) return;
}

// The same for every buffer of a ring that copies may still be on their way to; one that was never filled is not waited for
__device__ __forceinline__ void ring_drain(uint64_t *bars, unsigned used, int buffers)
{
    for (int s = 0; s < buffers; ++s) {
        const unsigned fills = ring_fills(used, s, buffers);
        if (fills > 0) bar_drain(bars + s, (fills - 1) & 1);
    }
}

// ---- two blocks of a cluster that work on one product (cta_group::2): the first of them leads ----
__device__ __forceinline__ unsigned cluster_rank()
{
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of the same place in the leading block's shared memory
__device__ __forceinline__ uint32_t leader_addr(const void *p)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(p)));
    return a;
}
__device__ __forceinline__ void leader_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(bar)) : "memory");
}
// into this block's shared memory, counted by the leader's barrier
__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

// columns [x, x + 64) of rows [y, y + box rows) of plane z
__device__ __forceinline__ void tma_load(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap *map)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// A box in shared memory to global memory, or added to what is there; boxes are cut off at the extents.  The issuing
// thread waits with store_wait_read before the box is written again and with store_wait_all before it leaves.
__device__ __forceinline__ void tma_store(const CUtensorMap *map, const void *src, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y),
                 "r"(z), "r"(smem_addr(src))
                 : "memory");
}
__device__ __forceinline__ void tma_add(const CUtensorMap *map, const void *src, int x, int y, int z)
{
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x),
                 "r"(y), "r"(z), "r"(smem_addr(src))
                 : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A run of memory (16-byte aligned on both sides, a multiple of 16 bytes) into shared memory, and back
__device__ __forceinline__ void bulk_load(void *dst, const void *src, unsigned bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(dst)), "l"(src),
                 "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void bulk_store(void *dst, const void *src, unsigned bytes)
{
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_addr(src)), "r"(bytes) : "memory");
}

__device__ __forceinline__ void tmem_alloc(uint32_t *slot, int cols)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t base, int cols)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_alloc_pair(uint32_t *slot, int cols)
{
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t base, int cols)
{
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
}
// the barrier at this place in both blocks
__device__ __forceinline__ void tc_commit_pair(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}

// arrives on the barrier once every product issued before by this thread has finished
__device__ __forceinline__ void tc_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Operand in shared memory, 128-byte swizzle.  Rows of 64 elements (128 bytes) in groups of eight (1024 bytes):
//   K-major  (the 64 elements run along the reduction): rows are the outer dimension, group after group;
//   MN-major (the 64 elements run along the outer dimension): rows are steps of the reduction; a second run of 64 outer
//   elements lies `run_bytes` further on.
// group_bytes / run_bytes: distance of eight-row groups, distance of 64-element runs.
__device__ __forceinline__ uint64_t umma_desc(const void *p, unsigned run_bytes, unsigned group_bytes)
{
    return (uint64_t)((smem_addr(p) & 0x3FFFFu) >> 4) | ((uint64_t)(run_bytes >> 4) << 16) | ((uint64_t)(group_bytes >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}

// m x n product of 16-bit operands with fp32 sums: m = 128, or 256 of two blocks
__device__ __forceinline__ uint32_t umma_idesc(bool bf16, bool a_mn, bool b_mn, int n, int m = 128)
{
    const uint32_t t = bf16 ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add)
                 : "memory");
}

// The product of two blocks: each has 128 rows of the first operand, half of the second's columns, 128 rows of the result
__device__ __forceinline__ void umma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add)
                 : "memory");
}

// The same with the first operand in tensor memory: lanes are its rows, a 32-bit column two steps of the reduction
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"((unsigned)add)
                 : "memory");
}

// 4 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_store4(uint32_t addr, const uint32_t (&r)[4])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this warp's 32 lanes (one row a thread)
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32])
{
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16])
{
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}

// Until the wait the registers of a load may not be touched.  The compiler is not told by the wait itself: what is read after it passes
// through here, so that no use can move in front.
__device__ __forceinline__ void tmem_load_wait(float (&v)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
          "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]),
          "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]),
          "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
        :
        : "memory");
}
__device__ __forceinline__ void tmem_load_wait(float (&v)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
          "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
        :
        : "memory");
}

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

#endif  // __CUDACC__
}  // namespace sgnn
