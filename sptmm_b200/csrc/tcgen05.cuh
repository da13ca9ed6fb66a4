// tcgen05.cuh -- the sm_100a instructions the tensor-core attention kernels issue: bounded mbarrier
// waits, TMA tile loads, tcgen05 products and tensor-memory access.
#pragma once
#include <cuda.h>

#include "attention.cuh"

namespace sptmm {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// One poll; the hardware may suspend the thread in it, here for up to a millisecond.  Without that time
// the waiting warps poll so often that they take issue slots from the others' exponentials: a prompt of
// 8192 tokens took 326 us (389 with a tighter loop) against 286.
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000000) : "memory");
    return ok;
}

__device__ __forceinline__ uint64_t nanoseconds()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// Every wait is bounded: after two seconds (and a thousand polls, in case the GPU was away in between), or
// this many polls, where a wait of the kernel takes microseconds, the waiter raises the CTA's abort word, which
// ends all other waits of the CTA at their next look at it.
constexpr uint32_t kWaitPolls = 1u << 24;
constexpr uint64_t kWaitNs = 2000000000ull;

__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t *abort_word)
{
    if (mbar_try(bar, parity)) return true;
    const uint64_t start = nanoseconds();
    for (uint32_t i = 0; i < kWaitPolls; i++) {
        if (mbar_try(bar, parity)) return true;
        if (*abort_word) return false;
        if (i >= 1000 && nanoseconds() - start > kWaitNs) break;
    }
    *abort_word = 1;
    return false;
}
// The same by a whole warp, with one answer for all lanes (an abort may be seen by some lanes first).
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t *abort_word)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_word));
}

// A wait that raises the abort word after `polls` looks, none of which suspends the thread.  Not inlined: the kernel's
// softmax loop would spill registers for it (a prompt of 8192 tokens 282 us for 276).
static __device__ __noinline__ void mbar_poll(uint32_t bar, uint32_t parity, volatile uint32_t *abort_word, uint32_t polls)
{
    for (uint32_t i = 0; i < polls; i++) {
        uint32_t ok;
        asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok || *abort_word) return;
    }
    *abort_word = 1;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z, int w)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// ---- tensor memory ----
__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, uint32_t cols)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 32 neighbouring 32-bit columns of the warp's 32 lanes; r[i] is column i of the thread's own lane
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// The registers of a load hold their values only after the wait: passing them through an empty
// statement behind it keeps the compiler from using them earlier.
__device__ __forceinline__ void pin32(uint32_t *r)
{
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
          "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
          "r"(r[30]), "r"(r[31])
        : "memory");
}

// ---- operands ----
// Shared-memory descriptor of a tile of 128-byte rows with the 128-byte swizzle (as TMA writes it),
// 1024-byte aligned.  K-major operands (the contracted index runs along a row): `stride` = 1024 from
// eight rows to the next eight, `lead` unused.  MN-major ones (the contracted index runs over rows):
// `stride` = 1024 likewise, `lead` from 64 columns to the next 64.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride)
{
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)((stride >> 4) & 0x3fff) << 32 |
           1ull << 46 | 2ull << 61;
}
// Instruction descriptor: fp32 accumulator, both operands of one 16-bit type, M = 128.
__host__ __device__ constexpr uint32_t mma_desc(bool bf16, uint32_t n, bool b_mn_major)
{
    return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (b_mn_major ? 1u : 0u) << 16 | (n >> 3) << 17 | (128u >> 4) << 24;
}
// Only the low word of a shared-memory descriptor changes from step to step (the address is there).
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, bool add)
{
    asm volatile("{ .reg .pred p; .reg .b64 a, b; setp.ne.b32 p, %6, 0; mov.b64 a, {%1, %2}; mov.b64 b, {%3, %4};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p; }"
                 ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, bool add)
{
    asm volatile("{ .reg .pred p; .reg .b64 b; setp.ne.b32 p, %5, 0; mov.b64 b, {%2, %3};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p; }"
                 ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"((uint32_t)add) : "memory");
}

// One lane of a converged warp.  The products are issued by code the whole warp walks through, with only
// the instructions themselves under this predicate: their operands then stay in uniform registers.
__device__ __forceinline__ bool elect_one()
{
    uint32_t ok;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(ok));
    return ok;
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// ---- host: tensor maps ----
// A map of 16-bit elements with 128-byte swizzle and boxes 64 elements wide (what lies beyond a
// dimension reads as zero).  dims[0] is the contiguous one; strides (bytes) belong to dims[1..].
int make_tensor_map(const char *who, CUtensorMap *map, const void *base, uint32_t dtype, uint32_t rank, const uint64_t *dims,
                    const uint64_t *strides, const uint32_t *box);
int attention_status_word(uint32_t **dev_word);      // device address of the library's word for expired waits
uint32_t attention_wait_polls();                     // of the calls from now on; 0: no limit

}  // namespace sptmm
