// Tensor-core and shared-memory primitives of the in-kernel-split ring GEMMs:
// kind::i8 descriptors and MMAs, bounded mbarrier waits, tensor-memory loads and
// the split of ring elements into byte planes.
#pragma once
#include "common.cuh"

namespace ddg {

int ring_gemm_err_word(uint32_t **out);  // ring_gemm_tc.cu

constexpr int TC_BM = 128;  // rows of an MMA tile (TMEM lanes)
constexpr uint64_t TC_WAIT_NS = 2000000000ull;

__device__ __forceinline__ uint32_t smem_addr(const void *p)
{
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ uint64_t global_ns()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// shared-memory matrix descriptor, no swizzle (layout type 0), version 1
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo)
{
    return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t((lbo >> 4) & 0x3FFFu) << 16) |
           (uint64_t((sbo >> 4) & 0x3FFFu) << 32) | (uint64_t(1) << 46);
}

// instruction descriptor of kind::i8: u8 x u8 -> s32, A K-major, M = 128
__host__ __device__ constexpr uint32_t i8_idesc(int bn, bool b_mn_major)
{
    return (2u << 4)                          // D format s32
           | (0u << 7) | (0u << 10)           // A, B unsigned 8-bit
           | ((b_mn_major ? 1u : 0u) << 16)   // B major
           | (uint32_t(bn >> 3) << 17)        // N >> 3
           | (uint32_t(TC_BM >> 4) << 24);    // M >> 4
}

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

// wait until the phase with the given parity of `bar` has completed; false
// after TC_WAIT_NS (or 2^26 polls) without completion
__device__ inline bool mbar_wait(uint64_t *bar, uint32_t parity)
{
    if (mbar_test(bar, parity)) return true;  // the usual case, without reading the timer
    const uint64_t t0 = global_ns();
    for (uint32_t it = 1; it < (1u << 26); ++it) {
        if (mbar_test(bar, parity)) return true;
        if ((it & 255u) == 0 && global_ns() - t0 > TC_WAIT_NS) return false;
    }
    return false;
}

// one arrival on an mbarrier (release: the caller's earlier writes are visible to who waits)
__device__ __forceinline__ void mbar_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// one arrival that also announces `bytes` of asynchronous copies to come
__device__ __forceinline__ void mbar_expect(uint64_t *bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}

// true in one lane of a converged warp.  MMAs issued by an elected lane of a
// warp-uniform loop keep their descriptors in uniform registers: 4 MMAs and a
// commit take 500 cycles to issue, against 750 under threadIdx.x == 0.
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
}

// the same with A in tensor memory: row m in lane m, four bytes of K to a column
__device__ __forceinline__ void mma_i8_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t db, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 16 columns of the calling warp's 32 lanes
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void mma_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&v)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
}

__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// the four byte planes of four consecutive 32-bit words: plane q holds byte q of e0..e3
__device__ __forceinline__ void byte_planes(uint32_t e0, uint32_t e1, uint32_t e2, uint32_t e3, uint32_t (&p)[4])
{
    const uint32_t lo01 = __byte_perm(e0, e1, 0x5140), lo23 = __byte_perm(e2, e3, 0x5140);
    const uint32_t hi01 = __byte_perm(e0, e1, 0x7362), hi23 = __byte_perm(e2, e3, 0x7362);
    p[0] = __byte_perm(lo01, lo23, 0x5410);
    p[1] = __byte_perm(lo01, lo23, 0x7632);
    p[2] = __byte_perm(hi01, hi23, 0x5410);
    p[3] = __byte_perm(hi01, hi23, 0x7632);
}

template <typename T>
__device__ __forceinline__ void store_planes(uint8_t *base, uint32_t plane_bytes, uint32_t off, const T (&e)[4])
{
    uint32_t p[4];
    byte_planes(uint32_t(e[0]), uint32_t(e[1]), uint32_t(e[2]), uint32_t(e[3]), p);
#pragma unroll
    for (int q = 0; q < 4; q++) *reinterpret_cast<uint32_t *>(base + q * plane_bytes + off) = p[q];
    if constexpr (sizeof(T) == 8) {
        byte_planes(uint32_t(uint64_t(e[0]) >> 32), uint32_t(uint64_t(e[1]) >> 32), uint32_t(uint64_t(e[2]) >> 32),
                    uint32_t(uint64_t(e[3]) >> 32), p);
#pragma unroll
        for (int q = 0; q < 4; q++) *reinterpret_cast<uint32_t *>(base + (4 + q) * plane_bytes + off) = p[q];
    }
}

// asynchronous copy of `bytes` of N (4 or 8) bytes, the rest zeros, to shared memory
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

constexpr int tmem_cols(int n)
{
    int c = 32;
    while (c < n) c <<= 1;
    return c;
}

}  // namespace ddg
