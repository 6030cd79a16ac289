// tc.cuh — barriers, TMA tile loads and tcgen05 instructions of one CTA, as
// the attention kernels use them.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace concord {
namespace tc {

// A wait runs out after 2 s in which its warp ran: of the time between two looks
// at the clock (wall time) at most 100 ms count, so a kernel that was taken off
// the GPU meanwhile has lost nothing.  Once a wait has run out somewhere on the
// device the others get 20 ms, so a grid of many blocks still ends soon.
constexpr uint64_t WAIT_NS = 2000000000ull, LATER_NS = 20000000ull, SLICE_NS = 100000000ull;

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void sts16(uint32_t a, const uint4& v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
struct Patience {
    uint64_t last = 0, ran = 0;
    __device__ __forceinline__ bool over(const int* err) {
        const uint64_t t = now_ns();
        ran += last ? min(t - last, SLICE_NS) : 0;
        last = t;
        return ran > LATER_NS && (ran > WAIT_NS || *reinterpret_cast<const volatile int*>(err) != 0);
    }
};
// The barriers of a block stand in 512 aligned bytes of shared memory, of which
// the last word says that a wait of the block has run out (the address of any
// of them leads there, so nothing is kept in registers for it).
constexpr uint32_t BARRIERS = 512;
__device__ __forceinline__ uint32_t gave_up_word(uint32_t bar) { return (bar & ~(BARRIERS - 1)) + BARRIERS - 4; }
__device__ __forceinline__ void set_gave_up(uint32_t bar, uint32_t v) {
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(gave_up_word(bar)), "r"(v) : "memory");
}
__device__ __forceinline__ bool gave_up(uint32_t bar) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(gave_up_word(bar)) : "memory");
    return v != 0;
}
// By one thread: false once the wait has run out, the first such wait's code then
// in *err, or at once where another of the block has.  (The loops are calls: as
// code in every place they made the forward of 64 x 256 tokens 4 us slower than
// its 31.)
__device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, int* err, int code) {
    Patience patience;
    for (int i = 1;; ++i) {
        if (mbar_try(bar, parity)) return true;
        if (gave_up(bar)) return false;
        if ((i & 15) == 0 && patience.over(err)) break;      // (reading the clock is slow)
    }
    set_gave_up(bar, 1);
    atomicCAS(err, 0, code);
    return false;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int* err, int code) {
    return mbar_try(bar, parity) || mbar_wait_slow(bar, parity, err, code);
}
// The same by a whole warp, which stays converged: every branch goes by a vote,
// so that all lanes go on or none does.
__device__ __noinline__ bool warp_wait_slow(uint32_t bar, uint32_t parity, int* err, int code) {
    Patience patience;
#pragma unroll 1
    for (int i = 1; !__all_sync(0xffffffffu, mbar_try(bar, parity)); ++i) {
        if (__any_sync(0xffffffffu, gave_up(bar))) return false;
        if ((i & 15) == 0 && __any_sync(0xffffffffu, patience.over(err))) {
            set_gave_up(bar, 1);
            atomicCAS(err, 0, code);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err, int code) {
    return __all_sync(0xffffffffu, mbar_try(bar, parity)) || warp_wait_slow(bar, parity, err, code);
}
// Given up after `sent` tiles into a ring of `stages` (their barriers 8 bytes
// apart): what is on its way lands first, or that wait too runs out.
__device__ __noinline__ bool ring_landed(uint32_t full, int stages, int sent, int* err) {
    for (int x = max(0, sent - stages); x < sent; ++x) {
        const uint32_t bar = full + 8u * (x % stages), parity = (x / stages) & 1;
        Patience patience;
        while (!mbar_try(bar, parity))
            if (patience.over(err)) return false;
    }
    return true;
}

// one box {64 columns, 1 head, 128 rows} into 128 rows of 128 swizzled bytes
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int col, int head,
                                         int row) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(col), "r"(head), "r"(row)
        : "memory");
}

__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The products are issued by a whole warp, converged, the instruction itself
// predicated on one elected lane: the operands then stay in uniform registers.
// Issued from inside a branch on the lane, each needs its descriptors moved
// there first: eight take 750 cycles in place of 60 to 125 (and 512 to run).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p;
}
// a value that all lanes hold, known to be the same
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// D (tensor memory) = A (shared memory) B (shared memory) [+ D]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
        : "memory");
}
// D (tensor memory) = A (tensor memory) B (shared memory) [+ D]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
        : "memory");
}
// one arrival on `bar` once every MMA that the elected lane has issued is complete
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(one)
        : "memory");
}

template <int COLS> __device__ __forceinline__ void tmem_alloc(uint32_t slot) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int COLS> __device__ __forceinline__ void tmem_free(uint32_t base) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(COLS));
}

// 32 columns of this warp's 32 lanes (one lane a thread); no wait
__device__ __forceinline__ void ld32(uint32_t a, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a));
}
__device__ __forceinline__ void st32(uint32_t a, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void st16(uint32_t a, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// shared-memory matrix descriptor, 128-byte swizzle (start, leading and
// stride byte offsets >> 4, version 1, layout type 2)
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 |
           (uint64_t)((sbo >> 4) & 0x3FFF) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// A tile of 128 rows x 64 or 128 columns is one or two boxes of 128 rows x 64
// columns (16 KB each, 8-row groups of swizzled 128-byte rows 1024 B apart).
constexpr uint32_t BOX = 16384;
// columns are the reduction (K-major); the kk-th 16 columns are at + step_k(kk)
__device__ __forceinline__ uint64_t desc_k(uint32_t tile) { return smem_desc(tile, 16, 1024); }
__host__ __device__ constexpr uint64_t step_k(int kk) { return ((kk >> 2) * BOX + (kk & 3) * 32) >> 4; }
// rows are the reduction (MN-major), the second 64 columns one box on; the kk-th 16 rows are at + step_mn(kk)
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile) { return smem_desc(tile, BOX, 1024); }
__host__ __device__ constexpr uint64_t step_mn(int kk) { return (kk * 2048) >> 4; }

// 128 rows of 16 columns (K-major, one step), no swizzle: 8 rows of 8 columns
// are 128 consecutive bytes, the second 8 columns 128 B on, the next rows 256 B
constexpr uint32_t THIN = 4096;
__device__ __forceinline__ uint64_t desc_thin(uint32_t tile) {
    return (uint64_t)((tile >> 4) & 0x3FFF) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(256 >> 4) << 32 | (uint64_t)1 << 46;
}
__device__ __forceinline__ uint32_t thin_row(int r) { return (r >> 3) * 256 + (r & 7) * 16; }    // its first 8 columns

// instruction descriptor: fp32 accumulator, A and B of one 16-bit type, M = 128
__host__ __device__ constexpr uint32_t instr_desc(int bf16, int n, int b_mn) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// zero rows [from, 128) of a tile in shared memory (whole warp)
template <int DP> __device__ __forceinline__ void zero_rows(uint8_t* tile, int from) {
    const int lane = threadIdx.x & 31;
    const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll 1
    for (int b = 0; b < DP / 64; ++b)
        for (int i = from * 8 + lane; i < 128 * 8; i += 32) reinterpret_cast<uint4*>(tile + b * BOX)[i] = z;
    fence_async();
    __syncwarp();
}

}  // namespace tc
}  // namespace concord
