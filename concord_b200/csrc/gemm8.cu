// gemm8.cu — the weight gradient of a linear layer from its input in 8 bits.
//
//   dw[n, k] = sum over tokens t of dy[t, n] x[t, k],  x as kept (eight.cuh)
//
// Transposed on the tensor cores: a CTA pair (cta_group::2) owns 256 features x 256
// outputs, features along the accumulator's rows.  x is the A operand and goes
// through tensor memory: a lane there is one feature, so a thread reads 64
// tokens of its feature as four 16-byte pieces, makes bf16 of them (exact: a
// code has 7 bits and the scale is a power of two) and stores 32 columns.  x
// thus never takes the 16-bit round trip through memory, and shared memory,
// which holds a half of dy's tile a CTA as the B operand and is read once a
// pair for it, is less busy than with two 16-bit operands.
//
// Warp roles: warp 0 loads (dy by TMA tiles, a tile of codes and scales by one bulk copy),
// warp 1 of the leader issues the products, warps 4-11 convert, alternate stages
// of 64 tokens by the two groups of four, and afterwards store the
// accumulator (256 columns; the other 256 hold 8 stages of A).
//
// Whole tiles go round the pairs, which walk the tokens in step, so that a stage's
// data come from memory once and are in the L2 for everybody else (parts of equal
// length but different beginnings read 16384 x 2048 x 2048 from memory eight times:
// 150 us for the loads alone).  The tiles that are left over when rounds no longer fill
// are cut: each has a pair for its first tokens, as many as shared out evenly, and
// the other pairs share the line of their ends.  Cut tiles leave fp32 pieces in
// the workspace, which a second kernel adds in token order: the same bits on every run of one device.
//
// Every wait is bounded (tc.cuh): where one runs out, loads and products stop,
// what both CTAs have in flight lands (bounded again), the pair's remaining outputs become NaN and
// the device's error word is set, and its copy in host memory, by which later calls refuse (concord_gemm_dw8_error).
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "common.cuh"
#include "eight.cuh"
#include "errwords.cuh"
#include "tc.cuh"

namespace concord {
int bind_current_context(const char* name);

namespace g8 {

using namespace tc;

constexpr int THREADS = 384;
constexpr int FEATS = 128, OUTS = 128;            // of one CTA; a pair has twice both
constexpr int TOKENS = 64;                        // a stage
constexpr int STAGES = 8;
constexpr int DY_BYTES = TOKENS * OUTS * 2, X_BYTES = eight::TILE_BYTES;
static_assert(FEATS == eight::FEATS && TOKENS == eight::TOKENS, "a stage reads one tile of codes");
constexpr int CODES = STAGES * DY_BYTES, BARS = CODES + STAGES * X_BYTES;
constexpr int NBARS = 4 * STAGES + 3;
static_assert(BARS % BARRIERS == 0 && NBARS * 8 + 8 <= (int)BARRIERS - 4, "barriers, the tensor memory's address, tiles sent, the word");
constexpr size_t SMEM = BARS + BARRIERS + 1024;
constexpr int ACC = 256;                          // columns of the accumulator; stage s of A stands at ACC + 32 s
constexpr int TILE = 256;

struct Params {
    int64_t M;
    int N, K, tiles_n, stages;                    // stages of a tile
    int full, rest, cut, helpers;                 // tiles of full rounds, the others, their first part's stages, pairs for the ends
    const uint8_t* saved;
    __nv_bfloat16* dw;
    float* part;                                  // pieces of the rest: [2 pairs][256 outputs][256 features]
    int *err, *err_host;
};

// The rest's ends, tile after tile, are one line of stages.  Where helper h of them begins:
__device__ __forceinline__ int64_t end_start(const Params& P, int64_t h) {
    return h * ((int64_t)P.rest * (P.stages - P.cut)) / P.helpers;
}
// and whose part stage t is in
__device__ __forceinline__ int helper_of(const Params& P, int64_t t) {
    return (int)(((t + 1) * P.helpers - 1) / ((int64_t)P.rest * (P.stages - P.cut)));
}

// one piece of a pair's work after another
struct Pieces {
    int64_t at, end;                              // a helper's part of the line
    int next_tile, pairs, pair;
    int tile, s0, s1, slot;                       // slot: of the workspace; -1: a whole tile
    __device__ __forceinline__ Pieces(const Params& P) : at(0), end(0) {
        pairs = (int)(gridDim.x >> 1);
        next_tile = pair = (int)(blockIdx.x >> 1);
        const int h = pair - P.rest;
        if (h >= 0 && h < P.helpers) {
            at = end_start(P, h);
            end = end_start(P, h + 1);
        }
    }
    __device__ __forceinline__ bool next(const Params& P) {
        if (next_tile < P.full + P.rest) {
            tile = next_tile;
            next_tile += pairs;
            s0 = 0;
            s1 = tile < P.full ? P.stages : P.cut;
            slot = s1 == P.stages ? -1 : tile - P.full;
            return true;
        }
        if (at >= end) return false;
        const int len = P.stages - P.cut, j = (int)(at / len);
        tile = P.full + j;
        s0 = P.cut + (int)(at % len);
        s1 = (int)min((int64_t)P.stages, s0 + (end - at));
        slot = pair + j;                          // (grows from piece to piece along the line)
        at += s1 - s0;
        return true;
    }
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// this address in the shared memory of a CTA of the pair; 0 is the leader
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t leaders(uint32_t addr) { return in_cta(addr, 0); }
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t load_cluster(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// What the arrival says is ordered is in tensor memory alone (tcgen05.wait::st or ::ld
// and the fence before it), so it need not release memory to the cluster: that
// takes 1400 cycles, which the stages' arrivals would wait for one after another.
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(leaders(bar)) : "memory");
}
// By a converged warp, one elected lane: a tile {64 outputs, 64 tokens} of dy
// into this CTA, counted on the leader's barrier
__device__ __forceinline__ void load_dy(uint32_t dst, const CUtensorMap* map, uint32_t bar, int n, int t, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(n), "r"(t), "r"(one)
        : "memory");
}
__device__ __forceinline__ void load_bytes(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %4, 0;\n\t"
        "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(dst),
        "l"(src), "r"(bytes), "r"(bar), "r"(one)
        : "memory");
}
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %2, 0;\n\t"
        "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
        "r"(bytes), "r"(one)
        : "memory");
}
// What a CTA of a pair in which a wait has run out sent lands, or that wait too runs out (false): one thread of each CTA,
// between two barriers of the cluster.  `sent`: the word in which each CTA left its number of stages.  Its codes count on its
// own barriers; both halves of dy on the leader's, which expects them as far as it sent stages itself: for those that the
// other CTA alone sent it now expects that half, and a half that was not sent is taken off.  (Neither is a whole
// ring ahead: it waits for products that need both.)
__device__ __noinline__ bool pair_landed(uint32_t cfull, uint32_t bfull, uint32_t sent, uint32_t half, uint32_t rank, int* err) {
    const int mine = (int)load_cluster(in_cta(sent, rank));
    bool ok = ring_landed(cfull, STAGES, mine, err);
    if (rank == 0) {
        const int theirs = (int)load_cluster(in_cta(sent, 1));
        for (int x = mine; x < theirs; ++x) mbar_expect(bfull + 8u * (x % STAGES), half);
        for (int x = theirs; x < mine; ++x)
            asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bfull + 8u * (x % STAGES)), "r"(half) : "memory");
        ok = ring_landed(bfull, STAGES, max(mine, theirs), err) && ok;
    }
    return ok;
}
// accumulator (both CTAs' tensor memory) = A (tensor memory) B (both CTAs' shared memory) [+ itself]
__device__ __forceinline__ void mma_pair(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
        : "memory");
}
// one arrival on this barrier of both CTAs once every product so far is complete
__device__ __forceinline__ void commit_pair(uint32_t bar, uint32_t one) {
    const uint16_t both = 3;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
        "h"(both), "r"(one)
        : "memory");
}
// 256 features (A, tensor memory) x 256 outputs (B, rows are the reduction), bf16, fp32 accumulator
constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((256u >> 3) << 17) | ((256u >> 4) << 24);

__device__ __forceinline__ uint32_t lds1(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// Two codes (the low bytes of both halves) as bf16.  128 + their low 7 bits is
// 0x4300 | bits; what has to come off, 128 or (negative ones) 256, is 0x4300 |
// the sign bit, which is where bf16 has the last bit of its exponent.
__device__ __forceinline__ uint32_t two(uint32_t word, uint32_t pick, uint32_t scale2) {
    const uint32_t w = __byte_perm(word, 0, pick);
    const uint32_t a = (w & 0x007f007fu) | 0x43004300u, c = (w & 0x00800080u) | 0x43004300u;
    uint32_t v;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(c));
    asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(scale2));
    return v;
}

__device__ __forceinline__ void tell_host(const int* err, int* err_host) {
    *reinterpret_cast<volatile int*>(err_host) = *reinterpret_cast<const volatile int*>(err);
    __threadfence_system();
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    dw8_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ Params P) {
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + BARS);
    uint32_t* slot = reinterpret_cast<uint32_t*>(bars + NBARS);
    const uint32_t base = smem_u32(smem), bar0 = smem_u32(bars), sent_word = bar0 + NBARS * 8 + 4;
    auto cfull = [&](int s) { return bar0 + 8u * s; };                       // this CTA's codes and scales have landed
    auto bfull = [&](int s) { return bar0 + 8u * (STAGES + s); };            // leader: both halves of dy have
    auto afull = [&](int s) { return bar0 + 8u * (2 * STAGES + s); };        // leader: both CTAs' A is in tensor memory
    auto empty = [&](int s) { return bar0 + 8u * (3 * STAGES + s); };        // the stage's products are done
    const uint32_t tfull = bar0 + 8u * (4 * STAGES), tempty = tfull + 8, drained = tfull + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(cfull(s), 1);
            mbar_init(bfull(s), 1);
            mbar_init(afull(s), 8);               // four warps of each CTA
            mbar_init(empty(s), 1);
        }
        mbar_init(tfull, 1);
        mbar_init(tempty, 16);                    // eight warps of each CTA
        mbar_init(drained, 1);
        set_gave_up(bar0, 0);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    cluster_sync();
    fence_after();
    const uint32_t tm = *slot;

    if (warp == 0) {
        const uint32_t one = elect_one();
        const int64_t row = eight::row_bytes(P.K);
        Pieces pc(P);
        int s = 0, sent = 0;
        uint32_t ph = 0;
        bool ok = true;
        while (ok && pc.next(P)) {
            const int k0 = pc.tile / P.tiles_n * TILE + (int)rank * FEATS, n0 = pc.tile % P.tiles_n * TILE + (int)rank * OUTS;
            const uint32_t bytes = max(0, min(FEATS, (int)eight::padded(P.K) - k0)) * (TOKENS + 2);
            const uint8_t* x = P.saved + pc.s0 * row + (int64_t)(k0 / FEATS) * X_BYTES;
            for (int i = pc.s0; i < pc.s1; ++i, x += row) {
                if (!(ok = warp_wait(empty(s), ph ^ 1, P.err, 1))) break;
                const uint32_t dy = uniform(base + s * DY_BYTES), lb = uniform(leaders(bfull(s))), cb = uniform(cfull(s));
                if (rank == 0) expect(uniform(bfull(s)), 2 * DY_BYTES, one);
                expect(cb, bytes, one);
                load_dy(dy, &map_dy, lb, n0, i * TOKENS, one);
                load_dy(dy + DY_BYTES / 2, &map_dy, lb, n0 + 64, i * TOKENS, one);
                if (bytes) load_bytes(uniform(base + CODES + s * X_BYTES), x, bytes, cb, one);
                ++sent;
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
        }
        if (lane == 0) store_cluster(in_cta(sent_word, rank), sent);
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t one = elect_one();
            Pieces pc(P);
            int s = 0;
            uint32_t ph = 0, turn = 0;
            bool ok = true;
            while (ok && pc.next(P)) {
                if (!(ok = warp_wait(tempty, turn ^ 1, P.err, 2))) break;
                turn ^= 1;
                fence_after();
                for (int i = pc.s0; i < pc.s1; ++i) {
                    if (!(ok = warp_wait(afull(s), ph, P.err, 3) && warp_wait(bfull(s), ph, P.err, 4))) break;
                    fence_after();
                    const uint64_t b = smem_desc(uniform(base + s * DY_BYTES), DY_BYTES / 2, 1024);
                    const uint32_t a = uniform(tm + ACC + s * 32);
#pragma unroll
                    for (int kk = 0; kk < TOKENS / 16; ++kk)
                        mma_pair(tm, a + kk * 8, b + step_mn(kk), IDESC, i != pc.s0 || kk, one);
                    commit_pair(empty(s), one);
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
                if (ok) commit_pair(tfull, one);
            }
        }
    } else if (warp >= 4) {
        const int half = (warp - 4) >> 2, q = warp & 3;       // stages of this parity; lanes of the tensor memory
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        Pieces pc(P);
        int s = 0, parity = 0;
        uint32_t ph = 0, turn = 0;
        bool ok = true;
        while (pc.next(P)) {
            // (a lane beyond the tile's features converts what stands there: its row of A is no output)
            const int width = max(16, min(FEATS, (int)eight::padded(P.K) - (pc.tile / P.tiles_n * TILE + (int)rank * FEATS)));
            for (int i = pc.s0; ok && i < pc.s1; ++i) {
                if (parity == half) {
                    if (!(ok = warp_wait(cfull(s), ph, P.err, 5))) break;
                    fence_after();
                    const uint32_t at = base + CODES + s * X_BYTES + (q * 32 + lane) * 16;
                    const uint32_t sc = base + CODES + s * X_BYTES + TOKENS * width + q * 32 + lane;
                    uint4 c[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[j] = lds16(at + j * width * 16);
                    const uint32_t s0 = lds1(sc) * 0x00800080u, s1 = lds1(sc + width) * 0x00800080u;
                    uint32_t r[32];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t w[4] = {c[j].x, c[j].y, c[j].z, c[j].w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            r[j * 8 + 2 * k] = two(w[k], 0x4140, j < 2 ? s0 : s1);
                            r[j * 8 + 2 * k + 1] = two(w[k], 0x4342, j < 2 ? s0 : s1);
                        }
                    }
                    st32(tm + ACC + s * 32 + lanes, r);
                    wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_leader(afull(s));
                }
                parity ^= 1;
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
            ok = ok && warp_wait(tfull, turn, P.err, 6);
            turn ^= 1;
            fence_after();
            // 32 features x 128 outputs a warp, a feature a lane
            const int f0 = (int)rank * FEATS + q * 32 + lane, k = pc.tile / P.tiles_n * TILE + f0;
            const int n0 = pc.tile % P.tiles_n * TILE + half * 128;
            const bool whole = pc.slot < 0;
            float* part = P.part + (int64_t)max(pc.slot, 0) * (TILE * TILE) + half * 128 * TILE + f0;
#pragma unroll 1
            for (int c = 0; c < 128; c += 32) {
                uint32_t r[32];
                ld32(tm + half * 128 + c + lanes, r);
                wait_ld();
                if (!ok) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = 0x7fffffffu;
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) part[(c + j) * TILE] = __uint_as_float(r[j]);
                } else if (k < P.K) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (n0 + c + j < P.N) P.dw[(int64_t)(n0 + c + j) * P.K + k] = __float2bfloat16_rn(__uint_as_float(r[j]));
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) arrive_leader(tempty);
        }
    }
    fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && gave_up(bar0)) store_cluster(in_cta(gave_up_word(bar0), rank ^ 1), 1);
    __syncwarp();                                 // (the cluster's barrier wants whole warps)
    cluster_sync();
    if (gave_up(bar0)) {                          // here or in the other CTA: copies and products in flight end first
        if (threadIdx.x == 0) {
            tell_host(P.err, P.err_host);
            pair_landed(cfull(0), bfull(0), sent_word, DY_BYTES, rank, P.err);
        }
        if (warp == 1) {
            if (rank == 0) commit_pair(drained, elect_one());
            Patience patience;
            while (!__all_sync(0xffffffffu, mbar_try(drained, 0)) && !__any_sync(0xffffffffu, patience.over(P.err))) {}
        }
        __syncthreads();
        __syncwarp();
        cluster_sync();
    }
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512));
    }
}

// A rehearsal of a wait that runs out.  First pair_landed where the CTAs have sent as many stages, or one of them more: code
// 98 where it does not see them land; then a wait on a barrier that nobody arrives on: code 99.  dy: 64 x 64.
constexpr int CHECKS = 3, CHECK_CODES = CODES / 2, CHECK_BARS = CHECK_CODES + STAGES * 1024;
constexpr size_t CHECK_SMEM = CHECK_BARS + BARRIERS + 1024;
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(32)
    wait_check_kernel(const __grid_constant__ CUtensorMap map_dy, const void* codes, int* err, int* err_host) {
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023) & ~1023u, bar0 = base + CHECK_BARS, one = elect_one(), rank = cluster_rank();
    const uint32_t alone = bar0 + CHECKS * 2 * STAGES * 8, sent_word = alone + 8;
    static_assert((CHECKS * 2 * STAGES + 1) * 8 + 4 <= (int)BARRIERS - 4, "barriers, tiles sent, the word");
    if (threadIdx.x == 0) {
        for (int i = 0; i <= CHECKS * 2 * STAGES; ++i) mbar_init(bar0 + 8u * i, 1);
        set_gave_up(bar0, 0);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    cluster_sync();
    for (int i = 0; i < CHECKS; ++i) {
        const int first = i == 1 ? 7 : 3, second = i == 2 ? 8 : 3, mine = rank ? second : first;
        const uint32_t cfull = bar0 + i * 2 * STAGES * 8, bfull = cfull + STAGES * 8;
        for (int s = 0; s < mine; ++s) {
            if (rank == 0) expect(bfull + 8u * s, DY_BYTES, one);
            expect(cfull + 8u * s, 1024, one);
            load_dy(base + s * (DY_BYTES / 2), &map_dy, leaders(bfull + 8u * s), 0, 0, one);
            load_bytes(base + CHECK_CODES + s * 1024, codes, 1024, cfull + 8u * s, one);
        }
        if (threadIdx.x == 0) store_cluster(in_cta(sent_word, rank), mine);
        __syncwarp();
        cluster_sync();
        if (threadIdx.x == 0 && !pair_landed(cfull, bfull, sent_word, DY_BYTES / 2, rank, err)) atomicCAS(err, 0, 98);
        __syncwarp();
        cluster_sync();
    }
    if (rank == 0) {
        warp_wait(alone, 0, err, 99);
        if (threadIdx.x == 0 && gave_up(alone)) tell_host(err, err_host);
    }
}

// The pieces of every tile that was cut, in token order: a block four rows of 256
// features, four features a thread.
constexpr int JOIN_ROWS = 4;
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Params P) {
    const int j = blockIdx.x, tile = P.full + j, len = P.stages - P.cut;
    const int first = helper_of(P, (int64_t)j * len), pieces = helper_of(P, (int64_t)(j + 1) * len - 1) - first + 1;
    const int fk = (threadIdx.x & 63) * 4, k0 = tile / P.tiles_n * TILE + fk;
    const int row = blockIdx.y * JOIN_ROWS + (threadIdx.x >> 6), n = tile % P.tiles_n * TILE + row;
    if (n >= P.N || k0 >= P.K) return;
    const float* at = P.part + (int64_t)row * TILE + fk;
    float4 sum = *reinterpret_cast<const float4*>(at + (int64_t)j * (TILE * TILE));
#pragma unroll 4
    for (int p = 0; p < pieces; ++p) {
        const float4 v = *reinterpret_cast<const float4*>(at + (int64_t)(P.rest + j + first + p) * (TILE * TILE));
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
    }
    __nv_bfloat16* out = P.dw + (int64_t)n * P.K + k0;
    if (P.K % 4 == 0) {
        *reinterpret_cast<uint2*>(out) = make_uint2(pack2(sum.x, sum.y, __nv_bfloat16()), pack2(sum.z, sum.w, __nv_bfloat16()));
    } else {
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
        for (int i = 0; i < 4; ++i)
            if (k0 + i < P.K) out[i] = __float2bfloat16_rn(v[i]);
    }
}

// ---------------------------------------------------------------- host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

bool make_map(CUtensorMap* m, const void* dy, int64_t M, int64_t N, int64_t ld) {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M}, strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {64, TOKENS}, steps[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(dy), dims, strides, box, steps,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

__device__ int g_err;      // first wait that ran out (0: none), per device
__device__ __align__(128) uint8_t g_check[8192];           // what the rehearsal copies
ErrorWords g_words(&g_err, "weight gradient's kernel", "concord_gemm_dw8_error");

// CTA pairs that are resident together, asked for once per device with the
// kernel's shared memory; 0: refused
constexpr int MAX_DEVICES = 64, MAX_PAIRS = 74;
int resident_pairs() {
    static std::atomic<int> known[MAX_DEVICES];
    static std::mutex mu;
    int d = 0;
    if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= MAX_DEVICES) return 0;
    int n = known[d].load();
    if (n > 0) return n;
    std::lock_guard<std::mutex> hold(mu);
    if ((n = known[d].load()) > 0) return n;
    if (cudaFuncSetAttribute(dw8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * MAX_PAIRS, 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = SMEM;
    if (cudaOccupancyMaxActiveClusters(&n, dw8_kernel, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = MAX_PAIRS;
    }
    n = std::min(n, MAX_PAIRS);
    known[d].store(n);
    return n;
}

// The pairs, and which tiles are cut: those beyond full rounds, unless cutting
// saves no more than 16 stages, about what storing and adding the pieces takes.
int share_out(Params& P, int64_t M, int64_t N, int64_t K, int resident) {
    P.M = M;
    P.N = (int)N;
    P.K = (int)K;
    P.tiles_n = (int)((N + TILE - 1) / TILE);
    P.stages = (int)((M + TOKENS - 1) / TOKENS);
    const int64_t tiles = (int64_t)P.tiles_n * ((K + TILE - 1) / TILE), total = tiles * P.stages;
    const int pairs = (int)std::min<int64_t>(resident, std::max<int64_t>(tiles, total / 4));
    P.rest = (int)(tiles % pairs);
    P.full = (int)(tiles - P.rest);
    P.cut = (int)(((int64_t)P.stages * P.rest + pairs - 1) / pairs);
    if (P.stages - P.cut <= 16) P.cut = P.stages;
    P.helpers = (int)std::min<int64_t>(pairs - P.rest, (int64_t)P.rest * (P.stages - P.cut));
    return pairs;
}
// slots of the workspace: each cut tile's first piece, and the steps along the line of ends
int64_t slots(const Params& P) { return P.helpers > 0 ? 2 * P.rest + P.helpers - 1 : 0; }

bool fits(int64_t M, int64_t N, int64_t K) { return K <= (1 << 20) && N <= (1 << 20) && M <= INT32_MAX - TOKENS; }

}  // namespace g8
}  // namespace concord

using namespace concord;

extern "C" size_t concord_gemm_dw8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || !g8::fits(M, N, K)) return 0;
    const int resident = g8::resident_pairs();
    g8::Params P{};
    g8::share_out(P, M, N, K, resident > 0 ? resident : g8::MAX_PAIRS);
    return (size_t)g8::slots(P) * g8::TILE * g8::TILE * sizeof(float);
}

extern "C" int concord_gemm_dw8(const uint16_t* dy, int64_t lddy, const void* saved, uint16_t* dw, int64_t M, int64_t N,
                                int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace g8;
    const char* name = "concord_gemm_dw8";
    if (M < 0 || N <= 0 || K <= 0 || lddy < N || N % 8 || lddy % 8)
        return fail(CONCORD_ESHAPE, std::string(name) + ": N and dy's row stride must be multiples of 8, extents positive");
    if (!fits(M, N, K) || lddy > ((int64_t)1 << 38))
        return fail(CONCORD_ETOOBIG, std::string(name) + ": more than 2^20 features or outputs, or 2^31 tokens");
    if (!dw) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    cudaStream_t st = as_stream(stream);
    if (M == 0) {
        cudaMemsetAsync(dw, 0, (size_t)N * K * 2, st);
        return check_launch(name);
    }
    if (!dy || !saved) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    if (!aligned(dy, 16) || !aligned(saved, 32) || !aligned(dw, 8)) return fail(CONCORD_EALIGN, std::string(name) + ": dy must be 16-byte aligned, saved 32, dw 8");
    const size_t need = concord_gemm_dw8_workspace_bytes(M, N, K);
    if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return fail(CONCORD_EWORKSPACE, std::string(name) + ": workspace too small, or not 16-byte aligned");
    if (int rc = bind_current_context(name)) return rc;
    Params P{};
    if (int rc = g_words.take(&P.err, &P.err_host, name)) return rc;
    CUtensorMap map;
    if (!make_map(&map, dy, M, N, lddy)) return fail(CONCORD_ELAUNCH, std::string(name) + ": TMA descriptor encoding failed");
    P.saved = static_cast<const uint8_t*>(saved);
    P.dw = reinterpret_cast<__nv_bfloat16*>(dw);
    P.part = static_cast<float*>(workspace);
    const int resident = resident_pairs();
    if (resident <= 0) return fail(CONCORD_ELAUNCH, std::string(name) + ": shared memory refused");
    const int pairs = share_out(P, M, N, K, resident);
    dw8_kernel<<<2 * pairs, THREADS, SMEM, st>>>(map, P);
    if (int rc = check_launch(name)) return rc;
    if (P.helpers > 0) {
        join_kernel<<<dim3((unsigned)P.rest, TILE / JOIN_ROWS), 256, 0, st>>>(P);
        return check_launch(name);
    }
    return CONCORD_OK;
}

extern "C" int concord_gemm_dw8_error(int32_t reset) { return g8::g_words.read(reset); }

extern "C" int32_t* concord_gemm_dw8_error_word(void) { return const_cast<int32_t*>(g8::g_words.host()); }

extern "C" int concord_gemm_dw8_wait_check(void* stream) {
    const char* name = "concord_gemm_dw8_wait_check";
    if (int rc = bind_current_context(name)) return rc;
    int *err, *err_host;
    if (int rc = g8::g_words.take(&err, &err_host, name)) return rc;
    void* src = nullptr;
    CUtensorMap map;
    if (cudaGetSymbolAddress(&src, g8::g_check) != cudaSuccess || !g8::make_map(&map, src, 64, 64, 64) ||
        cudaFuncSetAttribute(g8::wait_check_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)g8::CHECK_SMEM) != cudaSuccess)
        return fail(CONCORD_ELAUNCH, std::string(name) + ": device set-up failed");
    g8::wait_check_kernel<<<2, 32, g8::CHECK_SMEM, as_stream(stream)>>>(map, src, err, err_host);
    return check_launch(name);
}
