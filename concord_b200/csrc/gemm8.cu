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
// Warp roles: warp 0 loads (dy by TMA tiles, codes and scales by bulk copies),
// warp 1 of the leader issues the products, warps 4-11 convert, alternate stages
// of 64 tokens by the two groups of four, and afterwards store the
// accumulator (256 columns; the other 256 hold 8 stages of A).
//
// Work is the line of all (output tile, stage) in order; pair p takes an equal
// part of it.  Tiles cut by parts' ends leave fp32 pieces in the workspace, which a
// second kernel adds in token order: the same bits on every run of one device.
// Where the tiles themselves share out well, parts end at tiles' ends.
//
// Every wait is bounded (tc.cuh): where one runs out, loads and products stop,
// what is in flight lands (bounded again), the pair's remaining outputs become NaN and
// the device's error word is set (concord_gemm_dw8_error).
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "common.cuh"
#include "eight.cuh"
#include "tc.cuh"

namespace concord {
int bind_current_context(const char* name);

namespace g8 {

using namespace tc;

constexpr int THREADS = 384;
constexpr int FEATS = 128, OUTS = 128;            // of one CTA; a pair has twice both
constexpr int TOKENS = 64;                        // a stage
constexpr int STAGES = 8;
constexpr int DY_BYTES = TOKENS * OUTS * 2, CODE_BYTES = TOKENS * FEATS, SCALE_BYTES = 2 * FEATS;
constexpr int CODES = STAGES * DY_BYTES, SCALES = CODES + STAGES * CODE_BYTES;
constexpr int BARS = SCALES + STAGES * SCALE_BYTES;
constexpr int NBARS = 4 * STAGES + 3;
static_assert(BARS % BARRIERS == 0 && NBARS * 8 + 4 <= (int)BARRIERS - 4, "barriers, the tensor memory's address, the word");
constexpr size_t SMEM = BARS + BARRIERS + 1024;
constexpr int ACC = 256;                          // columns of the accumulator; stage s of A stands at ACC + 32 s
constexpr int TILE = 256;

struct Params {
    int64_t M;
    int N, K, tiles_n, stages;                    // stages of a tile
    int64_t quanta;                               // the line, in units of `unit` stages
    int unit;
    const int8_t* codes;
    const uint8_t* scales;
    __nv_bfloat16* dw;
    float* part;                                  // [pairs][2][256 outputs][256 features]
    int* err;
};

// the first stage of pair p's part
__host__ __device__ inline int64_t part_start(const Params& P, int64_t p, int64_t pairs) {
    return p * P.quanta / pairs * P.unit;
}

// one piece of a pair's part after another
struct Pieces {
    int64_t at, end;
    int first;                                    // 1: the part's first piece
    int tile, s0, s1;
    __device__ __forceinline__ Pieces(const Params& P) {
        const int64_t pairs = gridDim.x >> 1, p = blockIdx.x >> 1;
        at = part_start(P, p, pairs);
        end = part_start(P, p + 1, pairs);
        first = 2;
    }
    __device__ __forceinline__ bool next(const Params& P) {
        if (at >= end) return false;
        first = first == 2;
        tile = (int)(at / P.stages);
        s0 = (int)(at % P.stages);
        s1 = (int)min((int64_t)P.stages, s0 + (end - at));
        at += s1 - s0;
        return true;
    }
    __device__ __forceinline__ bool whole(const Params& P) const { return s0 == 0 && s1 == P.stages; }
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// this address in the leader's shared memory
__device__ __forceinline__ uint32_t leaders(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leaders(bar)) : "memory");
}
// a tile {64 outputs, 64 tokens} of dy into this CTA, counted on the leader's barrier
__device__ __forceinline__ void load_dy(uint32_t dst, const CUtensorMap* map, uint32_t bar, int n, int t) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(n), "r"(t)
        : "memory");
}
__device__ __forceinline__ void load_bytes(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
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

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    dw8_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ Params P) {
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + BARS);
    uint32_t* slot = reinterpret_cast<uint32_t*>(bars + NBARS);
    const uint32_t base = smem_u32(smem), bar0 = smem_u32(bars);
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
        if (lane == 0) {
            Pieces pc(P);
            int s = 0, sent = 0;
            uint32_t ph = 0;
            bool ok = true;
            const int64_t blocks = eight::blocks(P.M);
            while (ok && pc.next(P)) {
                const int k0 = pc.tile / P.tiles_n * TILE + (int)rank * FEATS, n0 = pc.tile % P.tiles_n * TILE + (int)rank * OUTS;
                const int feats = max(0, min(FEATS, P.K - k0)), padded = max(0, min(FEATS, (int)eight::scale_row(P.K) - k0));
                for (int i = pc.s0; i < pc.s1; ++i) {
                    if (!(ok = mbar_wait(empty(s), ph ^ 1, P.err, 1))) break;
                    if (rank == 0) mbar_expect(bfull(s), 2 * DY_BYTES);
                    const uint32_t lb = leaders(bfull(s)), dy = base + s * DY_BYTES;
                    load_dy(dy, &map_dy, lb, n0, i * TOKENS);
                    load_dy(dy + DY_BYTES / 2, &map_dy, lb, n0 + 64, i * TOKENS);
                    const int64_t b0 = 2 * (int64_t)i;
                    const int nb = b0 + 1 < blocks ? 2 : 1;          // blocks of 32 tokens that there are
                    mbar_expect(cfull(s), nb * (2 * feats * 16 + padded));
                    if (feats > 0) {
                        const uint32_t c = base + CODES + s * CODE_BYTES, sc = base + SCALES + s * SCALE_BYTES;
                        for (int j = 0; j < 2 * nb; ++j)
                            load_bytes(c + j * FEATS * 16, P.codes + ((2 * b0 + j) * P.K + k0) * 16, feats * 16, cfull(s));
                        for (int j = 0; j < nb; ++j)
                            load_bytes(sc + j * FEATS, P.scales + (b0 + j) * eight::scale_row(P.K) + k0, padded, cfull(s));
                    }
                    ++sent;
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
            if (!ok) {
                ring_landed(cfull(0), STAGES, sent, P.err);
                if (rank == 0) ring_landed(bfull(0), STAGES, sent, P.err);
            }
        }
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
            if (!ok) {
                commit_pair(drained, one);
                Patience patience;
                while (!__all_sync(0xffffffffu, mbar_try(drained, 0)) && !__any_sync(0xffffffffu, patience.over(P.err))) {}
            }
        }
    } else if (warp >= 4) {
        const int half = (warp - 4) >> 2, q = warp & 3;       // stages of this parity; lanes of the tensor memory
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        Pieces pc(P);
        int s = 0, parity = 0;
        uint32_t ph = 0, turn = 0;
        bool ok = true;
        const int64_t blocks = eight::blocks(P.M);
        while (pc.next(P)) {
            for (int i = pc.s0; ok && i < pc.s1; ++i) {
                if (parity == half) {
                    if (!(ok = warp_wait(cfull(s), ph, P.err, 5))) break;
                    fence_after();
                    const uint32_t at = base + CODES + s * CODE_BYTES + (q * 32 + lane) * 16;
                    const uint8_t* sc = smem + SCALES + s * SCALE_BYTES + q * 32 + lane;
                    const bool both = 2 * (int64_t)i + 1 < blocks;
                    uint32_t r[32];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 c = lds16(at + j * FEATS * 16);
                        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
                        const uint32_t scale2 = sc[(j >> 1) * FEATS] * 0x00800080u;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t x0 = two(w[k], 0x4140, scale2), x1 = two(w[k], 0x4342, scale2);
                            r[j * 8 + 2 * k] = j < 2 || both ? x0 : 0u;
                            r[j * 8 + 2 * k + 1] = j < 2 || both ? x1 : 0u;
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
            float* part = P.part + ((int64_t)(blockIdx.x >> 1) * 2 + !pc.first) * (TILE * TILE) + half * 128 * TILE + f0;
            const bool whole = pc.whole(P);
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
    cluster_sync();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512));
    }
}

// The pieces of every tile that was cut, in token order: a block a row of 256 features.
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Params P, int pairs) {
    const int tile = blockIdx.x, row = blockIdx.y;
    const int64_t t0 = (int64_t)tile * P.stages, t1 = t0 + P.stages;
    // the pair whose part holds stage t0
    int64_t lo = 0, hi = pairs - 1;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) / 2;
        if (part_start(P, mid, pairs) <= t0) lo = mid;
        else hi = mid - 1;
    }
    if (part_start(P, lo + 1, pairs) >= t1) return;              // whole
    const int n = tile % P.tiles_n * TILE + row, k = tile / P.tiles_n * TILE + threadIdx.x;
    if (n >= P.N || k >= P.K) return;
    float sum = 0.f;
    for (int64_t p = lo; p < pairs; ++p) {
        const int64_t a = part_start(P, p, pairs), b = part_start(P, p + 1, pairs);
        if (a >= t1) break;
        if (a == b) continue;
        sum += P.part[(p * 2 + (a < t0)) * (TILE * TILE) + row * TILE + threadIdx.x];
    }
    P.dw[(int64_t)n * P.K + k] = __float2bfloat16_rn(sum);
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

__device__ int g_err;
int* error_word() {
    int* p = nullptr;
    return cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_err) == cudaSuccess ? p : nullptr;
}

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

// Tiles go whole to pairs where that costs at most a tenth more stages than equal parts do.
void share_out(Params& P, int64_t tiles, int pairs, int* used) {
    const int64_t total = tiles * P.stages, rounds = (tiles + pairs - 1) / pairs;
    const bool whole = rounds * P.stages * pairs <= total + total / 10 + 8 * pairs;
    P.unit = whole ? P.stages : 1;
    P.quanta = whole ? tiles : total;
    *used = (int)std::min<int64_t>(pairs, whole ? tiles : std::max<int64_t>(tiles, total / 4));
}

}  // namespace g8
}  // namespace concord

using namespace concord;

extern "C" size_t concord_gemm_dw8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return (size_t)g8::MAX_PAIRS * 2 * g8::TILE * g8::TILE * sizeof(float);
}

extern "C" int concord_gemm_dw8(const uint16_t* dy, int64_t lddy, const void* saved, uint16_t* dw, int64_t M, int64_t N,
                                int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace g8;
    const char* name = "concord_gemm_dw8";
    if (M < 0 || N <= 0 || K <= 0 || lddy < N || N % 8 || lddy % 8)
        return fail(CONCORD_ESHAPE, std::string(name) + ": N and dy's row stride must be multiples of 8, extents positive");
    if (K > (1 << 20) || N > (1 << 20) || M > INT32_MAX - TOKENS || lddy > ((int64_t)1 << 38))
        return fail(CONCORD_ETOOBIG, std::string(name) + ": more than 2^20 features or outputs, or 2^31 tokens");
    if (!dw) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    cudaStream_t st = as_stream(stream);
    if (M == 0) {
        cudaMemsetAsync(dw, 0, (size_t)N * K * 2, st);
        return check_launch(name);
    }
    if (!dy || !saved) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    if (!aligned(dy, 16) || !aligned(saved, 16)) return fail(CONCORD_EALIGN, std::string(name) + ": operands must be 16-byte aligned");
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < concord_gemm_dw8_workspace_bytes(M, N, K))
        return fail(CONCORD_EWORKSPACE, std::string(name) + ": workspace too small, or not 16-byte aligned");
    if (int rc = bind_current_context(name)) return rc;
    CUtensorMap map;
    if (!make_map(&map, dy, M, N, lddy)) return fail(CONCORD_ELAUNCH, std::string(name) + ": TMA descriptor encoding failed");
    Params P{};
    P.M = M;
    P.N = (int)N;
    P.K = (int)K;
    P.tiles_n = (int)((N + TILE - 1) / TILE);
    P.stages = (int)((M + TOKENS - 1) / TOKENS);
    P.codes = static_cast<const int8_t*>(saved);
    P.scales = static_cast<const uint8_t*>(saved) + eight::code_bytes(M, K);
    P.dw = reinterpret_cast<__nv_bfloat16*>(dw);
    P.part = static_cast<float*>(workspace);
    P.err = error_word();
    const int resident = resident_pairs();
    if (!P.err || resident <= 0) return fail(CONCORD_ELAUNCH, std::string(name) + ": no error word, or shared memory refused");
    const int64_t tiles = (int64_t)P.tiles_n * ((K + TILE - 1) / TILE);
    int pairs = 1;
    share_out(P, tiles, resident, &pairs);
    dw8_kernel<<<2 * pairs, THREADS, SMEM, st>>>(map, P);
    if (int rc = check_launch(name)) return rc;
    if (P.unit == 1) {
        join_kernel<<<dim3((unsigned)tiles, TILE), 256, 0, st>>>(P, pairs);
        return check_launch(name);
    }
    return CONCORD_OK;
}

extern "C" int concord_gemm_dw8_error(int32_t reset) {
    int* err = g8::error_word();
    if (!err) return -1;
    int v = 0;
    cudaMemcpy(&v, err, sizeof(int), cudaMemcpyDeviceToHost);
    if (reset) cudaMemset(err, 0, sizeof(int));
    return v;
}
