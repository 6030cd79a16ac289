// norm.cu — layer norm over the last dimension, forward and backward.
//
//   y  = (x - mean) rstd w + b,           rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)),  g = dy w, xh = (x - mean) rstd
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Bound by memory: the forward reads x and writes y once, the backward reads
// x and dy and writes dx once.  A row stays in the registers of the threads
// that own it (16 elements each, 32 in the forward above 512 columns), so the
// variance is the mean of squared deviations from the finished mean and nothing
// is read twice.  The grid is one wave of resident blocks that walk the rows;
// each thread keeps its columns' weight and bias, and in the
// backward its columns' sums of dy xh and dy, from row to row.  Rows whose
// pieces are 16 bytes come through a ring in shared memory, three rows ahead
// of their use: a thread copies only what it reads itself, so the ring needs no
// barrier, and the loads in flight do not depend on the registers.  The blocks'
// sums are added in block order by a second kernel: no atomics, so the
// gradients are the same bits on every run of one device.
#include <atomic>

#include "common.cuh"
#include "vec.cuh"

namespace concord {
namespace norm {

constexpr int PER = 16;             // elements of a row that one thread holds
constexpr int MAX_DIM = 1024 * PER;

// sums of (a, b) over the `tpr` threads of this row; every thread of the block calls it
template <int NB>
__device__ __forceinline__ void row_sum(float& a, float& b, int tpr, float2* red, int& turn) {
    a = warp_sum(a);
    if (NB == 2) b = warp_sum(b);
    if (tpr == 32) return;
    float2* r = red + (turn ? 32 : 0);          // two buffers: one barrier per sum
    turn ^= 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = tpr >> 5;
    if (lane == 0) r[warp] = make_float2(a, b);
    __syncthreads();
    const int w0 = warp & ~(nw - 1);
    if (nw <= 4) {
        float2 s = r[w0];
        a = s.x;
        b = s.y;
        for (int i = 1; i < nw; ++i) {
            s = r[w0 + i];
            a += s.x;
            if (NB == 2) b += s.y;
        }
        return;
    }
    const float2 s = lane < nw ? r[w0 + lane] : make_float2(0.f, 0.f);
    a = warp_sum(s.x);
    if (NB == 2) b = warp_sum(s.y);
}

// A thread's elements of a row, in pairs (two columns an instruction): element
// i * VEC + j is column (i * tpr + t) * VEC + j.
template <int PER> struct PairsOf {
    uint64_t v[PER / 2];
    __device__ __forceinline__ void fill(float a) {
#pragma unroll
        for (int e = 0; e < PER / 2; ++e) v[e] = f2(a, a);
    }
    __device__ __forceinline__ float sum() const {
        uint64_t s = v[0];
        float a, b;
#pragma unroll
        for (int e = 1; e < PER / 2; ++e) s = add2(s, v[e]);
        unf2(s, a, b);
        return a + b;
    }
    __device__ __forceinline__ float get(int e) const {
        float a, b;
        unf2(v[e / 2], a, b);
        return e & 1 ? b : a;
    }
    __device__ __forceinline__ void set(int e, float x) {
        float a, b;
        unf2(v[e / 2], a, b);
        v[e / 2] = e & 1 ? f2(a, x) : f2(x, b);
    }
    // VEC columns from / to memory as piece i
    template <int VEC, typename T> __device__ __forceinline__ void load(int i, const T* p) {
        if constexpr (VEC == 1) set(i, to_f32(*p));
        else {
            float x[8];
            load_vec<8>(p, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i * 4 + j] = f2(x[2 * j], x[2 * j + 1]);
        }
    }
    template <int VEC, typename T> __device__ __forceinline__ void store(int i, T* p) const {
        if constexpr (VEC == 1) *p = from_f32<T>(get(i));
        else {
            float x[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) unf2(v[i * 4 + j], x[2 * j], x[2 * j + 1]);
            store_vec<8>(p, x);
        }
    }
    template <int VEC> __device__ __forceinline__ void clear(int i) {
        if constexpr (VEC == 1) set(i, 0.f);
        else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i * 4 + j] = 0;
        }
    }
};

using Pairs = PairsOf<PER>;

// rows of a ring: three or two on their way (1024 threads of 4-byte pieces fill 192 KB with three stages)
template <typename TX, typename TY> constexpr int ring_stages() { return sizeof(TX) + sizeof(TY) > 4 ? 3 : 4; }

// A thread's pieces of rows, STAGES deep: [stage][piece][thread] of 16 bytes.
// Addresses are 32-bit offsets and pointers that move by a constant a row:
// computed anew for every piece they were half of all instructions issued.
// Piece groups (8 elements) of a thread are `gap` bytes apart in memory.
template <typename T, int STAGES, int EL = PER> struct Ring {
    static constexpr int HALF = (int)sizeof(T) / 2, GROUPS = EL / 8;      // HALF: pieces of 8 elements
    static constexpr int BYTES = STAGES * GROUPS * HALF * 16;             // per thread
    const char* src;         // this thread's part of the next row to fetch
    int64_t row_bytes;       // from one of its rows to the next
    uint32_t base, piece, stage_bytes, put, get;
    __device__ __forceinline__ Ring(uint32_t smem, const T* first, int64_t stride)
        : src(reinterpret_cast<const char*>(first)), row_bytes(stride * (int64_t)sizeof(T)),
          base(smem + threadIdx.x * 16), piece(blockDim.x * 16), stage_bytes(GROUPS * HALF * piece), put(0), get(0) {}
    __device__ __forceinline__ void fetch(bool row, int gap, int here, int D, int cols) {
        if (row) {
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                if (here + i * cols < D) {
#pragma unroll
                    for (int h = 0; h < HALF; ++h)
                        copy16(base + put + (i * HALF + h) * piece, src + i * gap + h * 16);
                }
            }
        }
        copy_commit();
        src += row_bytes;
        put += stage_bytes;
        if (put == STAGES * stage_bytes) put = 0;
    }
    __device__ __forceinline__ void read(int i, PairsOf<EL>& p) const {
        float x[8];
#pragma unroll
        for (int h = 0; h < HALF; ++h)
            Pack16<T>::unpack(read16(base + get + (i * HALF + h) * piece), x + h * Pack16<T>::N);
#pragma unroll
        for (int j = 0; j < 4; ++j) p.v[i * 4 + j] = f2(x[2 * j], x[2 * j + 1]);
    }
    __device__ __forceinline__ void next() {
        get += stage_bytes;
        if (get == STAGES * stage_bytes) get = 0;
    }
};

template <typename TX> constexpr int fwd_stages() { return sizeof(TX) == 4 ? 3 : 4; }

// EL elements a thread, whose weight and bias stay in its registers (VEC 8).
// Measured for 65533 x 2048 bf16 (82 us of bytes): 16 elements, four warps a
// row, 135 us (25 instructions an element, half of them the two sums); 64, one
// warp a row, weight and bias from the L1, 125 us (90 without them: the L1
// gives 128 bytes a cycle, they are 8 an element); 32 in registers, two warps a
// row, 105 us (5.1 TB/s).  ONE: a row is one warp's (the columns' distances are constants).
template <typename TX, typename TY, int VEC, int EL, bool ONE>
__global__ void __launch_bounds__(VEC == 1 ? 1024 : 512)
    fwd_kernel(const TX* __restrict__ x, int64_t ldx, const float* __restrict__ w, const float* __restrict__ b,
               TY* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, int64_t N, int D, float eps,
               int threads_per_row) {
    constexpr int NV = EL / VEC, STAGES = fwd_stages<TX>();
    extern __shared__ __align__(16) uint8_t dyn_f[];
    __shared__ float2 red[64];
    int turn = 0;
    const int tpr = ONE ? 32 : threads_per_row;
    const int t = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const int64_t step = (int64_t)gridDim.x * groups;
    const float inv = 1.0f / (float)D;
    const bool whole = D == tpr * EL;            // every piece of every thread is there
    int64_t row = (int64_t)blockIdx.x * groups + group;
    const int cols = tpr * VEC, here = t * VEC;
    Ring<TX, STAGES, EL> ring(static_cast<uint32_t>(__cvta_generic_to_shared(dyn_f)), x + row * ldx + here,
                              step * ldx);
    TY* dst = y + row * D + here;
    PairsOf<EL> wv, bv;
    if constexpr (VEC == 8) {
        wv.fill(1.0f);
        bv.fill(0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (here + i * cols < D) {
                if (w) wv.template load<VEC>(i, w + here + i * cols);
                if (b) bv.template load<VEC>(i, b + here + i * cols);
            }
        }
#pragma unroll
        for (int k = 0; k < STAGES - 1; ++k)
            ring.fetch(row + k * step < N, cols * (int)sizeof(TX), here, D, cols);
    }
    for (; row - group < N; row += step) {
        const bool live = row < N;
        PairsOf<EL> v;
        if constexpr (VEC == 8) {
            ring.fetch(row + (STAGES - 1) * step < N, cols * (int)sizeof(TX), here, D, cols);
            copy_wait<STAGES - 1>();
        }
        if (!whole || !live) v.fill(0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (live && here + i * cols < D) {
                if constexpr (VEC == 8) ring.read(i, v);
                else v.template load<VEC>(i, x + row * ldx + here + i * cols);
            }
        }
        ring.next();
        float sum = v.sum(), none = 0.f;
        row_sum<1>(sum, none, tpr, red, turn);
        const float mu = sum * inv;
        const uint64_t mu2 = f2(-mu, -mu);
#pragma unroll
        for (int e = 0; e < EL / 2; ++e) v.v[e] = add2(v.v[e], mu2);
        if (!whole) {                             // deviations of columns that are not there weigh nothing
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (here + i * cols >= D) v.template clear<VEC>(i);
        }
        uint64_t sq2 = 0;
#pragma unroll
        for (int e = 0; e < EL / 2; ++e) sq2 = fma2(v.v[e], v.v[e], sq2);
        float sq, sq_b;
        unf2(sq2, sq, sq_b);
        sq += sq_b;
        row_sum<1>(sq, none, tpr, red, turn);
        const float rs = rsqrtf(sq * inv + eps);
        const uint64_t rs2 = f2(rs, rs);
#pragma unroll
        for (int e = 0; e < EL / 2; ++e) {
            v.v[e] = mul2(v.v[e], rs2);
            if constexpr (VEC == 8) v.v[e] = fma2(v.v[e], wv.v[e], bv.v[e]);
        }
        if (live) {
            if (mean && t == 0) {
                mean[row] = mu;
                rstd[row] = rs;
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = here + i * cols;
                if (c < D) {
                    if constexpr (VEC == 1) v.set(i, fmaf(v.get(i), w ? w[c] : 1.0f, b ? b[c] : 0.0f));
                    v.template store<VEC>(i, dst + i * cols);
                }
            }
        }
        dst += step * D;
    }
}

// 65533 x 2048 bf16: 152 us, 5.3 TB/s of x, dy and dx (82 % of a plain copy's
// rate); issue slots 59 %.
// dx, and this block's column sums to part[block][0: dy xh, 1: dy][D].  WIDE
// (above 8192 columns, 1024 threads of at most 64 registers): the column sums
// live in the thread's own shared-memory slots instead of its registers.
template <typename TX, typename TY, int VEC, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 1024 : 512)
    bwd_kernel(const TX* __restrict__ x, int64_t ldx, const TY* __restrict__ dy, int64_t lddy,
               const float* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
               TX* __restrict__ dx, float* __restrict__ part, int64_t N, int D, int tpr) {
    constexpr int NV = PER / VEC, STAGES = ring_stages<TX, TY>();
    // WIDE: 2 * PER * 1024 sums; else the rings, whose place the groups' sums take at the end
    extern __shared__ __align__(16) uint8_t dyn_b[];
    float* dyn = reinterpret_cast<float*>(dyn_b);
    __shared__ float2 red[64];
    int turn = 0;
    const int t = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const int64_t step = (int64_t)gridDim.x * groups;
    const float inv = 1.0f / (float)D;
    const bool whole = D == tpr * PER;
    constexpr bool RING = VEC == 8 && !WIDE;     // WIDE has no room beside its sums
    int64_t row = (int64_t)blockIdx.x * groups + group;
    const int cols = tpr * VEC, here = t * VEC;
    const uint32_t smem = static_cast<uint32_t>(__cvta_generic_to_shared(dyn_b));
    Ring<TX, STAGES> xr(smem, x + row * ldx + here, step * ldx);
    Ring<TY, STAGES> yr(smem + Ring<TX, STAGES>::BYTES * blockDim.x, dy + row * lddy + here, step * lddy);
    TX* dst = dx + row * D + here;
    // (two groups of copies a row)
    auto fetch = [&](bool there) {
        xr.fetch(there, cols * (int)sizeof(TX), here, D, cols);
        yr.fetch(there, cols * (int)sizeof(TY), here, D, cols);
    };
    if constexpr (RING) {
#pragma unroll
        for (int k = 0; k < STAGES - 1; ++k) fetch(row + k * step < N);
    }
    Pairs aw, ab;                                 // column sums of dy xh and dy (not WIDE)
    if constexpr (WIDE) {
#pragma unroll
        for (int e = 0; e < 2 * PER; ++e) dyn[e * 1024 + threadIdx.x] = 0.f;
    } else {
        aw.fill(0.f);
        ab.fill(0.f);
    }
    Pairs wv;
    wv.fill(1.0f);
    if (!WIDE && w) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + t) * VEC;
            if (c < D) wv.template load<VEC>(i, w + c);
        }
    }
    float mu = 0.f, rs = 0.f;                     // of this row, fetched a row ahead
    if (row < N) { mu = mean[row]; rs = rstd[row]; }
    for (; row - group < N; row += step) {
        const bool live = row < N;
        float next_mu = 0.f, next_rs = 0.f;
        if (row + step < N) { next_mu = mean[row + step]; next_rs = rstd[row + step]; }
        Pairs xh, g;
        if constexpr (RING) {
            fetch(row + (STAGES - 1) * step < N);
            copy_wait<2 * (STAGES - 1)>();
        }
        if (!whole || !live) {                    // g = 0: what is not there weighs nothing
            xh.fill(0.f);
            g.fill(0.f);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = here + i * cols;
            if (live && c < D) {
                if constexpr (RING) {
                    xr.read(i, xh);
                    yr.read(i, g);
                } else {
                    xh.template load<VEC>(i, x + row * ldx + c);
                    g.template load<VEC>(i, dy + row * lddy + c);
                }
            }
        }
        xr.next();
        yr.next();
        // (x - mean first, as in the forward: the rounding of mean * rstd would
        // give rows far off centre a deviation that they do not have)
        const uint64_t rs2 = f2(rs, rs), mu2 = f2(-mu, -mu);
#pragma unroll
        for (int e = 0; e < PER / 2; ++e) {
            xh.v[e] = mul2(add2(xh.v[e], mu2), rs2);
            if constexpr (WIDE) {
                float ga, gb, xa, xb;
                unf2(g.v[e], ga, gb);
                unf2(xh.v[e], xa, xb);
                dyn[(2 * e) * 1024 + threadIdx.x] += ga * xa;
                dyn[(2 * e + 1) * 1024 + threadIdx.x] += gb * xb;
                dyn[(PER + 2 * e) * 1024 + threadIdx.x] += ga;
                dyn[(PER + 2 * e + 1) * 1024 + threadIdx.x] += gb;
            } else {
                aw.v[e] = fma2(g.v[e], xh.v[e], aw.v[e]);
                ab.v[e] = add2(g.v[e], ab.v[e]);
            }
        }
        if (WIDE && w) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * tpr + t) * VEC;
                if (c < D) wv.template load<VEC>(i, w + c);
            }
        }
        uint64_t gx = 0;
#pragma unroll
        for (int e = 0; e < PER / 2; ++e) {
            g.v[e] = mul2(g.v[e], wv.v[e]);
            gx = fma2(g.v[e], xh.v[e], gx);
        }
        float s1 = g.sum(), s2, s2_b;
        unf2(gx, s2, s2_b);
        s2 += s2_b;
        row_sum<2>(s1, s2, tpr, red, turn);
        // dx = rs g - rs mean(g) - rs mean(g xh) xh
        const uint64_t c1 = f2(-rs * (s1 * inv), -rs * (s1 * inv)), c2 = f2(-rs * (s2 * inv), -rs * (s2 * inv));
#pragma unroll
        for (int e = 0; e < PER / 2; ++e) g.v[e] = fma2(xh.v[e], c2, fma2(g.v[e], rs2, c1));
        if (live) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (here + i * cols < D) g.template store<VEC>(i, dst + i * cols);
            }
        }
        dst += step * D;
        mu = next_mu;
        rs = next_rs;
    }
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * 2 * D;
    if constexpr (WIDE) {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int c = ((e / VEC) * tpr + t) * VEC + e % VEC;
            if (c < D) { out[c] = dyn[e * 1024 + threadIdx.x]; out[D + c] = dyn[(PER + e) * 1024 + threadIdx.x]; }
        }
    } else {
        // the groups' sums meet in shared memory and are added in group order
        if constexpr (RING) {
            copy_wait<0>();
            __syncthreads();
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int c = ((e / VEC) * tpr + t) * VEC + e % VEC;
            if (c < D) { dyn[group * 2 * D + c] = aw.get(e); dyn[group * 2 * D + D + c] = ab.get(e); }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * D; c += blockDim.x) {
            float s = dyn[c];
            for (int k = 1; k < groups; ++k) s += dyn[k * 2 * D + c];
            out[c] = s;
        }
    }
}

// dw / db from the blocks' sums, in a fixed order: 8 columns x 32 strides per block
__global__ void __launch_bounds__(256) sum_kernel(const float* __restrict__ part, int blocks, int D,
                                                  float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float red[32][9];
    const int cx = threadIdx.x & 7, ry = threadIdx.x >> 3;
    const int c = blockIdx.x * 8 + cx;
    float s = 0.f;
    if (c < 2 * D) {
#pragma unroll 4
        for (int k = ry; k < blocks; k += 32) s += part[(int64_t)k * 2 * D + c];
    }
    red[ry][cx] = s;
    __syncthreads();
    if (ry == 0 && c < 2 * D) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += red[k][cx];
        float* out = c < D ? dw : db;
        if (out) out[c < D ? c : c - D] = s;
    }
}

int threads_per_row(int64_t D) {
    int t = 32;
    while (t * PER < D) t *= 2;
    return t;
}

int sm_count() {
    int d = 0, n = 148;
    if (cudaGetDevice(&d) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d);
    return n;
}

// more than 48 KB of shared memory a block, 1 KB of it static here, has to be asked for (per device; asking again changes nothing)
template <typename K> int allow_smem(K k, size_t smem, const char* name) {
    if (smem <= 47 * 1024) return CONCORD_OK;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    return e == cudaSuccess ? CONCORD_OK : fail(CONCORD_ELAUNCH, std::string(name) + ": " + cudaGetErrorString(e));
}

// blocks of the backward: one wave of 512 threads per SM (1024 where a row takes 1024)
int bwd_blocks(int64_t N, int64_t D, int* threads) {
    const int tpr = threads_per_row(D);
    *threads = tpr > 256 ? tpr : 256;
    const int64_t groups = *threads / tpr, need = (N + groups - 1) / groups;
    const int64_t wave = (int64_t)sm_count() * (*threads >= 512 ? 1 : 512 / *threads);
    return (int)(need < wave ? need : wave);
}

template <typename TX, typename TY, int VEC, int EL>
int launch_fwd(const void* x, int64_t ldx, const float* w, const float* b, void* y, float* mean, float* rstd,
               int64_t N, int64_t D, float eps, cudaStream_t st) {
    int tpr = 32;
    while (tpr * EL < D) tpr *= 2;
    const int threads = VEC == 1 ? (tpr > 256 ? tpr : 256) : (tpr > 128 ? tpr : 128);
    const int64_t groups = threads / tpr, need = (N + groups - 1) / groups;
    auto k = tpr == 32 ? fwd_kernel<TX, TY, VEC, EL, true> : fwd_kernel<TX, TY, VEC, EL, false>;
    const size_t smem = VEC == 8 ? (size_t)Ring<TX, fwd_stages<TX>(), EL>::BYTES * threads : 0;
    if (int rc = allow_smem(k, smem, "concord_layer_norm_fwd")) return rc;
    // one wave of resident blocks (asked for once per form; the answer is the architecture's)
    static std::atomic<int> resident[8];
    std::atomic<int>& known = resident[__builtin_ctz(tpr) - 5];
    int per_sm = known.load();
    if (per_sm == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, threads, smem) != cudaSuccess || per_sm < 1)
            per_sm = 1;
        known.store(per_sm);
    }
    const int64_t wave = (int64_t)sm_count() * per_sm;
    k<<<(int)(need < wave ? need : wave), threads, smem, st>>>(static_cast<const TX*>(x), ldx, w, b,
                                                               static_cast<TY*>(y), mean, rstd, N, (int)D, eps, tpr);
    return check_launch("concord_layer_norm_fwd");
}

template <typename TX, typename TY>
int forward(const void* x, int64_t ldx, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t N,
            int64_t D, float eps, bool vec, cudaStream_t st) {
    if (!vec) return launch_fwd<TX, TY, 1, 16>(x, ldx, w, b, y, mean, rstd, N, D, eps, st);
    if (D <= 512) return launch_fwd<TX, TY, 8, 16>(x, ldx, w, b, y, mean, rstd, N, D, eps, st);
    return launch_fwd<TX, TY, 8, 32>(x, ldx, w, b, y, mean, rstd, N, D, eps, st);
}

template <typename TX, typename TY>
int backward(const void* x, int64_t ldx, const void* dy, int64_t lddy, const float* w, const float* mean,
             const float* rstd, void* dx, float* dw, float* db, int64_t N, int64_t D, bool vec, float* part,
             cudaStream_t st) {
    int threads = 0;
    const int grid = bwd_blocks(N, D, &threads), tpr = threads_per_row(D);
    const bool wide = tpr == 1024;
    const size_t sums = (size_t)(threads / tpr) * 2 * D * sizeof(float);
    constexpr int ST = ring_stages<TX, TY>();
    const size_t rings = vec ? (size_t)(Ring<TX, ST>::BYTES + Ring<TY, ST>::BYTES) * threads : 0;
    const size_t smem = wide ? 2 * PER * 1024 * sizeof(float) : sums > rings ? sums : rings;
    auto k = wide ? (vec ? bwd_kernel<TX, TY, 8, true> : bwd_kernel<TX, TY, 1, true>)
                  : (vec ? bwd_kernel<TX, TY, 8, false> : bwd_kernel<TX, TY, 1, false>);
    if (int rc = allow_smem(k, smem, "concord_layer_norm_bwd")) return rc;
    if (!dw && !db) part = nullptr;
    k<<<grid, threads, smem, st>>>(static_cast<const TX*>(x), ldx, static_cast<const TY*>(dy), lddy, w, mean, rstd,
                                   static_cast<TX*>(dx), part, N, (int)D, tpr);
    if (int rc = check_launch("concord_layer_norm_bwd")) return rc;
    if (part) {
        sum_kernel<<<(int)((2 * D + 7) / 8), 256, 0, st>>>(part, grid, (int)D, dw, db);
        return check_launch("concord_layer_norm_bwd");
    }
    return CONCORD_OK;
}

// calls f<TX, TY> for the two type codes
#define NORM_TYPES(tx, ty, F, ...)                                                              \
    switch ((tx) * 3 + (ty)) {                                                                  \
        case 0: return F<float, float>(__VA_ARGS__);                                            \
        case 1: return F<float, __nv_bfloat16>(__VA_ARGS__);                                    \
        case 2: return F<float, __half>(__VA_ARGS__);                                           \
        case 3: return F<__nv_bfloat16, float>(__VA_ARGS__);                                    \
        case 4: return F<__nv_bfloat16, __nv_bfloat16>(__VA_ARGS__);                            \
        case 5: return F<__nv_bfloat16, __half>(__VA_ARGS__);                                   \
        case 6: return F<__half, float>(__VA_ARGS__);                                           \
        case 7: return F<__half, __nv_bfloat16>(__VA_ARGS__);                                   \
        default: return F<__half, __half>(__VA_ARGS__);                                         \
    }

int check_shape(const char* name, int32_t tx, int32_t ty, int64_t N, int64_t D, int64_t ldx) {
    if (tx < 0 || tx > 2 || ty < 0 || ty > 2) return fail(CONCORD_EINVAL, std::string(name) + ": unknown element type");
    if (N < 0 || D <= 0 || ldx < D) return fail(CONCORD_ESHAPE, std::string(name) + ": bad extents or row stride");
    if (D > MAX_DIM) return fail(CONCORD_ETOOBIG, std::string(name) + ": more than 16384 columns");
    return CONCORD_OK;
}

size_t esize(int32_t t) { return t == 0 ? 4 : 2; }

}  // namespace norm
}  // namespace concord

using namespace concord;

extern "C" int concord_layer_norm_fwd(const void* x, int32_t x_type, int64_t ldx, const float* w, const float* b,
                                      void* y, int32_t y_type, float* mean, float* rstd, int64_t N, int64_t D,
                                      float eps, void* stream) {
    if (int rc = norm::check_shape("concord_layer_norm_fwd", x_type, y_type, N, D, ldx)) return rc;
    if (N == 0) return CONCORD_OK;
    if (!x || !y || !mean != !rstd) return fail(CONCORD_EINVAL, "concord_layer_norm_fwd: null pointer");
    const bool vec = D % 8 == 0 && ldx * norm::esize(x_type) % 16 == 0 && aligned(x, 16) && aligned(y, 16) &&
                     aligned(w, 16) && aligned(b, 16);
    NORM_TYPES(x_type, y_type, norm::forward, x, ldx, w, b, y, mean, rstd, N, D, eps, vec, as_stream(stream))
}

extern "C" size_t concord_layer_norm_bwd_workspace_bytes(int64_t N, int64_t D) {
    if (N <= 0 || D <= 0 || D > norm::MAX_DIM) return 0;
    int threads = 0;
    return (size_t)norm::bwd_blocks(N, D, &threads) * 2 * D * sizeof(float);
}

extern "C" int concord_layer_norm_bwd(const void* x, int32_t x_type, int64_t ldx, const void* dy, int32_t dy_type,
                                      int64_t lddy, const float* w, const float* mean, const float* rstd, void* dx,
                                      float* dw, float* db, int64_t N, int64_t D, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    if (int rc = norm::check_shape("concord_layer_norm_bwd", x_type, dy_type, N, D, ldx < lddy ? ldx : lddy)) return rc;
    cudaStream_t st = as_stream(stream);
    if (N == 0) {
        if (dw) cudaMemsetAsync(dw, 0, D * sizeof(float), st);
        if (db) cudaMemsetAsync(db, 0, D * sizeof(float), st);
        return check_launch("concord_layer_norm_bwd");
    }
    if (!x || !dy || !mean || !rstd || !dx) return fail(CONCORD_EINVAL, "concord_layer_norm_bwd: null pointer");
    if ((dw || db) && (!workspace || workspace_bytes < concord_layer_norm_bwd_workspace_bytes(N, D)))
        return fail(CONCORD_EWORKSPACE, "concord_layer_norm_bwd: workspace too small");
    const bool vec = D % 8 == 0 && ldx * norm::esize(x_type) % 16 == 0 && lddy * norm::esize(dy_type) % 16 == 0 &&
                     aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16) && aligned(w, 16);
    NORM_TYPES(x_type, dy_type, norm::backward, x, ldx, dy, lddy, w, mean, rstd, dx, dw, db, N, D, vec,
               static_cast<float*>(workspace), st)
}
