// eight.cu — activations kept in 8 bits for the backward pass (the format: eight.cuh):
// saved, read back, and the gated unit whose gradient is computed from them.
//
//   h = act(g) u,  act(g) = g sigmoid(g) or g Phi(g)
//   dg = dh u act'(g),  du = dh act(g),  g and u as kept (8 bits, or the inputs themselves)
//   silu'(g) = q + g q (1 - q), q = sigmoid(g);  gelu'(g) = Phi(g) + g phi(g)
//
// Bound by memory (save8 of 16384 x 5504 bf16: 42 us, 6.5 TB/s; the unit on it in 8 bits:
// forward 123 us, backward 121, 5.9 and 6.0 TB/s).  A thread owns a block's 32 tokens of a few neighbouring
// features (8 bytes of each row): the largest magnitude needs no exchange, all its
// loads are on their way at once, and what it writes are whole pieces of 16 codes.
#include "common.cuh"
#include "eight.cuh"

namespace concord {
namespace eight {

constexpr int THREADS = 128;
// Bytes of a row that a thread of each kernel takes: whole pieces of the codes' 32
// bytes want two features at least; the unit's forward holds two tiles and keeps more warps on
// an SM with two features of 16 bits (16384 x 5504 bf16: 123 us, with four 152), the
// others do better with four (save 17, with two the same; the unit's backward 121, with two 132).
// (a row of the elementwise kernels by single elements: so many tokens a thread,
// to keep enough on its way; 16384 x 5503 bf16: 200 and 247 us, with one 322 and 374)
constexpr int TALL = 4;
constexpr int SAVE_BYTES = 8, FWD_BYTES = 4, BWD_BYTES = 8;


template <int EL> __device__ __forceinline__ void load_codes(const uint8_t* p, uint4* c) {
    if constexpr (EL == 1) c[0] = *reinterpret_cast<const uint4*>(p);
    else {
#pragma unroll
        for (int j = 0; j < EL; j += 2) load32(p + j * 16, c[j], c[j + 1]);
    }
}

template <typename T, int EL>
__global__ void __launch_bounds__(THREADS)
    save_kernel(const T* x, int64_t ldx, uint8_t* saved, int64_t M, int K) {
    const int k = (blockIdx.y * blockDim.x + threadIdx.x) * EL;
    const int64_t tb = blockIdx.x, t0 = tb * BLOCK;
    if (k >= K) return;
    Tile<T, EL> A;
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) A.load_row(i, x + (t0 + i) * ldx + k, t0 + i < M);
    A.save(saved, tb, K, k);
}

// a thread: 16 tokens of EL features
template <typename T, int EL>
__global__ void __launch_bounds__(THREADS)
    dense_kernel(const uint8_t* saved, T* out, int64_t ldo, int64_t M, int K) {
    const int k = (blockIdx.y * blockDim.x + threadIdx.x) * EL;
    const int64_t tb = blockIdx.x, t0 = tb * 16;
    if (k >= K || t0 >= M) return;
    const Place at(tb >> 2, k, K);
    uint4 c[EL];
    float scale[EL];
    load_codes<EL>(saved + at.codes(tb & 3), c);
#pragma unroll
    for (int j = 0; j < EL; ++j) scale[j] = scale_of(saved[at.scale((tb >> 1) & 1) + j]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (t0 + i >= M) break;
        T v[EL];
#pragma unroll
        for (int j = 0; j < EL; ++j) {
            const uint32_t w = (i < 4 ? c[j].x : i < 8 ? c[j].y : i < 12 ? c[j].z : c[j].w) ^ 0x80808080u;
            v[j] = from_f32<T>(value(w, i & 3, scale[j]));
        }
        T* p = out + (t0 + i) * ldo + k;
        if constexpr (EL * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(v);
        else if constexpr (EL * sizeof(T) == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v);
        else if constexpr (EL * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<uint32_t*>(v);
        else p[0] = v[0];
    }
}

// ---------------------------------------------------------------- the gated unit
constexpr int SILU = 0, GELU = 1;

// The functions for results of 16 bits, whose roundings are 2^-11 and 2^-8: the hardware's exponential and reciprocal, and
// for gelu Hastings' rational form of Phi.  Results of fp32 (EXACT) take expf, erfcf and a division: relative errors of a few
// 2^-24 far out too (an argument's rounding counts g^2 times there).  By the functions below 16384 x 5504 fp32 took, forward and
// backward, silu 170 and 283 us, gelu 170 and 281, in 8 bits 240 and 211, 252 and 215; so silu takes
// 170 and 283, gelu 190 and 283, in 8 bits 233 and 211, 299 and 293.
__device__ __forceinline__ float sigmoid(float g) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2f(-1.4426950408889634f * g)));
    return r;
}

// Phi(g), and exp(-g^2 / 2): erfc(x) = e^(-x^2) (a1 t + .. + a5 t^5), t = 1 / (1 + p x), x = |g| / sqrt(2) (Hastings,
// Approximations for Digital Computers, 1955; Abramowitz and Stegun 7.1.26): erfc off by 1.5e-7 at most in exact
// arithmetic, Phi as evaluated here by 2.9e-7; relative to Phi 5e-5 down to g = -3, 5e-4 to -4, 1.6e-3 to -5 (fp16's
// rounding is 4.9e-4, and g Phi there below its normal numbers).  The derivative needs the exponential anyway; with
// erff the UNet's unit (4096 x 5120 fp16) took 53 and 47 us, forward and backward, in place of 37 and 35.
__device__ __forceinline__ float2 normal(float g) {
    const float e = ex2f(-0.7213475204444817f * g * g);
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(fabsf(g), 0.3275911f * 0.7071067811865476f, 1.f)));
    float q = fmaf(t, 1.061405429f * 0.5f, -1.453152027f * 0.5f);
    q = fmaf(t, q, 1.421413741f * 0.5f);
    q = fmaf(t, q, -0.284496736f * 0.5f);
    q = fmaf(t, q, 0.254829592f * 0.5f);
    q = q * t * e;
    return make_float2(g < 0.f ? q : 1.f - q, e);
}

// Phi(g) for results of fp32, and as a call: the forward that keeps 8 bits holds 32 of them a feature (446 us inline, 299 as
// a call, the elementwise forward 190 and 203; 16384 x 5504)
__device__ __forceinline__ float exact_phi(float g) { return 0.5f * erfcf(-0.7071067811865476f * g); }
__device__ __noinline__ float exact_phi_call(float g) { return exact_phi(g); }

template <int ACT, bool EXACT, bool CALL = false> __device__ __forceinline__ float act(float g) {
    if constexpr (ACT == SILU) return g * (EXACT ? 1.f / (1.f + expf(-g)) : sigmoid(g));
    else if constexpr (EXACT) return g * (CALL ? exact_phi_call(g) : exact_phi(g));
    else return g * normal(g).x;
}
// act(g) and its derivative
template <int ACT, bool EXACT> __device__ __forceinline__ float2 act2(float g) {
    if constexpr (ACT == SILU) {
        const float q = EXACT ? 1.f / (1.f + expf(-g)) : sigmoid(g), a = g * q;
        return make_float2(a, q + a * (1.f - q));
    } else {
        const float2 n = EXACT ? make_float2(exact_phi(g), expf(-0.5f * g * g)) : normal(g);
        return make_float2(g * n.x, n.x + 0.3989422804014327f * g * n.y);
    }
}

struct Unit {
    const void *gate, *up;       // NULL gate in the backward: from the codes
    int64_t ldg, ldu;
    uint8_t *g8, *u8, *h8;       // NULL: not kept
    int64_t M;
    int K;
};

// forward of 32 tokens x EL features a thread, with what is asked for kept in 8 bits
template <typename T, int EL, int ACT>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 ? 5 : 1) fwd8_kernel(const __grid_constant__ Unit U, T* h) {
    const int k = (blockIdx.y * blockDim.x + threadIdx.x) * EL;
    const int64_t tb = blockIdx.x, t0 = tb * BLOCK;
    if (k >= U.K) return;
    Tile<T, EL> G, P;
    const T *g = static_cast<const T*>(U.gate) + t0 * U.ldg + k, *u = static_cast<const T*>(U.up) + t0 * U.ldu + k;
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) G.load_row(i, g + i * U.ldg, t0 + i < U.M);
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) P.load_row(i, u + i * U.ldu, t0 + i < U.M);
    if (U.g8) G.save(U.g8, tb, U.K, k);
    if (U.u8) P.save(U.u8, tb, U.K, k);
    T* out = h + t0 * U.K + k;
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) {
        float v[EL];
#pragma unroll
        for (int j = 0; j < EL; ++j) v[j] = act<ACT, sizeof(T) == 4, true>(G.get(i, j)) * P.get(i, j);
        G.set_row(i, v);
        if (t0 + i < U.M) G.store_row(i, out + (int64_t)i * U.K);
    }
    if (U.h8) G.save(U.h8, tb, U.K, k);
}

// backward from the codes, 16 tokens x EL features a thread
template <typename T, int EL, int ACT>
__global__ void __launch_bounds__(THREADS)
    bwd8_kernel(const __grid_constant__ Unit U, const T* dh, int64_t lddh, T* dg, int64_t lddg, T* du, int64_t lddu) {
    const int k = (blockIdx.y * blockDim.x + threadIdx.x) * EL;
    const int64_t tb = blockIdx.x, t0 = tb * 16;
    if (k >= U.K || t0 >= U.M) return;
    const Place at(tb >> 2, k, U.K);
    Tile<T, EL> D;
    uint4 cg[EL], cu[EL];
    float sg[EL], su[EL];
    load_codes<EL>(U.g8 + at.codes(tb & 3), cg);
    load_codes<EL>(U.u8 + at.codes(tb & 3), cu);
#pragma unroll
    for (int i = 0; i < 16; ++i) D.load_row(i, dh + (t0 + i) * lddh + k, t0 + i < U.M);
#pragma unroll
    for (int j = 0; j < EL; ++j) {
        sg[j] = scale_of(U.g8[at.scale((tb >> 1) & 1) + j]);
        su[j] = scale_of(U.u8[at.scale((tb >> 1) & 1) + j]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float a[EL], b[EL];
#pragma unroll
        for (int j = 0; j < EL; ++j) {
            const uint32_t wg = (i < 4 ? cg[j].x : i < 8 ? cg[j].y : i < 12 ? cg[j].z : cg[j].w) ^ 0x80808080u;
            const uint32_t wu = (i < 4 ? cu[j].x : i < 8 ? cu[j].y : i < 12 ? cu[j].z : cu[j].w) ^ 0x80808080u;
            const float g = value(wg, i & 3, sg[j]), u = value(wu, i & 3, su[j]);
            const float2 f = act2<ACT, sizeof(T) == 4>(g);
            const float d = D.get(i, j);
            a[j] = d * u * f.y;
            b[j] = d * f.x;
        }
        if (t0 + i < U.M) {
            Tile<T, EL> O;
            O.set_row(0, a);
            O.store_row(0, dg + (t0 + i) * lddg + k);
            O.set_row(0, b);
            O.store_row(0, du + (t0 + i) * lddu + k);
        }
    }
}

// forward and backward on the inputs themselves: VEC features of ROWS tokens a thread
template <typename T, int VEC, int ROWS, int ACT>
__global__ void __launch_bounds__(256) fwd_kernel(const __grid_constant__ Unit U, T* h) {
    const int k = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    const int64_t t0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * ROWS;
    if (k >= U.K) return;
    float g[ROWS][VEC], u[ROWS][VEC];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (t0 + r >= U.M) break;
        load_vec<VEC>(static_cast<const T*>(U.gate) + (t0 + r) * U.ldg + k, g[r]);
        load_vec<VEC>(static_cast<const T*>(U.up) + (t0 + r) * U.ldu + k, u[r]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (t0 + r >= U.M) break;
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[r][j] = act<ACT, sizeof(T) == 4>(g[r][j]) * u[r][j];
        store_vec<VEC>(h + (t0 + r) * U.K + k, g[r]);
    }
}

template <typename T, int VEC, int ROWS, int ACT>
__global__ void __launch_bounds__(256)
    bwd_kernel(const __grid_constant__ Unit U, const T* dh, int64_t lddh, T* dg, int64_t lddg, T* du, int64_t lddu) {
    const int k = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    const int64_t t0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * ROWS;
    if (k >= U.K) return;
    float g[ROWS][VEC], u[ROWS][VEC], d[ROWS][VEC];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (t0 + r >= U.M) break;
        load_vec<VEC>(static_cast<const T*>(U.gate) + (t0 + r) * U.ldg + k, g[r]);
        load_vec<VEC>(static_cast<const T*>(U.up) + (t0 + r) * U.ldu + k, u[r]);
        load_vec<VEC>(dh + (t0 + r) * lddh + k, d[r]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (t0 + r >= U.M) break;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float2 f = act2<ACT, sizeof(T) == 4>(g[r][j]);
            g[r][j] = d[r][j] * u[r][j] * f.y;
            u[r][j] = d[r][j] * f.x;
        }
        store_vec<VEC>(dg + (t0 + r) * lddg + k, g[r]);
        store_vec<VEC>(du + (t0 + r) * lddu + k, u[r]);
    }
}

// ---------------------------------------------------------------- host side
size_t esize(int32_t t) { return t == CONCORD_F32 ? 4 : 2; }

// blocks of whole warps over pieces of `el` features
void across(int64_t K, int el, int* threads, int* blocks) {
    const int64_t pieces = (K + el - 1) / el, n = (pieces + THREADS - 1) / THREADS;
    *blocks = (int)n;
    *threads = (int)(((pieces + n - 1) / n + 31) / 32 * 32);
}
// the same for the elementwise kernels, several rows a block
void tall(int64_t K, int vec, dim3* threads, int* blocks) {
    const int64_t pieces = (K + vec - 1) / vec, x = pieces < 256 ? pieces : 256;
    *threads = dim3((unsigned)x, (unsigned)(256 / x), 1);
    *blocks = (int)((pieces + x - 1) / x);
}

int check_shape(const char* name, int32_t type, int64_t M, int64_t K, int64_t ld) {
    if (type < 0 || type > 2) return fail(CONCORD_EINVAL, std::string(name) + ": unknown element type");
    if (M < 0 || K <= 0 || ld < K) return fail(CONCORD_ESHAPE, std::string(name) + ": bad extents or row stride");
    if (K > (1 << 20) || M > ((int64_t)1 << 31))
        return fail(CONCORD_ETOOBIG, std::string(name) + ": more than 2^20 features or 2^31 tokens");
    return CONCORD_OK;
}
// the widest piece of a row, in elements, up to `most` bytes, that the given rows are made of (K, their strides and
// addresses in turn: `same` is all of these or-ed together)
template <typename T> int piece(uint64_t same, int most) {
    int el = most / (int)sizeof(T);
    while (el > 1 && same % (el * sizeof(T))) el /= 2;
    return el;
}
uint64_t bytes_of(const void* p, int64_t ld, int32_t type) { return reinterpret_cast<uintptr_t>(p) | (uint64_t)ld * esize(type); }

template <typename T> int save(const void* x, int64_t ldx, int32_t type, uint8_t* saved, int64_t M, int64_t K, cudaStream_t st) {
    constexpr int MOST = SAVE_BYTES / sizeof(T);
    const int el = piece<T>(bytes_of(x, ldx, type) | (uint64_t)K * sizeof(T), SAVE_BYTES);
    int threads, blocks_k;
    across(K, el, &threads, &blocks_k);
    auto k = el == MOST ? save_kernel<T, MOST> : el == 2 ? save_kernel<T, 2> : save_kernel<T, 1>;
    k<<<dim3((unsigned)blocks(M), blocks_k), threads, 0, st>>>(static_cast<const T*>(x), ldx, saved, M, (int)K);
    return check_launch("concord_save8");
}

template <typename T> int dense(const uint8_t* saved, void* out, int64_t ldo, int32_t type, int64_t M, int64_t K, cudaStream_t st) {
    constexpr int MOST = SAVE_BYTES / sizeof(T);
    const int el = piece<T>(bytes_of(out, ldo, type) | (uint64_t)K * sizeof(T), SAVE_BYTES);
    int threads, blocks_k;
    across(K, el, &threads, &blocks_k);
    auto k = el == MOST ? dense_kernel<T, MOST> : el == 2 ? dense_kernel<T, 2> : dense_kernel<T, 1>;
    k<<<dim3((unsigned)(2 * blocks(M)), blocks_k), threads, 0, st>>>(saved, static_cast<T*>(out), ldo, M, (int)K);
    return check_launch("concord_dense8");
}

template <typename T, int ACT> int forward(const Unit& U, void* h, int32_t type, cudaStream_t st) {
    T* out = static_cast<T*>(h);
    const uint64_t rows = bytes_of(U.gate, U.ldg, type) | bytes_of(U.up, U.ldu, type) | (uint64_t)U.K * sizeof(T);
    if (U.g8 || U.u8 || U.h8) {
        constexpr int MOST = FWD_BYTES / sizeof(T);
        const int el = piece<T>(rows | reinterpret_cast<uintptr_t>(h), FWD_BYTES);
        int threads, blocks_k;
        across(U.K, el, &threads, &blocks_k);
        auto k = el == MOST ? fwd8_kernel<T, MOST, ACT> : fwd8_kernel<T, 1, ACT>;
        k<<<dim3((unsigned)blocks(U.M), blocks_k), threads, 0, st>>>(U, out);
        return check_launch("concord_gated_fwd");
    }
    constexpr int VEC = 16 / sizeof(T);
    const bool vec = (rows | reinterpret_cast<uintptr_t>(h)) % 16 == 0;
    dim3 threads;
    int blocks_k;
    tall(U.K, vec ? VEC : 1, &threads, &blocks_k);
    const int64_t each = (vec ? 2 : TALL) * (int64_t)threads.y;
    auto k = vec ? fwd_kernel<T, VEC, 2, ACT> : fwd_kernel<T, 1, TALL, ACT>;
    k<<<dim3((unsigned)((U.M + each - 1) / each), blocks_k), threads, 0, st>>>(U, out);
    return check_launch("concord_gated_fwd");
}

template <typename T, int ACT>
int backward(const Unit& U, const void* dh, int64_t lddh, void* dg, int64_t lddg, void* du, int64_t lddu, int32_t type,
             cudaStream_t st) {
    const T* up = static_cast<const T*>(dh);
    T *og = static_cast<T*>(dg), *ou = static_cast<T*>(du);
    uint64_t rows = bytes_of(dh, lddh, type) | bytes_of(dg, lddg, type) | bytes_of(du, lddu, type) | (uint64_t)U.K * sizeof(T);
    if (U.g8) {
        constexpr int MOST = BWD_BYTES / sizeof(T);
        const int el = piece<T>(rows, BWD_BYTES);
        int threads, blocks_k;
        across(U.K, el, &threads, &blocks_k);
        auto k = el == MOST ? bwd8_kernel<T, MOST, ACT> : el == 2 ? bwd8_kernel<T, 2, ACT> : bwd8_kernel<T, 1, ACT>;
        k<<<dim3((unsigned)(2 * blocks(U.M)), blocks_k), threads, 0, st>>>(U, up, lddh, og, lddg, ou, lddu);
        return check_launch("concord_gated_bwd");
    }
    rows |= bytes_of(U.gate, U.ldg, type) | bytes_of(U.up, U.ldu, type);
    constexpr int VEC = 16 / sizeof(T);
    const bool vec = rows % 16 == 0;
    dim3 threads;
    int blocks_k;
    tall(U.K, vec ? VEC : 1, &threads, &blocks_k);
    const int64_t each = (vec ? 1 : TALL) * (int64_t)threads.y;
    auto k = vec ? bwd_kernel<T, VEC, 1, ACT> : bwd_kernel<T, 1, TALL, ACT>;
    k<<<dim3((unsigned)((U.M + each - 1) / each), blocks_k), threads, 0, st>>>(U, up, lddh, og, lddg, ou, lddu);
    return check_launch("concord_gated_bwd");
}

#define EIGHT_TYPES(type, F, ...)                                         \
    switch (type) {                                                       \
        case CONCORD_F32: return F<float>(__VA_ARGS__);                   \
        case CONCORD_BF16: return F<__nv_bfloat16>(__VA_ARGS__);          \
        default: return F<__half>(__VA_ARGS__);                           \
    }
#define GATED_TYPES(type, a, F, ...)                                                                                    \
    switch ((type) * 2 + (a)) {                                                                                         \
        case 0: return F<float, SILU>(__VA_ARGS__);                                                                     \
        case 1: return F<float, GELU>(__VA_ARGS__);                                                                     \
        case 2: return F<__nv_bfloat16, SILU>(__VA_ARGS__);                                                             \
        case 3: return F<__nv_bfloat16, GELU>(__VA_ARGS__);                                                             \
        case 4: return F<__half, SILU>(__VA_ARGS__);                                                                    \
        default: return F<__half, GELU>(__VA_ARGS__);                                                                   \
    }

int save_any(const void* x, int64_t ldx, int32_t type, uint8_t* saved, int64_t M, int64_t K, cudaStream_t st) {
    EIGHT_TYPES(type, save, x, ldx, type, saved, M, K, st)
}
int dense_any(const uint8_t* saved, void* out, int64_t ldo, int32_t type, int64_t M, int64_t K, cudaStream_t st) {
    EIGHT_TYPES(type, dense, saved, out, ldo, type, M, K, st)
}
int forward_any(const Unit& U, void* h, int32_t type, int a, cudaStream_t st) {
    GATED_TYPES(type, a, forward, U, h, type, st)
}
int backward_any(const Unit& U, const void* dh, int64_t lddh, void* dg, int64_t lddg, void* du, int64_t lddu,
                 int32_t type, int a, cudaStream_t st) {
    GATED_TYPES(type, a, backward, U, dh, lddh, dg, lddg, du, lddu, type, st)
}

}  // namespace eight
}  // namespace concord

using namespace concord;

extern "C" size_t concord_saved8_bytes(int64_t M, int64_t K) {
    if (M <= 0 || K <= 0 || K > (1 << 20) || M > ((int64_t)1 << 31)) return 0;
    return (size_t)eight::all_bytes(M, K);
}

extern "C" int concord_save8(const void* x, int32_t type, int64_t ldx, void* saved, int64_t M, int64_t K, void* stream) {
    if (int rc = eight::check_shape("concord_save8", type, M, K, ldx)) return rc;
    if (M == 0) return CONCORD_OK;
    if (!x || !saved) return fail(CONCORD_EINVAL, "concord_save8: null pointer");
    if (!aligned(saved, 32)) return fail(CONCORD_EALIGN, "concord_save8: saved must be 32-byte aligned");
    return eight::save_any(x, ldx, type, static_cast<uint8_t*>(saved), M, K, as_stream(stream));
}

extern "C" int concord_dense8(const void* saved, void* out, int32_t type, int64_t ldo, int64_t M, int64_t K, void* stream) {
    if (int rc = eight::check_shape("concord_dense8", type, M, K, ldo)) return rc;
    if (M == 0) return CONCORD_OK;
    if (!out || !saved) return fail(CONCORD_EINVAL, "concord_dense8: null pointer");
    if (!aligned(saved, 32)) return fail(CONCORD_EALIGN, "concord_dense8: saved must be 32-byte aligned");
    return eight::dense_any(static_cast<const uint8_t*>(saved), out, ldo, type, M, K, as_stream(stream));
}

extern "C" int concord_gated_fwd(const void* gate, int64_t ldg, const void* up, int64_t ldu, int32_t type, int32_t act,
                                 void* h, void* saved_gate, void* saved_up, void* saved_h, int64_t M, int64_t K,
                                 void* stream) {
    if (int rc = eight::check_shape("concord_gated_fwd", type, M, K, ldg < ldu ? ldg : ldu)) return rc;
    if (act < 0 || act > 1) return fail(CONCORD_EINVAL, "concord_gated_fwd: unknown activation");
    if (M == 0) return CONCORD_OK;
    if (!gate || !up || !h) return fail(CONCORD_EINVAL, "concord_gated_fwd: null pointer");
    if (!aligned(saved_gate, 32) || !aligned(saved_up, 32) || !aligned(saved_h, 32))
        return fail(CONCORD_EALIGN, "concord_gated_fwd: saved tensors must be 32-byte aligned");
    const eight::Unit U{gate, up, ldg, ldu, static_cast<uint8_t*>(saved_gate), static_cast<uint8_t*>(saved_up),
                        static_cast<uint8_t*>(saved_h), M, (int)K};
    return eight::forward_any(U, h, type, act, as_stream(stream));
}

extern "C" int concord_gated_bwd(const void* gate, int64_t ldg, const void* up, int64_t ldu, const void* saved_gate,
                                 const void* saved_up, int32_t type, int32_t act, const void* dh, int64_t lddh,
                                 void* dgate, int64_t lddg, void* dup, int64_t lddu, int64_t M, int64_t K, void* stream) {
    const char* name = "concord_gated_bwd";
    const int64_t lo = lddh < lddg ? lddh : lddg;
    if (int rc = eight::check_shape(name, type, M, K, lo < lddu ? lo : lddu)) return rc;
    if (act < 0 || act > 1) return fail(CONCORD_EINVAL, std::string(name) + ": unknown activation");
    if (M == 0) return CONCORD_OK;
    if (!dh || !dgate || !dup || !saved_gate != !saved_up || (!saved_gate && (!gate || !up)))
        return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    if (!saved_gate && (ldg < K || ldu < K)) return fail(CONCORD_ESHAPE, std::string(name) + ": bad row stride");
    if (!aligned(saved_gate, 32) || !aligned(saved_up, 32))
        return fail(CONCORD_EALIGN, std::string(name) + ": saved tensors must be 32-byte aligned");
    const eight::Unit U{gate, up, ldg, ldu, static_cast<uint8_t*>(const_cast<void*>(saved_gate)),
                        static_cast<uint8_t*>(const_cast<void*>(saved_up)), nullptr, M, (int)K};
    return eight::backward_any(U, dh, lddh, dgate, lddg, dup, lddu, type, act, as_stream(stream));
}
