// vec.cuh — element types of the training operators: loads and stores of VEC
// consecutive elements as fp32, and sums over a warp.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace concord {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t u, __half) {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}

// 16 bytes of T (4 floats or 8 halves) <-> fp32
template <typename T> struct Pack16 {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& u, float* v) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2(w[i], T());
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        return make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()),
                          pack2(v[6], v[7], T()));
    }
};
template <> struct Pack16<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& u, float* v) {
        v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y);
        v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};

// VEC = 8: 16-byte accesses (the address must be 16-byte aligned); VEC = 1: one element
template <int VEC, typename T> __device__ __forceinline__ void load_vec(const T* p, float* v) {
    if constexpr (VEC == 1) v[0] = to_f32(*p);
    else {
        const uint4* q = reinterpret_cast<const uint4*>(p);
#pragma unroll
        for (int i = 0; i < VEC / Pack16<T>::N; ++i) Pack16<T>::unpack(q[i], v + i * Pack16<T>::N);
    }
}
template <int VEC, typename T> __device__ __forceinline__ void store_vec(T* p, const float* v) {
    if constexpr (VEC == 1) *p = from_f32<T>(v[0]);
    else {
        uint4* q = reinterpret_cast<uint4*>(p);
#pragma unroll
        for (int i = 0; i < VEC / Pack16<T>::N; ++i) q[i] = Pack16<T>::pack(v + i * Pack16<T>::N);
    }
}

// asynchronous copies of 16 bytes into shared memory, in groups of this thread
__device__ __forceinline__ void copy16(uint32_t smem, const void* g) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(g) : "memory");
}
__device__ __forceinline__ uint4 read16(uint32_t smem) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(smem)
                 : "memory");
    return v;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// 2^x, subnormal results flushed to 0 (without .ftz each call costs three more instructions)
__device__ __forceinline__ float ex2f(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// two fp32 values as one operand of the packed instructions
__device__ __forceinline__ uint64_t f2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unf2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// the same, a NaN among them wins
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^x of two values on the fma pipe, beside the special-function unit (which
// gives 4 a cycle and scheduler): x = n + f with n the nearest whole number, a
// polynomial in f whose relative error is least on [-1/2, 1/2] (2.6e-6; fitted
// by least squares reweighted by the error, Lawson's method), n added to the
// exponent.  x below -126 counts as -126; x is not NaN and below 128.
__device__ __forceinline__ void ex2_fma2(uint64_t x, float& a, float& b) {
    unf2(x, a, b);
    x = f2(fmaxf(a, -126.f), fmaxf(b, -126.f));
    const uint64_t shift = f2(12582912.f, 12582912.f), back = f2(-12582912.f, -12582912.f);     // 1.5 * 2^23
    const uint64_t r = add2(x, shift), n = add2(r, back);
    const uint64_t f = fma2(n, f2(-1.f, -1.f), x);
    uint64_t p = fma2(f, f2(0.009570101434f, 0.009570101434f), f2(0.05591786028f, 0.05591786028f));
    p = fma2(p, f, f2(0.2402474484f, 0.2402474484f));
    p = fma2(p, f, f2(0.6931218147f, 0.6931218147f));
    p = fma2(p, f, f2(0.9999992614f, 0.9999992614f));
    float ra, rb;
    unf2(r, ra, rb);
    unf2(p, a, b);
    a = __uint_as_float(__float_as_uint(a) + (__float_as_uint(ra) << 23));
    b = __uint_as_float(__float_as_uint(b) + (__float_as_uint(rb) << 23));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_maxf(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// 32 bytes at once
__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
                 "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
}
__device__ __forceinline__ void load32(const void* p, uint4& a, uint4& b) {
    asm("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
        : "l"(p));
}

}  // namespace concord
