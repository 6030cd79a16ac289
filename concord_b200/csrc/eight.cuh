// eight.cuh — values kept in 8 bits.
//
// 32 tokens of one feature share a power of two 2^e, the least with |x| <= 127
// 2^e; each value is the whole number nearest to x / 2^e (ties to even), so it is
// off by at most half a step, 2^(e - 1) < max|x| / 127.  Powers of two make both
// directions exact: x / 2^e before its one rounding, and what is read back has at
// most 7 significant bits, so it is the same in fp32, bf16 and fp16.  A block
// is one feature's because features differ in size far more than a feature does from token to token.
//
// Stored: codes [ceil(M / 32) * 2][K][16], 16 tokens of a feature side by side
// (the piece that a lane of the weight gradient's product reads at once), rows
// beyond M as zeros; then one byte e + 127 a block, [ceil(M / 32)][K rounded up to 16].  A block
// with a NaN or an infinity has the byte 255 and codes 0: 0 * 2^128 reads as NaN.
#pragma once

#include "vec.cuh"

namespace concord {
namespace eight {

constexpr int BLOCK = 32;

__host__ __device__ constexpr int64_t blocks(int64_t M) { return (M + BLOCK - 1) / BLOCK; }
__host__ __device__ constexpr int64_t code_bytes(int64_t M, int64_t K) { return blocks(M) * BLOCK * K; }
__host__ __device__ constexpr int64_t scale_row(int64_t K) { return (K + 15) / 16 * 16; }

// the byte of a block whose largest magnitude has these bits (a NaN's are the largest)
__device__ __forceinline__ uint32_t scale_byte(uint32_t most) {
    if (most >= 0x7f800000u) return 255;
    const int e = (int)((most + 0x1ffffu) >> 23) - 6;          // beyond 127/64 of its power of two: the next one
    return e < 1 ? 1 : (uint32_t)e;
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// The largest values of a type lie half a step below what the type cannot hold:
// the block's byte where 64 steps would pass it (127 elsewhere).
template <typename T> constexpr uint32_t TOP = 249;
template <> constexpr uint32_t TOP<__half> = 137;

// four codes (as the low bytes of 1.5 * 2^23 + code)
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
    const uint32_t ab = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
    const uint32_t cd = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
}
// byte j of four codes with their signs flipped (x ^ 0x80808080), times scale: 2^23 + 128 + code is exact, and
// so is what the fma leaves
__device__ __forceinline__ float value(uint32_t flipped, int j, float scale, float off) {
    return fmaf(__uint_as_float(__byte_perm(flipped, 0x4b000000u, 0x7650 + j)), scale, off);
}
__device__ __forceinline__ float value_off(float scale) { return -8388736.f * scale; }

// EL features of 32 tokens in registers, as loaded
template <typename T, int EL> struct Tile {
    static constexpr int W = EL * (int)sizeof(T) / 4 > 0 ? EL * (int)sizeof(T) / 4 : 1;
    uint32_t raw[BLOCK][W];
    __device__ __forceinline__ void load_row(int i, const T* p, bool have) {
        if (!have) {
#pragma unroll
            for (int w = 0; w < W; ++w) raw[i][w] = 0;
        } else if constexpr (EL == 1) {
            if constexpr (sizeof(T) == 4) raw[i][0] = *reinterpret_cast<const uint32_t*>(p);
            else raw[i][0] = *reinterpret_cast<const uint16_t*>(p);
        } else {
            static_assert(W == 2, "8 bytes a row");
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            raw[i][0] = v.x;
            raw[i][1] = v.y;
        }
    }
    __device__ __forceinline__ void store_row(int i, T* p) const {
        if constexpr (EL == 1) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = raw[i][0];
            else *reinterpret_cast<uint16_t*>(p) = (uint16_t)raw[i][0];
        } else {
            *reinterpret_cast<uint2*>(p) = make_uint2(raw[i][0], raw[i][1]);
        }
    }
    __device__ __forceinline__ float get(int i, int j) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(raw[i][j]);
        else {
            const float2 f = unpack2(raw[i][j / 2], T());
            return j & 1 ? f.y : f.x;
        }
    }
    __device__ __forceinline__ void set_row(int i, const float* v) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < EL; ++j) raw[i][j] = __float_as_uint(v[j]);
        } else if constexpr (EL == 1) {
            raw[i][0] = pack2(v[0], 0.f, T());
        } else {
#pragma unroll
            for (int w = 0; w < W; ++w) raw[i][w] = pack2(v[2 * w], v[2 * w + 1], T());
        }
    }
    // feature j's byte and codes
    __device__ __forceinline__ uint32_t quantize(int j, uint4* lo, uint4* hi) const {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < BLOCK; ++i) most = max(most, __float_as_uint(get(i, j)) & 0x7fffffffu);
        const uint32_t byte = scale_byte(most);
        const float inv = byte == 255 ? 0.f : __uint_as_float((254 - byte) << 23), magic = 12582912.f;
        const float cap = byte == TOP<T> ? 63.f : 127.f;
        uint32_t word[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = get(4 * w + i, j);
                if (byte >= TOP<T>) x = byte == 255 ? 0.f : fminf(fmaxf(x * inv, -cap), cap) * scale_of(byte);
                f[i] = fmaf(x, inv, magic);
            }
            word[w] = pack_codes(f[0], f[1], f[2], f[3]);
        }
        *lo = make_uint4(word[0], word[1], word[2], word[3]);
        *hi = make_uint4(word[4], word[5], word[6], word[7]);
        return byte;
    }
    // all features of token block tb, k the first of them
    __device__ __forceinline__ void save(int8_t* codes, uint8_t* scales, int64_t tb, int64_t K, int k) const {
        uint4* at = reinterpret_cast<uint4*>(codes) + 2 * tb * K + k;
        uint32_t bytes = 0;
#pragma unroll
        for (int j = 0; j < EL; ++j) {
            uint4 lo, hi;
            const uint32_t b = quantize(j, &lo, &hi);
            at[j] = lo;
            at[K + j] = hi;
            bytes |= b << (8 * j);
        }
#pragma unroll
        for (int j = 0; j < EL; ++j) scales[tb * scale_row(K) + k + j] = (uint8_t)(bytes >> (8 * j));
    }
};

}  // namespace eight
}  // namespace concord
