// eight.cuh — values kept in 8 bits.
//
// 32 tokens of one feature share a power of two 2^e, the least with |x| <= 127
// 2^e, -126 at least; each value is the whole number nearest to x / 2^e (ties to even), so it is
// off by at most half a step, 2^(e - 1), which is below max|x| / 127 (where max|x| is above 2^-120).  In the block of
// a type's largest values (fp16: above 127 2^9, else above 127 2^121) codes end at 63, as 64 steps
// are more than the type holds: values there are off by less than one step.  Powers of two make both
// directions exact: x / 2^e before its one rounding, and what is read back has at
// most 7 significant bits, so it is the same in fp32, bf16 and fp16.  A block
// is one feature's because features differ in size far more than a feature does from token to token.
//
// Stored in tiles of 64 tokens x 128 features, a tile's bytes together (one
// copy fetches what a step of the weight gradient's product reads): codes
// [4][features][16], 16 tokens of a feature side by side, then the bytes e +
// 127, [2][features].  Tiles stand in order of tokens, then features; features
// are filled up to a multiple of 16 (the last tile of a row of tiles is narrower),
// tokens to one of 64, with zeros.  A block with a NaN or an infinity has the byte
// 255 and codes 0: 0 * 2^128 reads as NaN.
#pragma once

#include "vec.cuh"

namespace concord {
namespace eight {

constexpr int BLOCK = 32;

constexpr int TOKENS = 64, FEATS = 128, TILE_BYTES = TOKENS * FEATS + 2 * FEATS;

__host__ __device__ constexpr int64_t token_tiles(int64_t M) { return (M + TOKENS - 1) / TOKENS; }
__host__ __device__ constexpr int64_t blocks(int64_t M) { return 2 * token_tiles(M); }     // of 32 tokens
// features of a row of tiles, its bytes, and those of all rows
__host__ __device__ constexpr int64_t padded(int64_t K) { return (K + 15) / 16 * 16; }
__host__ __device__ constexpr int64_t row_bytes(int64_t K) { return padded(K) * (TOKENS + 2); }
__host__ __device__ constexpr int64_t all_bytes(int64_t M, int64_t K) { return token_tiles(M) * row_bytes(K); }

// where the codes of 16 tokens (t16: the token's number / 16) of feature k stand, and the byte of block tb
struct Place {
    int64_t tile;             // offset of the tile
    int width, k;             // its features, and k's place among them
    __host__ __device__ __forceinline__ Place(int64_t token_tile, int feature, int64_t K) {
        const int col = feature / FEATS;
        tile = token_tile * row_bytes(K) + (int64_t)col * TILE_BYTES;
        const int64_t left = padded(K) - (int64_t)col * FEATS;
        width = left < FEATS ? (int)left : FEATS;
        k = feature % FEATS;
    }
    __host__ __device__ __forceinline__ int64_t codes(int t16) const { return tile + ((int64_t)t16 * width + k) * 16; }
    __host__ __device__ __forceinline__ int64_t scale(int block) const { return tile + TOKENS * width + block * width + k; }
};

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
// both operations after it (one fma instead would take 2^23 times the largest scales, which is infinite)
__device__ __forceinline__ float value(uint32_t flipped, int j, float scale) {
    return (__uint_as_float(__byte_perm(flipped, 0x4b000000u, 0x7650 + j)) - 8388736.f) * scale;
}

// EL features of 32 tokens in registers, as loaded
template <typename T, int EL> struct Tile {
    static constexpr int W = EL * (int)sizeof(T) / 4 > 0 ? EL * (int)sizeof(T) / 4 : 1;
    uint32_t raw[BLOCK][W];
    __device__ __forceinline__ void load_row(int i, const T* p, bool have) {
        if (!have) {
#pragma unroll
            for (int w = 0; w < W; ++w) raw[i][w] = 0;
        } else if constexpr (EL * sizeof(T) == 2) {
            raw[i][0] = *reinterpret_cast<const uint16_t*>(p);
        } else if constexpr (W == 1) {
            raw[i][0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            static_assert(W == 2, "up to 8 bytes a row");
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            raw[i][0] = v.x;
            raw[i][1] = v.y;
        }
    }
    __device__ __forceinline__ void store_row(int i, T* p) const {
        if constexpr (EL * sizeof(T) == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)raw[i][0];
        else if constexpr (W == 1) *reinterpret_cast<uint32_t*>(p) = raw[i][0];
        else *reinterpret_cast<uint2*>(p) = make_uint2(raw[i][0], raw[i][1]);
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
    // the bits of feature j's largest magnitude, as fp32; word w's two features at once where types are 16 bits wide
    __device__ __forceinline__ void largest(uint32_t* most) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < EL; ++j) {
                most[j] = 0;
#pragma unroll
                for (int i = 0; i < BLOCK; ++i) most[j] = max(most[j], raw[i][j] & 0x7fffffffu);
            }
        } else {
#pragma unroll
            for (int w = 0; w < W; ++w) {
                uint32_t m = 0;           // magnitudes of 16 bits are ordered as signed whole numbers
#pragma unroll
                for (int i = 0; i < BLOCK; i += 2)
                    m = __vimax3_s16x2(m, raw[i][w] & 0x7fff7fffu, raw[i + 1][w] & 0x7fff7fffu);
                const float2 f = unpack2(m, T());
                most[2 * w] = __float_as_uint(f.x);
                if (EL > 1) most[2 * w + 1] = __float_as_uint(f.y);
            }
        }
    }
    // feature j's codes
    template <bool CAPPED> __device__ __forceinline__ void quantize(int j, uint32_t byte, uint4* lo, uint4* hi) const {
        const float inv = __uint_as_float((254 - byte) << 23), magic = 12582912.f;
        uint32_t word[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = get(4 * w + i, j);
                f[i] = CAPPED ? fminf(fmaxf(x * inv, -63.f), 63.f) + magic : fmaf(x, inv, magic);
            }
            word[w] = pack_codes(f[0], f[1], f[2], f[3]);
        }
        *lo = make_uint4(word[0], word[1], word[2], word[3]);
        *hi = make_uint4(word[4], word[5], word[6], word[7]);
    }
    // all features of token block tb, k the first of them
    __device__ __forceinline__ void save(uint8_t* saved, int64_t tb, int64_t K, int k) const {
        const Place at(tb >> 1, k, K);
        const int block = (int)(tb & 1);
        uint4* lo = reinterpret_cast<uint4*>(saved + at.codes(2 * block));
        uint4* hi = reinterpret_cast<uint4*>(saved + at.codes(2 * block + 1));
        uint32_t bytes = 0, most[EL > 1 ? EL : 2];
        largest(most);
        uint4 a[EL], b[EL];
#pragma unroll
        for (int j = 0; j < EL; ++j) {
            const uint32_t byte = scale_byte(most[j]);
            if (byte < TOP<T>) quantize<false>(j, byte, &a[j], &b[j]);
            else if (byte < 255) quantize<true>(j, byte, &a[j], &b[j]);
            else a[j] = b[j] = make_uint4(0, 0, 0, 0);
            bytes |= byte << (8 * j);
            if constexpr (EL == 1) {
                lo[0] = a[0];
                hi[0] = b[0];
            } else if (j % 2) {
                store32(lo + j - 1, a[j - 1], a[j]);
                store32(hi + j - 1, b[j - 1], b[j]);
            }
        }
        uint8_t* sc = saved + at.scale(block);
        if constexpr (EL == 4) *reinterpret_cast<uint32_t*>(sc) = bytes;
        else if constexpr (EL == 2) *reinterpret_cast<uint16_t*>(sc) = (uint16_t)bytes;
        else {
#pragma unroll
            for (int j = 0; j < EL; ++j) sc[j] = (uint8_t)(bytes >> (8 * j));
        }
        // the features that fill the row of tiles up
        if (k + EL >= K) {
            for (int j = 0; k + EL + j < padded(K); ++j) {
                lo[EL + j] = hi[EL + j] = make_uint4(0, 0, 0, 0);
                sc[EL + j] = 1;
            }
        }
    }
};

}  // namespace eight
}  // namespace concord
