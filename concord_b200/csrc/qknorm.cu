// qknorm.cu — root-mean-square norm of every query and key head with the
// position rotation in the same pass, and the gradient of both.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w            (n = x without the norm)
//   (a, b) -> (a c - b s, a s + b c)                      for every rotated pair of n, c and s of the token's position
//   backward: dn = the rotation undone on dy,  g = dn w,
//   dx = r g - x r^3 sum(g x) / D,  dw = sum over tokens and heads of dn x r
//
// Bound by memory: the forward reads and writes q and k once, the backward reads
// dy and x and writes dx.  A row (one head of one token) stays in the
// registers of a group of lanes, 4 or 2 pairs each, a pair's two halves in one lane
// whichever way pairs are laid out, so that the rotation needs no exchange; the
// group's lanes share sums by shuffles (both sums of the backward in one go:
// neither needs r).  Blocks belong to q or to k; a thread walks its tokens' heads
// with the rows after the present one on their way, as they come from memory, and keeps its
// part of cos and sin for a token and its columns' weights for all of
// them.  The weights' gradients are added per thread, then per block,
// then over blocks in a fixed order: no atomics, the same bits on every run of
// one device.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "vec.cuh"

namespace concord {
namespace qkn {

constexpr int MAX_DIM = 256, THREADS = 256;
// Rows that a thread has on their way or in hand where its part of them goes through shared memory: asynchronous
// copies into its own place there, which it reads back itself, so that nothing waits but the
// thread.  (16384 tokens, 2 x 16 heads of 128 bf16, neighbours and halves: forward 45 and 46 us, backward 67 and
// 69; the rows in registers, two or three ahead, 51 and 55, 76 and 85.  fp32 does better in registers:
// halves 93 and 150, through shared memory 161 and 239; so do pieces of 4 bytes, below.)
constexpr int RING = 6;

// q or k
struct Side {
    const void *x, *dy;
    void* out;                    // contiguous [T, heads, D]
    const float* w;               // NULL: ones
    int64_t ts, hs, dts, dhs;     // token and head strides of x and dy, elements
    int heads, share;             // share: row groups of a block beside one another in a token's heads
};

struct Params {
    const float *cos, *sin;       // [positions, rot / 2]
    const void* pos;              // [T], or NULL: the token's number
    int pos64;
    int64_t T, positions;
    int D, rot, interleaved;
    float eps, inv_d;
    Side side[2];
    int blocks0;                  // blocks of q; the others are k's
    int lanes;                    // of a row, where the kernel does not say
    float* part;                  // backward: [blocks][D]
};

// Where a lane's pairs stand in a row.  VEC: N rotated pairs, or 2 N plain columns,
// as two runs of N columns (PAIRED: pairs, and plain columns, side by side; else first and second
// halves of the pairs); else N pairs 32 apart, for any size and stride.
enum Kind { ANY, HALVES, PAIRED };
template <int N, Kind KIND> struct Lane {
    static constexpr bool VEC = KIND != ANY;
    // VEC: the runs' first columns; else the first pair, and the columns of all (not there: column 0, as loads
    // need no condition, and `have` without their bits)
    int at[VEC ? 2 : 1 + 2 * N];
    uint32_t have;
    bool live, turns;             // VEC: any columns, rotated ones
    int rot;
    __device__ __forceinline__ Lane(const Params& P, int lane) : have(0), rot(P.rot) {
        if constexpr (VEC) {
            live = lane * 2 * N < P.D;
            turns = lane * 2 * N < rot;
            at[0] = !live ? 0 : turns && KIND == HALVES ? lane * N : lane * 2 * N;
            at[1] = !live ? N : turns && KIND == HALVES ? rot / 2 + lane * N : lane * 2 * N + N;    // (not live: loads need no condition)
        } else {
            live = turns = true;
            at[0] = lane;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int p = lane + 32 * j, half = rot / 2;
                int a = rot + 2 * (p - half), b = a + 1;
                if (p < half) {
                    a = P.interleaved ? 2 * p : p;
                    b = P.interleaved ? 2 * p + 1 : half + p;
                }
                have |= (a < P.D ? 1u : 0u) << (2 * j) | (b < P.D ? 2u : 0u) << (2 * j);
                at[1 + 2 * j] = a < P.D ? a : 0;
                at[2 + 2 * j] = b < P.D ? b : 0;
            }
        }
    }
    __device__ __forceinline__ bool rotated(int j) const { return VEC ? turns : at[0] + 32 * j < rot / 2; }
};

// a lane's part of a row as it comes from memory
template <typename T, int N, Kind KIND> struct Raw {
    static constexpr bool VEC = KIND != ANY;
    static constexpr int RUN = N * (int)sizeof(T), WORDS = VEC ? 2 * RUN / 4 : 2 * N;
    uint32_t v[WORDS];
    __device__ __forceinline__ void fetch(const Lane<N, KIND>& L, const T* row) {
        if constexpr (KIND == PAIRED && N == 4 && RUN == 8) {           // both runs side by side
            const uint4 u = *reinterpret_cast<const uint4*>(row + L.at[0]);
            v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
        } else if constexpr (VEC) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if constexpr (RUN == 4) v[r] = *reinterpret_cast<const uint32_t*>(row + L.at[r]);
                else if constexpr (RUN == 8) {
                    const uint2 u = *reinterpret_cast<const uint2*>(row + L.at[r]);
                    v[2 * r] = u.x;
                    v[2 * r + 1] = u.y;
                } else {
#pragma unroll
                    for (int i = 0; i < RUN / 16; ++i) {
                        const uint4 u = reinterpret_cast<const uint4*>(row + L.at[r])[i];
                        v[r * RUN / 4 + 4 * i] = u.x;
                        v[r * RUN / 4 + 4 * i + 1] = u.y;
                        v[r * RUN / 4 + 4 * i + 2] = u.z;
                        v[r * RUN / 4 + 4 * i + 3] = u.w;
                    }
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2 * N; ++j) v[j] = __float_as_uint(to_f32(row[L.at[1 + j]]));
#pragma unroll
            for (int j = 0; j < 2 * N; ++j)
                if (!(L.have >> j & 1)) v[j] = 0;
        }
    }
    static constexpr bool ASYNC = VEC && RUN == 8 && N == 4;
    static constexpr int SLOT = 4 * WORDS;                        // bytes of a thread's place in the ring
    __device__ __forceinline__ static void start(const Lane<N, KIND>& L, const T* row, uint32_t slot) {
        if constexpr (KIND == PAIRED) copy16(slot, row + L.at[0]);
        else {
#pragma unroll
            for (int r = 0; r < 2; ++r)
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(slot + r * RUN), "l"(row + L.at[r]), "n"(RUN) : "memory");
        }
    }
    __device__ __forceinline__ void take(uint32_t slot) {
        const uint4 u = read16(slot);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
    __device__ __forceinline__ float element(int i) const {       // VEC: the i-th of both runs
        if constexpr (sizeof(T) == 4) return __uint_as_float(v[i]);
        else {
            const float2 f = unpack2(v[i / 2], T());
            return i & 1 ? f.y : f.x;
        }
    }
    // as pairs' first and second elements, two a register pair (packed arithmetic)
    __device__ __forceinline__ void pairs(uint64_t* a, uint64_t* b) const {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            if constexpr (!VEC) {
                a[j] = f2(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 2]));
                b[j] = f2(__uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 3]));
            } else if constexpr (KIND == PAIRED) {
                a[j] = f2(element(4 * j), element(4 * j + 2));
                b[j] = f2(element(4 * j + 1), element(4 * j + 3));
            } else {
                a[j] = f2(element(2 * j), element(2 * j + 1));
                b[j] = f2(element(N + 2 * j), element(N + 2 * j + 1));
            }
        }
    }
};

template <typename T, int N, Kind KIND>
__device__ __forceinline__ void store_pairs(const Lane<N, KIND>& L, T* row, const uint64_t* a2, const uint64_t* b2) {
    float a[N], b[N];
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        unf2(a2[j], a[2 * j], a[2 * j + 1]);
        unf2(b2[j], b[2 * j], b[2 * j + 1]);
    }
    if constexpr (KIND != ANY) {
        float r[2 * N];
        if constexpr (KIND == PAIRED) {
#pragma unroll
            for (int j = 0; j < N; ++j) { r[2 * j] = a[j]; r[2 * j + 1] = b[j]; }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) { r[j] = a[j]; r[N + j] = b[j]; }
        }
        if constexpr (KIND == PAIRED && N == 4 && sizeof(T) == 2) {
            *reinterpret_cast<uint4*>(row + L.at[0]) = Pack16<T>::pack(r);
            return;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            T* p = row + L.at[k];
            if constexpr (N * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = pack2(r[k * N], r[k * N + 1], T());
            else if constexpr (N == 2) *reinterpret_cast<float2*>(p) = make_float2(r[k * N], r[k * N + 1]);
            else if constexpr (N * sizeof(T) == 8)
                *reinterpret_cast<uint2*>(p) = make_uint2(pack2(r[k * N], r[k * N + 1], T()), pack2(r[k * N + 2], r[k * N + 3], T()));
            else {
                uint4* q = reinterpret_cast<uint4*>(p);
#pragma unroll
                for (int i = 0; i < N * (int)sizeof(T) / 16; ++i) q[i] = Pack16<T>::pack(r + k * N + i * Pack16<T>::N);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (L.have >> (2 * j) & 1) row[L.at[1 + 2 * j]] = from_f32<T>(a[j]);
            if (L.have >> (2 * j + 1) & 1) row[L.at[2 + 2 * j]] = from_f32<T>(b[j]);
        }
    }
}

// cos, sin and -sin of position p; NaN where the tables have none
template <int N, Kind KIND>
__device__ __forceinline__ void angles(const Params& P, const Lane<N, KIND>& L, int64_t p, uint64_t* c2, uint64_t* s2,
                                       uint64_t* n2) {
    const bool there = p >= 0 && p < P.positions;
    const int64_t row = p * (P.rot / 2);
    float c[N], s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) c[j] = s[j] = __int_as_float(0x7fffffff);
    if constexpr (KIND != ANY) {
        if (L.live && L.turns && there) {
            const int64_t at = row + (KIND == PAIRED ? L.at[0] / 2 : L.at[0]);
            if constexpr (N == 2) {
                const float2 u = *reinterpret_cast<const float2*>(P.cos + at), v = *reinterpret_cast<const float2*>(P.sin + at);
                c[0] = u.x; c[1] = u.y; s[0] = v.x; s[1] = v.y;
            }
#pragma unroll
            for (int j = 0; j + 4 <= N; j += 4) {
                const float4 u = *reinterpret_cast<const float4*>(P.cos + at + j), v = *reinterpret_cast<const float4*>(P.sin + at + j);
                c[j] = u.x; c[j + 1] = u.y; c[j + 2] = u.z; c[j + 3] = u.w;
                s[j] = v.x; s[j + 1] = v.y; s[j + 2] = v.z; s[j + 3] = v.w;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!L.rotated(j)) {              // (not used: turn leaves these columns alone)
                c[j] = 1.f;
                s[j] = 0.f;
            } else if (there) {
                c[j] = P.cos[row + L.at[0] + 32 * j];
                s[j] = P.sin[row + L.at[0] + 32 * j];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        c2[j] = f2(c[2 * j], c[2 * j + 1]);
        s2[j] = f2(s[2 * j], s[2 * j + 1]);
        n2[j] = f2(-s[2 * j], -s[2 * j + 1]);
    }
}
// (a, b) -> (a c + b m, b c + a s): m = -s turns, with s and -s in each other's place it turns back
template <int N, Kind KIND>
__device__ __forceinline__ void turn(const Lane<N, KIND>& L, uint64_t* a, uint64_t* b, const uint64_t* c, const uint64_t* s,
                                     const uint64_t* m) {
    if (KIND != ANY && !L.turns) return;
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        const uint64_t u = fma2(b[j], m[j], mul2(a[j], c[j])), v = fma2(a[j], s[j], mul2(b[j], c[j]));
        if constexpr (KIND != ANY) {
            a[j] = u;
            b[j] = v;
        } else {
            float ua, ub, va, vb, oa, ob, pa, pb;
            unf2(u, ua, ub);
            unf2(v, va, vb);
            unf2(a[j], oa, ob);
            unf2(b[j], pa, pb);
            const bool first = L.rotated(2 * j), second = L.rotated(2 * j + 1);
            a[j] = f2(first ? ua : oa, second ? ub : ob);
            b[j] = f2(first ? va : pa, second ? vb : pb);
        }
    }
}

__device__ __forceinline__ int64_t position(const Params& P, int64_t t) {
    if (!P.pos || !P.rot) return t;
    return P.pos64 ? static_cast<const int64_t*>(P.pos)[t] : (int64_t)static_cast<const int32_t*>(P.pos)[t];
}

// A thread's row group and its lane there: LANES of them in a row, or (LANES 0) `lanes`, as many groups of these as a warp
// has room for (what is left over has lane 32, which has no columns).
template <int LANES> struct Group {
    int lane, group, groups, lanes;
    __device__ __forceinline__ explicit Group(int of) : lanes(LANES ? LANES : of) {
        if constexpr (LANES != 0) {
            lane = threadIdx.x % LANES;
            group = threadIdx.x / LANES;
            groups = THREADS / LANES;
        } else {
            const int per = 32 / lanes, at = threadIdx.x % 32, in = at / lanes;
            lane = in < per ? at % lanes : 32;
            group = threadIdx.x / 32 * per + min(in, per - 1);
            groups = THREADS / 32 * per;
        }
    }
    // the sum over a row's lanes; every lane of the warp calls it
    __device__ __forceinline__ float sum(float v) const {
        if constexpr (LANES != 0) {
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            return v;
        } else {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) {             // (up to 16 lanes)
                const float u = __shfl_down_sync(0xffffffffu, v, o);
                if (lane + o < lanes) v += u;
            }
            return __shfl_sync(0xffffffffu, v, max((int)(threadIdx.x % 32) - lane, 0));
        }
    }
};

__device__ __forceinline__ float sum2(uint64_t v) {
    float a, b;
    unf2(v, a, b);
    return a + b;
}

// A row group's rows in order: its heads of a token (`share` apart, a divisor of the
// heads), then those of its next token.  Where it stands is the same in
// all groups of a block, so that branches are uniform; a group whose token lies
// beyond the last one reads the last one's (loads need no condition then) and stores nothing.
struct Rows {
    int base, mine, i, per, step, T;
    __device__ __forceinline__ Rows(const Params& P, const Side& S, int block, int blocks, int group, int groups) {
        const int tokens = groups / S.share;
        T = (int)P.T;
        mine = group / S.share;
        base = block * tokens;
        step = blocks * tokens;
        per = S.heads / S.share;
        i = 0;
    }
    __device__ __forceinline__ int token() const { return min(base + mine, T - 1); }
    __device__ __forceinline__ bool here() const { return base + mine < T; }
    __device__ __forceinline__ int64_t steps() const { return base < T ? (int64_t)((T - 1 - base) / step + 1) * per : 0; }
    // to the next row; whether it is another token's
    __device__ __forceinline__ bool next() {
        if (++i < per) return false;
        i = 0;
        base = min(base + step, T);               // (stays there: no overflow)
        return true;
    }
};
template <typename T> __device__ __forceinline__ const T* row_at(const void* p, int64_t ts, int64_t hs, int t, int h) {
    return static_cast<const T*>(p) + t * ts + h * hs;
}

template <typename T, int N, int LANES, Kind KIND, bool NORM>
__global__ void __launch_bounds__(THREADS, Raw<T, N, KIND>::ASYNC ? 3 : KIND == ANY ? 2 : 4) fwd_kernel(const __grid_constant__ Params P) {
    using Row = Raw<T, N, KIND>;
    // rows on their way, the present one included, and those of them in registers
    constexpr bool ASYNC = Row::ASYNC;
    constexpr int DEPTH = ASYNC ? RING : 3, HELD = ASYNC ? 1 : DEPTH, STAGE = THREADS * Row::SLOT;
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * Row::SLOT;
    const int which = blockIdx.x >= P.blocks0, block = blockIdx.x - (which ? P.blocks0 : 0);
    const Side& S = P.side[which];
    const Group<LANES> G(P.lanes);
    const int h0 = G.group % S.share;
    const Lane<N, KIND> L(P, G.lane);
    Rows now(P, S, block, which ? gridDim.x - P.blocks0 : P.blocks0, G.group, G.groups), far = now;
    const int64_t steps = now.steps(), ts = S.ts, hs = S.hs, in_step = hs * S.share, ld = (int64_t)S.heads * P.D;
    const int out_step = S.share * P.D;
    const T* in = row_at<T>(S.x, ts, hs, far.token(), h0);
    T* out = const_cast<T*>(row_at<T>(S.out, ld, P.D, now.token(), h0));
    Row raw[HELD];
    auto fetch = [&](int k) {
        if constexpr (ASYNC) {
            Row::start(L, in, ring + k * STAGE);
            copy_commit();
        } else raw[k].fetch(L, in);
        in += in_step;
        if (far.next()) in = row_at<T>(S.x, ts, hs, far.token(), h0);
    };
#pragma unroll
    for (int k = 0; k < DEPTH - 1; ++k) fetch(k);
    uint64_t wa[N / 2], wb[N / 2], c[N / 2], s[N / 2], m[N / 2];
    if (NORM && S.w) {
        Raw<float, N, KIND> w;
        w.fetch(L, S.w);
        w.pairs(wa, wb);
    } else {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) wa[j] = wb[j] = f2(1.f, 1.f);
    }
    const float inv_d = P.inv_d, eps = P.eps;
    const bool turns = P.rot > 0;
    bool fresh = turns, keep = now.here() && L.live;
    int64_t pos = turns ? position(P, now.token()) : 0;                 // of the next token, once this one's is used
    int stage = 0;
    for (int64_t n = 0; n < steps; n += HELD) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            if constexpr (ASYNC) {
                copy_wait<DEPTH - 2>();
                raw[0].take(ring + stage * STAGE);
            } else fetch((k + DEPTH - 1) % DEPTH);
            if (fresh) {
                angles<N, KIND>(P, L, pos, c, s, m);
                pos = position(P, min(now.base + now.mine + now.step, now.T - 1));
            }
            uint64_t a[N / 2], b[N / 2];
            raw[k].pairs(a, b);
            if constexpr (NORM) {
                uint64_t ss = mul2(a[0], a[0]);
                ss = fma2(b[0], b[0], ss);
#pragma unroll
                for (int j = 1; j < N / 2; ++j) ss = fma2(b[j], b[j], fma2(a[j], a[j], ss));
                const float r = rsqrtf(G.sum(L.live ? sum2(ss) : 0.f) * inv_d + eps);
                const uint64_t r2 = f2(r, r);
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    a[j] = mul2(a[j], mul2(wa[j], r2));
                    b[j] = mul2(b[j], mul2(wb[j], r2));
                }
            }
            if (turns) turn<N, KIND>(L, a, b, c, s, m);
            if (keep) store_pairs<T, N, KIND>(L, out, a, b);
            out += out_step;
            fresh = false;
            if (now.next()) {
                out = const_cast<T*>(row_at<T>(S.out, ld, P.D, now.token(), h0));
                fresh = turns;
                keep = now.here() && L.live;
            }
            if constexpr (ASYNC) {
                fetch(stage == 0 ? DEPTH - 1 : stage - 1);
                stage = stage + 1 == DEPTH ? 0 : stage + 1;
            }
        }
    }
    if constexpr (ASYNC) copy_wait<0>();          // (the last rows again, which nobody reads)
}

template <typename T, int N, int LANES, Kind KIND, bool NORM>
__global__ void __launch_bounds__(THREADS, Raw<T, N, KIND>::ASYNC || KIND != HALVES ? 2 : 3) bwd_kernel(const __grid_constant__ Params P) {
    using Row = Raw<T, N, KIND>;
    constexpr bool ASYNC = Row::ASYNC;            // (fp32: neighbours' rows three ahead 130 us, halves' one ahead and more blocks 150)
    constexpr int DEPTH = ASYNC ? RING : KIND == PAIRED ? 4 : 2, HELD = ASYNC ? 1 : DEPTH;
    constexpr int X = THREADS * Row::SLOT, STAGE = NORM ? 2 * X : X;              // dy's places, then x's
    extern __shared__ __align__(16) uint8_t smem[];
    float* sums = reinterpret_cast<float*>(smem + (ASYNC ? DEPTH * STAGE : 0));   // [row groups][D]
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * Row::SLOT;
    const int which = blockIdx.x >= P.blocks0, block = blockIdx.x - (which ? P.blocks0 : 0);
    const Side& S = P.side[which];
    const Group<LANES> G(P.lanes);
    const int h0 = G.group % S.share;
    const Lane<N, KIND> L(P, G.lane);
    Rows now(P, S, block, which ? gridDim.x - P.blocks0 : P.blocks0, G.group, G.groups), far = now;
    const int64_t steps = now.steps(), ts = S.ts, hs = S.hs, dts = S.dts, dhs = S.dhs, ld = (int64_t)S.heads * P.D;
    const int out_step = S.share * P.D, share = S.share;
    const T *in = row_at<T>(S.dy, dts, dhs, far.token(), h0), *inx = row_at<T>(S.x, ts, hs, far.token(), h0);
    T* out = const_cast<T*>(row_at<T>(S.out, ld, P.D, now.token(), h0));
    Row raw[HELD], rawx[HELD];
    auto fetch = [&](int k) {
        if constexpr (ASYNC) Row::start(L, in, ring + k * STAGE);
        else raw[k].fetch(L, in);
        in += dhs * share;
        if (NORM) {
            if constexpr (ASYNC) Row::start(L, inx, ring + k * STAGE + X);
            else rawx[k].fetch(L, inx);
            inx += hs * share;
        }
        if constexpr (ASYNC) copy_commit();
        if (far.next()) {
            in = row_at<T>(S.dy, dts, dhs, far.token(), h0);
            if (NORM) inx = row_at<T>(S.x, ts, hs, far.token(), h0);
        }
    };
#pragma unroll
    for (int k = 0; k < DEPTH - 1; ++k) fetch(k);
    uint64_t wa[N / 2], wb[N / 2], c[N / 2], s[N / 2], m[N / 2], ga[N / 2], gb[N / 2];   // ga, gb: of the weights' gradient
    if (NORM && S.w) {
        Raw<float, N, KIND> w;
        w.fetch(L, S.w);
        w.pairs(wa, wb);
    } else {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) wa[j] = wb[j] = f2(1.f, 1.f);
    }
#pragma unroll
    for (int j = 0; j < N / 2; ++j) ga[j] = gb[j] = 0;
    const float inv_d = P.inv_d, eps = P.eps;
    const bool turns = P.rot > 0;
    bool fresh = turns, keep = now.here() && L.live;
    int64_t pos = turns ? position(P, now.token()) : 0;
    int stage = 0;
    for (int64_t n = 0; n < steps; n += HELD) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            if constexpr (ASYNC) {
                copy_wait<DEPTH - 2>();
                raw[0].take(ring + stage * STAGE);
                if (NORM) rawx[0].take(ring + stage * STAGE + X);
            } else fetch((k + DEPTH - 1) % DEPTH);
            if (fresh) {
                angles<N, KIND>(P, L, pos, c, s, m);
                pos = position(P, min(now.base + now.mine + now.step, now.T - 1));
            }
            uint64_t a[N / 2], b[N / 2];
            raw[k].pairs(a, b);
            if (turns) turn<N, KIND>(L, a, b, c, m, s);
            if constexpr (NORM) {
                uint64_t xa[N / 2], xb[N / 2], ss = 0, gx = 0;
                rawx[k].pairs(xa, xb);
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    ss = fma2(xb[j], xb[j], fma2(xa[j], xa[j], ss));
                    gx = fma2(mul2(b[j], wb[j]), xb[j], fma2(mul2(a[j], wa[j]), xa[j], gx));
                }
                const float sq = G.sum(L.live ? sum2(ss) : 0.f), gs = G.sum(L.live ? sum2(gx) : 0.f);
                const float r = rsqrtf(sq * inv_d + eps), q = -(r * gs) * inv_d * r * r;          // (r^3 alone leaves fp32 beyond 2^+-42)
                const float rg = keep ? r : 0.f;           // (a row that is not there is another's copy)
                const uint64_t r2 = f2(r, r), q2 = f2(q, q), rg2 = f2(rg, rg);
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    ga[j] = fma2(a[j], mul2(xa[j], rg2), ga[j]);
                    gb[j] = fma2(b[j], mul2(xb[j], rg2), gb[j]);
                    a[j] = fma2(xa[j], q2, mul2(mul2(a[j], wa[j]), r2));
                    b[j] = fma2(xb[j], q2, mul2(mul2(b[j], wb[j]), r2));
                }
            }
            if (keep) store_pairs<T, N, KIND>(L, out, a, b);
            out += out_step;
            fresh = false;
            if (now.next()) {
                out = const_cast<T*>(row_at<T>(S.out, ld, P.D, now.token(), h0));
                fresh = turns;
                keep = now.here() && L.live;
            }
            if constexpr (ASYNC) {
                fetch(stage == 0 ? DEPTH - 1 : stage - 1);
                stage = stage + 1 == DEPTH ? 0 : stage + 1;
            }
        }
    }
    if constexpr (ASYNC) copy_wait<0>();          // (the last rows again, which nobody reads)
    if (NORM && P.part) {
        if (L.live) store_pairs<float, N, KIND>(L, sums + G.group * P.D, ga, gb);
        __syncthreads();
        for (int i = threadIdx.x; i < P.D; i += THREADS) {
            float v = sums[i];
            for (int g = 1; g < G.groups; ++g) v += sums[g * P.D + i];
            P.part[(int64_t)blockIdx.x * P.D + i] = v;
        }
    }
}

// the blocks' sums in a fixed order: 8 columns x 32 strides a block; the first
// blocks of this grid are q's
__global__ void __launch_bounds__(256) sum_kernel(const float* part, int blocks0, int blocks, int D, float* dqw, float* dkw) {
    __shared__ float red[32][9];
    const int per = (D + 7) / 8, side = blockIdx.x >= per;
    const int cx = threadIdx.x & 7, ry = threadIdx.x >> 3, c = (blockIdx.x - side * per) * 8 + cx;
    const int first = side ? blocks0 : 0, last = side ? blocks : blocks0;
    float v = 0.f;
    if (c < D) {
#pragma unroll 8
        for (int k = first + ry; k < last; k += 32) v += part[(int64_t)k * D + c];
    }
    red[ry][cx] = v;
    __syncthreads();
    if (ry == 0 && c < D) {
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) v += red[k][cx];
        float* out = side ? dkw : dqw;
        if (out) out[c] = v;
    }
}

// ---------------------------------------------------------------- host side
constexpr int MAX_DEVICES = 64;
constexpr int MAX_BLOCKS = 148 * 8;       // of the backward, whose blocks each leave a row of sums

// Groups of a block that share a token's heads, a divisor of both, and the blocks: so that the group with
// the most to do has least, a token's cos and sin counted as TOKEN_ROWS rows (16384 tokens, 2 x 32 heads of 64: 55
// and 84 us, with a group a token 59 and 103; counted as 4 rows 59 and 85).
constexpr int TOKEN_ROWS = 1;
int share_of(int64_t T, int heads, int groups, int64_t most, int* blocks) {
    int64_t least = INT64_MAX;
    int best = 1;
    for (int share = 1; groups % share == 0 && heads % share == 0; share *= 2) {
        const int64_t tokens = groups / share, n = std::min((T + tokens - 1) / tokens, most);
        const int64_t rows = (T + n * tokens - 1) / (n * tokens) * (heads / share + TOKEN_ROWS);
        if (rows >= least) continue;
        least = rows;
        best = share;
        *blocks = (int)n;
    }
    return best;
}

// whether rows can be read in runs of n columns: sizes of whole pairs of runs, addresses and strides of whole
// accesses (8 pairs a lane, of 16 columns, measured 60 us beside 56 and 124 beside 122, 16384 x 32 heads of 128)
bool rows_fit(const Params& P, int32_t type, bool bwd, int n) {
    const uintptr_t size = type == CONCORD_F32 ? 4 : 2, access = n * size * (n == 4 && P.interleaved && size == 2 ? 2 : 1);
    uintptr_t all = 0;
    for (const Side& S : P.side) {
        if (S.heads == 0) continue;
        all |= reinterpret_cast<uintptr_t>(S.x) | (uintptr_t)S.ts * size | (uintptr_t)S.hs * size | reinterpret_cast<uintptr_t>(S.out);
        if (bwd) all |= reinterpret_cast<uintptr_t>(S.dy) | (uintptr_t)S.dts * size | (uintptr_t)S.dhs * size;
        if (!aligned(S.w, 4 * n)) return false;
    }
    return P.D % (2 * n) == 0 && P.rot % (2 * n) == 0 && all % access == 0 && aligned(P.cos, 4 * n) && aligned(P.sin, 4 * n);
}

template <typename K> int resident_blocks(K k, size_t smem) {
    int per_sm = 0;
    cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, THREADS, smem) != cudaSuccess || per_sm < 1) {
        cudaGetLastError();
        per_sm = 1;
    }
    int d = 0, sms = 148;
    if (cudaGetDevice(&d) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, d);
    return sms * per_sm;
}

template <typename T, int N, int LANES, Kind KIND, bool NORM> int launch(Params P, bool bwd, float* dqw, float* dkw, cudaStream_t st) {
    using Row = Raw<T, N, KIND>;
    P.lanes = (P.D + 2 * N - 1) / (2 * N);
    const int groups = LANES ? THREADS / (LANES ? LANES : 1) : THREADS / 32 * (32 / P.lanes);
    constexpr size_t ring = Row::ASYNC ? (size_t)RING * THREADS * Row::SLOT : 0, both = NORM ? 2 * ring : ring;
    const size_t smem = !bwd ? ring : both + (NORM && P.part ? (size_t)groups * P.D * sizeof(float) : 0);
    // one wave of blocks, q's and k's by their heads; asked for once a device
    static std::atomic<int> known[2][MAX_DEVICES];
    int d = 0;
    if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= MAX_DEVICES) return fail(CONCORD_ELAUNCH, "concord_qk_norm_rope: no device");
    int most = known[bwd][d].load();
    if (most == 0) {
        most = bwd ? resident_blocks(bwd_kernel<T, N, LANES, KIND, NORM>, both + THREADS * 2 * N * sizeof(float))
                   : resident_blocks(fwd_kernel<T, N, LANES, KIND, NORM>, ring);
        if (most > MAX_BLOCKS) most = MAX_BLOCKS;
        known[bwd][d].store(most);
    }
    int blocks[2];
    const int heads = P.side[0].heads + P.side[1].heads;
    for (int k = 0; k < 2; ++k) {
        Side& S = P.side[k];
        const int64_t part = most * (int64_t)P.side[0].heads / heads;
        blocks[k] = 0;
        S.share = S.heads == 0 ? 1 : share_of(P.T, S.heads, groups, std::max<int64_t>(k ? most - part : part, 1), &blocks[k]);
    }
    P.blocks0 = blocks[0];
    const int all = blocks[0] + blocks[1];
    if (!bwd) {
        fwd_kernel<T, N, LANES, KIND, NORM><<<all, THREADS, smem, st>>>(P);
        return check_launch("concord_qk_norm_rope_fwd");
    }
    bwd_kernel<T, N, LANES, KIND, NORM><<<all, THREADS, smem, st>>>(P);
    if (int rc = check_launch("concord_qk_norm_rope_bwd")) return rc;
    if (NORM && P.part) {
        sum_kernel<<<2 * ((P.D + 7) / 8), 256, 0, st>>>(P.part, blocks[0], all, P.D, dqw, dkw);
        return check_launch("concord_qk_norm_rope_bwd");
    }
    return CONCORD_OK;
}

template <typename T, bool NORM> int run(const Params& P, int32_t type, bool bwd, float* dqw, float* dkw, cudaStream_t st) {
#define QK_LAUNCH(N, LANES)                                                                         \
    return P.interleaved ? launch<T, N, LANES, PAIRED, NORM>(P, bwd, dqw, dkw, st)                 \
                         : launch<T, N, LANES, HALVES, NORM>(P, bwd, dqw, dkw, st)
    if (rows_fit(P, type, bwd, 4)) {              // a lane 8 columns
        // where that makes room for more rows in a warp (64 heads of 32: 25 and 37 us, by 8 lanes 47 and 110; 25 heads of 80, 20011
        // tokens: 36 and 56, by 16 lanes 54 and 98)
        if (P.D <= 48 || (P.D > 64 && P.D <= 80)) QK_LAUNCH(4, 0);
        if (P.D <= 64) QK_LAUNCH(4, 8);
        if (P.D <= 128) QK_LAUNCH(4, 16);
        QK_LAUNCH(4, 32);
    }
    if (P.D <= 128 && rows_fit(P, type, bwd, 2)) {        // a lane 4 (heads of 72, 36 of them turned: 68 and 117 us; through the ring 100 and 174; by
        if (P.D <= 64) QK_LAUNCH(2, 16);                  // single columns 138 and 199, 16384 x 32 heads)
        QK_LAUNCH(2, 32);
    }
    return P.D <= 128 ? launch<T, 2, 32, ANY, NORM>(P, bwd, dqw, dkw, st) : launch<T, 4, 32, ANY, NORM>(P, bwd, dqw, dkw, st);
#undef QK_LAUNCH
}

int dispatch(const Params& P, const concord_qk_params* p, bool bwd, float* dqw, float* dkw, cudaStream_t st) {
    const int32_t t = p->type;
    if (t == CONCORD_F32) return p->norm ? run<float, true>(P, t, bwd, dqw, dkw, st) : run<float, false>(P, t, bwd, dqw, dkw, st);
    if (t == CONCORD_BF16)
        return p->norm ? run<__nv_bfloat16, true>(P, t, bwd, dqw, dkw, st) : run<__nv_bfloat16, false>(P, t, bwd, dqw, dkw, st);
    return p->norm ? run<__half, true>(P, t, bwd, dqw, dkw, st) : run<__half, false>(P, t, bwd, dqw, dkw, st);
}

int check_params(const char* name, const concord_qk_params* p) {
    if (!p || p->type < 0 || p->type > 2) return fail(CONCORD_EINVAL, std::string(name) + ": no parameters, or unknown element type");
    if (!(p->eps >= 0)) return fail(CONCORD_EINVAL, std::string(name) + ": eps must not be negative");
    if (p->tokens < 0 || p->heads < 0 || p->kv_heads < 0 || p->heads + p->kv_heads < 1 || p->head_dim < 1 || p->rot < 0 ||
        p->rot % 2 || p->rot > p->head_dim || (p->rot > 0 && p->positions < 1))
        return fail(CONCORD_ESHAPE, std::string(name) + ": bad extents");
    if (p->head_dim > MAX_DIM || p->heads > 65536 || p->kv_heads > 65536 || p->tokens > (int64_t)1 << 30)
        return fail(CONCORD_ETOOBIG, std::string(name) + ": heads of more than 256, or more than 65536 heads or 2^30 tokens");
    if (p->rot > 0 && (!p->cos || !p->sin)) return fail(CONCORD_EINVAL, std::string(name) + ": null table");
    return CONCORD_OK;
}

Params params(const concord_qk_params* p) {
    Params P{};
    P.cos = p->cos;
    P.sin = p->sin;
    P.pos = p->pos;
    P.pos64 = p->pos64;
    P.T = p->tokens;
    P.positions = p->positions;
    P.side[0].heads = (int)p->heads;
    P.side[1].heads = (int)p->kv_heads;
    P.D = (int)p->head_dim;
    P.rot = (int)p->rot;
    P.interleaved = p->interleaved;
    P.eps = p->eps;
    P.inv_d = 1.f / (float)p->head_dim;
    return P;
}

int operand(const char* name, Side& S, const void* x, int64_t ts, int64_t hs, const float* w, void* out) {
    S.x = x;
    S.ts = ts;
    S.hs = hs;
    S.w = w;
    S.out = out;
    if (S.heads > 0 && !out) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    if (ts < 0 || hs < 0) return fail(CONCORD_ESHAPE, std::string(name) + ": negative stride");
    return CONCORD_OK;
}

}  // namespace qkn
}  // namespace concord

using namespace concord;

extern "C" int concord_qk_norm_rope_fwd(const concord_qk_params* p, const void* q, int64_t q_ts, int64_t q_hs,
                                        const void* k, int64_t k_ts, int64_t k_hs, const float* q_weight,
                                        const float* k_weight, void* q_out, void* k_out, void* stream) {
    const char* name = "concord_qk_norm_rope_fwd";
    if (int rc = qkn::check_params(name, p)) return rc;
    if (p->tokens == 0) return CONCORD_OK;
    qkn::Params P = qkn::params(p);
    if (int rc = qkn::operand(name, P.side[0], q, q_ts, q_hs, q_weight, q_out)) return rc;
    if (int rc = qkn::operand(name, P.side[1], k, k_ts, k_hs, k_weight, k_out)) return rc;
    if ((p->heads && !q) || (p->kv_heads && !k)) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    return qkn::dispatch(P, p, false, nullptr, nullptr, as_stream(stream));
}

extern "C" size_t concord_qk_norm_rope_bwd_workspace_bytes(const concord_qk_params* p) {
    if (qkn::check_params("concord_qk_norm_rope_bwd_workspace_bytes", p) || !p->norm || p->tokens == 0) return 0;
    return (size_t)(qkn::MAX_BLOCKS + 2) * p->head_dim * sizeof(float);
}

extern "C" int concord_qk_norm_rope_bwd(const concord_qk_params* p, const void* q, int64_t q_ts, int64_t q_hs,
                                        const void* k, int64_t k_ts, int64_t k_hs, const float* q_weight,
                                        const float* k_weight, const void* dq_out, int64_t dq_ts, int64_t dq_hs,
                                        const void* dk_out, int64_t dk_ts, int64_t dk_hs, void* dq, void* dk,
                                        float* dq_weight, float* dk_weight, void* workspace, size_t workspace_bytes,
                                        void* stream) {
    const char* name = "concord_qk_norm_rope_bwd";
    if (int rc = qkn::check_params(name, p)) return rc;
    cudaStream_t st = as_stream(stream);
    const bool weights = p->norm && (dq_weight || dk_weight);
    if (p->tokens == 0) {
        if (weights && dq_weight) cudaMemsetAsync(dq_weight, 0, p->head_dim * sizeof(float), st);
        if (weights && dk_weight) cudaMemsetAsync(dk_weight, 0, p->head_dim * sizeof(float), st);
        return check_launch(name);
    }
    qkn::Params P = qkn::params(p);
    if (int rc = qkn::operand(name, P.side[0], q, q_ts, q_hs, q_weight, dq)) return rc;
    if (int rc = qkn::operand(name, P.side[1], k, k_ts, k_hs, k_weight, dk)) return rc;
    if ((p->heads && (!dq_out || (p->norm && !q))) || (p->kv_heads && (!dk_out || (p->norm && !k))))
        return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    if (dq_ts < 0 || dq_hs < 0 || dk_ts < 0 || dk_hs < 0) return fail(CONCORD_ESHAPE, std::string(name) + ": negative stride");
    P.side[0].dy = dq_out;
    P.side[0].dts = dq_ts;
    P.side[0].dhs = dq_hs;
    P.side[1].dy = dk_out;
    P.side[1].dts = dk_ts;
    P.side[1].dhs = dk_hs;
    if (weights) {
        if (!workspace || workspace_bytes < concord_qk_norm_rope_bwd_workspace_bytes(p))
            return fail(CONCORD_EWORKSPACE, std::string(name) + ": workspace too small");
        P.part = static_cast<float*>(workspace);
    }
    return qkn::dispatch(P, p, true, dq_weight, dk_weight, st);
}
