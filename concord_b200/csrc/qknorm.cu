// qknorm.cu — root-mean-square norm of every query and key head with the
// position rotation in the same pass, and the gradient of both.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w            (n = x without the norm)
//   (a, b) -> (a c - b s, a s + b c)                      for every rotated pair of n, c and s of the token's position
//   backward: dn = the rotation undone on dy,  g = dn w,
//   dx = r g - x r^3 sum(g x) / D,  dw = sum over tokens and heads of dn x r
//
// Bound by memory: the forward reads and writes q and k once, the backward
// reads dy and x and writes dx.  A row (one head of one token) stays in the
// registers of a group of lanes, 8 pairs each, a pair's two halves in one lane
// whichever way pairs are laid out, so that the rotation needs no exchange; the
// group's lanes share sums by shuffles (both sums of the backward in one go:
// neither needs r).  A thread keeps its part of cos and sin for all heads of a
// token, and its columns' weights for all tokens.  The weights' gradients are
// added per thread, then per block, then over blocks in a fixed order: no
// atomics, the same bits on every run of one device.
#include "common.cuh"
#include "vec.cuh"

namespace concord {
namespace qkn {

constexpr int MAX_DIM = 256, THREADS = 256;

struct Params {
    const float *cos, *sin;       // [positions, rot / 2]
    const void* pos;              // [T], or NULL: the token's number
    int pos64;
    int64_t T, positions;
    int heads[2], D, rot;         // heads of q and of k
    int interleaved;
    float eps, inv_d;
    const float* w[2];            // NULL: ones
    const void* x[2];
    int64_t ts[2], hs[2];         // token and head strides, elements
    const void* dy[2];
    int64_t dts[2], dhs[2];
    void* out[2];                 // contiguous [T, heads, D]
    float* part;                  // backward: [blocks][2][D]
    int share;                    // row groups of a block that share a token's heads
};

// What one lane holds of a row: PAIRS pairs (a, b).  VEC: 8 pairs, rotated ones or 16
// neighbouring plain columns; else 4 pairs 32 apart, for any size and stride.
template <bool VEC> struct Lane {
    static constexpr int PAIRS = VEC ? 8 : 4;
    int at[VEC ? 2 : 1];          // VEC: the first columns of two runs of 8; else the first pair
    bool live, turns;             // VEC: any columns, rotated ones
    int D, rot, interleaved;
    __device__ __forceinline__ Lane(const Params& P, int lane) : D(P.D), rot(P.rot), interleaved(P.interleaved) {
        if constexpr (VEC) {
            live = lane * 16 < D;
            turns = lane * 16 < rot;
            at[0] = turns && !interleaved ? lane * 8 : lane * 16;
            at[1] = turns && !interleaved ? rot / 2 + lane * 8 : lane * 16 + 8;
        } else {
            live = turns = true;
            at[0] = lane;
        }
    }
    // pair j's columns (not VEC); -1: none
    __device__ __forceinline__ void columns(int j, int* a, int* b) const {
        const int p = at[0] + 32 * j, half = rot / 2;
        if (p < half) {
            *a = interleaved ? 2 * p : p;
            *b = interleaved ? 2 * p + 1 : half + p;
        } else {
            *a = rot + 2 * (p - half);
            *b = *a + 1;
        }
        if (*a >= D) *a = -1;
        if (*b >= D) *b = -1;
    }
    template <typename T> __device__ __forceinline__ void load(const T* row, float* a, float* b) const {
        if constexpr (VEC) {
            load_vec<8>(row + at[0], a);
            load_vec<8>(row + at[1], b);
            if (interleaved && turns) {           // (a0 b0 a1 b1 ..) to (a0 a1 ..), (b0 b1 ..)
                float t[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) { t[j] = a[2 * j + 1]; a[j] = a[2 * j]; }
#pragma unroll
                for (int j = 0; j < 4; ++j) { a[4 + j] = b[2 * j]; t[4 + j] = b[2 * j + 1]; }
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = t[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
                int ca, cb;
                columns(j, &ca, &cb);
                a[j] = ca >= 0 ? to_f32(row[ca]) : 0.f;
                b[j] = cb >= 0 ? to_f32(row[cb]) : 0.f;
            }
        }
    }
    template <typename T> __device__ __forceinline__ void store(T* row, const float* a, const float* b) const {
        if constexpr (VEC) {
            if (interleaved && turns) {
                float lo[8], hi[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    lo[2 * j] = a[j];
                    lo[2 * j + 1] = b[j];
                    hi[2 * j] = a[4 + j];
                    hi[2 * j + 1] = b[4 + j];
                }
                store_vec<8>(row + at[0], lo);
                store_vec<8>(row + at[1], hi);
            } else {
                store_vec<8>(row + at[0], a);
                store_vec<8>(row + at[1], b);
            }
        } else {
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
                int ca, cb;
                columns(j, &ca, &cb);
                if (ca >= 0) row[ca] = from_f32<T>(a[j]);
                if (cb >= 0) row[cb] = from_f32<T>(b[j]);
            }
        }
    }
    __device__ __forceinline__ bool rotated(int j) const { return VEC ? turns : at[0] + 32 * j < rot / 2; }
    // cos and sin of token t's position; NaN where the tables have no such position
    __device__ __forceinline__ void angles(const Params& P, int64_t t, float* c, float* s) const {
        int64_t p = t;
        if (P.pos && rot) p = P.pos64 ? static_cast<const int64_t*>(P.pos)[t] : (int64_t)static_cast<const int32_t*>(P.pos)[t];
        const bool there = p >= 0 && p < P.positions;
        const int64_t row = p * (rot / 2);
        if constexpr (VEC) {
            if (live && turns && there) {
                load_vec<8>(P.cos + row + at[0] / (interleaved ? 2 : 1), c);
                load_vec<8>(P.sin + row + at[0] / (interleaved ? 2 : 1), s);
                return;
            }
        }
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            const bool here = !VEC && rotated(j) && there;
            c[j] = here ? P.cos[row + at[0] + 32 * j] : __int_as_float(0x7fffffff);
            s[j] = here ? P.sin[row + at[0] + 32 * j] : c[j];
        }
    }
};

// the sum over a row's lanes (a power of two of them)
template <bool VEC> __device__ __forceinline__ float lane_sum(float v, int lanes) {
    for (int o = (VEC ? lanes : 32) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// HEADS rows of a thread at a time, so that their loads are on their way together
constexpr int AHEAD = 4;

template <typename T, bool VEC, bool NORM>
__global__ void __launch_bounds__(THREADS) fwd_kernel(const __grid_constant__ Params P, int lanes) {
    constexpr int N = Lane<VEC>::PAIRS;
    const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = THREADS / lanes;
    const Lane<VEC> L(P, lane);
    const int64_t step = (int64_t)gridDim.x * (groups / P.share);
    // every thread of a warp goes round the same number of times (the sums are whole warps')
    const int64_t t0 = (int64_t)blockIdx.x * (groups / P.share), mine = group / P.share;
    for (int64_t base = t0; base < P.T; base += step) {
        const int64_t t = base + mine;
        const bool here = t < P.T && L.live;
        float c[N], s[N];
        L.angles(P, here ? t : base, c, s);
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
            const int heads = P.heads[which];
            const T* x = static_cast<const T*>(P.x[which]) + t * P.ts[which];
            T* out = static_cast<T*>(P.out[which]) + t * heads * P.D;
            float wa[N], wb[N];
#pragma unroll
            for (int j = 0; j < N; ++j) wa[j] = wb[j] = 1.f;
            if (NORM && P.w[which] && L.live) L.load(P.w[which], wa, wb);
#pragma unroll 1
            for (int h0 = group & (P.share - 1); h0 - (group & (P.share - 1)) < heads; h0 += AHEAD * P.share) {
                float a[AHEAD][N], b[AHEAD][N];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int h = h0 + i * P.share;
                    if (here && h < heads) L.load(x + h * P.hs[which], a[i], b[i]);
                }
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int h = h0 + i * P.share;
                    const bool row = here && h < heads;
                    if constexpr (NORM) {
                        float ss = 0.f;
                        if (row) {
#pragma unroll
                            for (int j = 0; j < N; ++j) ss += a[i][j] * a[i][j] + b[i][j] * b[i][j];
                        }
                        ss = lane_sum<VEC>(ss, lanes);
                        const float r = rsqrtf(ss * P.inv_d + P.eps);
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            a[i][j] *= r * wa[j];
                            b[i][j] *= r * wb[j];
                        }
                    }
                    if (!row) continue;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        if (!L.rotated(j)) continue;
                        const float u = a[i][j], v = b[i][j];
                        a[i][j] = u * c[j] - v * s[j];
                        b[i][j] = u * s[j] + v * c[j];
                    }
                    L.store(out + h * P.D, a[i], b[i]);
                }
            }
        }
    }
}

template <typename T, bool VEC, bool NORM>
__global__ void __launch_bounds__(THREADS) bwd_kernel(const __grid_constant__ Params P, int lanes) {
    constexpr int N = Lane<VEC>::PAIRS, AHEAD = 2;
    extern __shared__ float sums[];               // [row groups][2][D]
    const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = THREADS / lanes;
    const Lane<VEC> L(P, lane);
    const int64_t step = (int64_t)gridDim.x * (groups / P.share);
    const int64_t t0 = (int64_t)blockIdx.x * (groups / P.share), mine = group / P.share;
    float ga[2][N], gb[2][N];                     // this thread's part of the weights' gradients
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) ga[k][j] = gb[k][j] = 0.f;
    for (int64_t base = t0; base < P.T; base += step) {
        const int64_t t = base + mine;
        const bool here = t < P.T && L.live;
        float c[N], s[N];
        L.angles(P, here ? t : base, c, s);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int heads = P.heads[which];
            const T* x = static_cast<const T*>(P.x[which]) + t * P.ts[which];
            const T* dy = static_cast<const T*>(P.dy[which]) + t * P.dts[which];
            T* out = static_cast<T*>(P.out[which]) + t * heads * P.D;
            float wa[N], wb[N];
#pragma unroll
            for (int j = 0; j < N; ++j) wa[j] = wb[j] = 1.f;
            if (NORM && P.w[which] && L.live) L.load(P.w[which], wa, wb);
#pragma unroll 1
            for (int h0 = group & (P.share - 1); h0 - (group & (P.share - 1)) < heads; h0 += AHEAD * P.share) {
                float a[AHEAD][N], b[AHEAD][N], xa[AHEAD][N], xb[AHEAD][N];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int h = h0 + i * P.share;
                    if (here && h < heads) {
                        L.load(dy + h * P.dhs[which], a[i], b[i]);
                        if (NORM) L.load(x + h * P.hs[which], xa[i], xb[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int h = h0 + i * P.share;
                    const bool row = here && h < heads;
                    if (row) {
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            if (!L.rotated(j)) continue;
                            const float u = a[i][j], v = b[i][j];
                            a[i][j] = u * c[j] + v * s[j];
                            b[i][j] = v * c[j] - u * s[j];
                        }
                    }
                    if constexpr (NORM) {
                        float ss = 0.f, gx = 0.f;
                        if (row) {
#pragma unroll
                            for (int j = 0; j < N; ++j) {
                                ss += xa[i][j] * xa[i][j] + xb[i][j] * xb[i][j];
                                gx += a[i][j] * wa[j] * xa[i][j] + b[i][j] * wb[j] * xb[i][j];
                            }
                        }
                        ss = lane_sum<VEC>(ss, lanes);
                        gx = lane_sum<VEC>(gx, lanes);
                        const float r = rsqrtf(ss * P.inv_d + P.eps), m = r * r * gx * P.inv_d;
                        if (row) {
#pragma unroll
                            for (int j = 0; j < N; ++j) {
                                ga[which][j] += a[i][j] * (xa[i][j] * r);
                                gb[which][j] += b[i][j] * (xb[i][j] * r);
                                a[i][j] = r * (a[i][j] * wa[j] - xa[i][j] * m);
                                b[i][j] = r * (b[i][j] * wb[j] - xb[i][j] * m);
                            }
                        }
                    }
                    if (row) L.store(out + h * P.D, a[i], b[i]);
                }
            }
        }
    }
    if (NORM && P.part) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (L.live) L.store(sums + (group * 2 + k) * P.D, ga[k], gb[k]);
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * P.D; i += THREADS) {
            float v = sums[i];
            for (int g = 1; g < groups; ++g) v += sums[g * 2 * P.D + i];
            P.part[(int64_t)blockIdx.x * 2 * P.D + i] = v;
        }
    }
}

// the blocks' sums in a fixed order: 8 columns x 32 strides a block
__global__ void __launch_bounds__(256) sum_kernel(const float* part, int blocks, int D, float* dqw, float* dkw) {
    __shared__ float red[32][9];
    const int cx = threadIdx.x & 7, ry = threadIdx.x >> 3, c = blockIdx.x * 8 + cx;
    float v = 0.f;
    if (c < 2 * D) {
#pragma unroll 4
        for (int k = ry; k < blocks; k += 32) v += part[(int64_t)k * 2 * D + c];
    }
    red[ry][cx] = v;
    __syncthreads();
    if (ry == 0 && c < 2 * D) {
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) v += red[k][cx];
        float* out = c < D ? dqw : dkw;
        if (out) out[c < D ? c : c - D] = v;
    }
}

// ---------------------------------------------------------------- host side
constexpr int MAX_BLOCKS = 148 * 4;       // of the backward, whose blocks each leave a row of sums

int lanes_of(int64_t D, bool vec) {
    if (!vec) return 32;
    int n = 1;
    while (n * 16 < D) n *= 2;
    return n;
}

// Groups of a block that share a token: few where tokens are many (cos and sin
// are then read once for more heads, weights stay), all heads' side by side
// where they would not fill the GPU.
int share_of(int64_t T, int heads, int groups) {
    int share = 1;
    while (share < groups && share < heads && (share < 4 || T * share < (int64_t)groups * 148 * 4)) share *= 2;
    return share;
}

bool vec_of(const Params& P, const concord_qk_params* p, bool bwd) {
    const int per = p->type == CONCORD_F32 ? 4 : 8;
    bool ok = P.D % 16 == 0 && P.rot % 16 == 0 && aligned(P.cos, 16) && aligned(P.sin, 16);
    for (int k = 0; k < 2; ++k) {
        if (P.heads[k] == 0) continue;
        ok = ok && aligned(P.x[k], 16) && P.ts[k] % per == 0 && P.hs[k] % per == 0 && aligned(P.out[k], 16) &&
             aligned(P.w[k], 16);
        if (bwd) ok = ok && aligned(P.dy[k], 16) && P.dts[k] % per == 0 && P.dhs[k] % per == 0;
    }
    return ok;
}

int64_t blocks_of(const Params& P, int lanes, int share, bool bwd) {
    const int64_t tokens = THREADS / lanes / share, need = (P.T + tokens - 1) / tokens;
    const int64_t most = bwd ? MAX_BLOCKS : 148 * 16;
    return need < most ? need : most;
}

template <typename T, bool VEC, bool NORM> int launch(Params P, bool bwd, cudaStream_t st) {
    const int lanes = lanes_of(P.D, VEC), groups = THREADS / lanes;
    P.share = share_of(P.T, P.heads[0] > P.heads[1] ? P.heads[0] : P.heads[1], groups);
    const int blocks = (int)blocks_of(P, lanes, P.share, bwd);
    if (!bwd) {
        fwd_kernel<T, VEC, NORM><<<blocks, THREADS, 0, st>>>(P, lanes);
        return check_launch("concord_qk_norm_rope_fwd");
    }
    const size_t smem = NORM && P.part ? (size_t)groups * 2 * P.D * sizeof(float) : 0;
    bwd_kernel<T, VEC, NORM><<<blocks, THREADS, smem, st>>>(P, lanes);
    return check_launch("concord_qk_norm_rope_bwd");
}

template <typename T> int run(const Params& P, bool vec, bool norm, bool bwd, cudaStream_t st) {
    if (vec) return norm ? launch<T, true, true>(P, bwd, st) : launch<T, true, false>(P, bwd, st);
    return norm ? launch<T, false, true>(P, bwd, st) : launch<T, false, false>(P, bwd, st);
}

int dispatch(const Params& P, const concord_qk_params* p, bool bwd, cudaStream_t st) {
    const bool vec = vec_of(P, p, bwd);
    if (p->type == CONCORD_F32) return run<float>(P, vec, p->norm != 0, bwd, st);
    if (p->type == CONCORD_BF16) return run<__nv_bfloat16>(P, vec, p->norm != 0, bwd, st);
    return run<__half>(P, vec, p->norm != 0, bwd, st);
}

int check_params(const char* name, const concord_qk_params* p) {
    if (!p || p->type < 0 || p->type > 2) return fail(CONCORD_EINVAL, std::string(name) + ": no parameters, or unknown element type");
    if (!(p->eps >= 0)) return fail(CONCORD_EINVAL, std::string(name) + ": eps must not be negative");
    if (p->tokens < 0 || p->heads < 0 || p->kv_heads < 0 || p->heads + p->kv_heads < 1 || p->head_dim < 1 || p->rot < 0 ||
        p->rot % 2 || p->rot > p->head_dim || (p->rot > 0 && p->positions < 1))
        return fail(CONCORD_ESHAPE, std::string(name) + ": bad extents");
    if (p->head_dim > MAX_DIM || p->heads > 65536 || p->kv_heads > 65536 || p->tokens > (int64_t)1 << 40)
        return fail(CONCORD_ETOOBIG, std::string(name) + ": heads of more than 256, or more than 65536 heads or 2^40 tokens");
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
    P.heads[0] = (int)p->heads;
    P.heads[1] = (int)p->kv_heads;
    P.D = (int)p->head_dim;
    P.rot = (int)p->rot;
    P.interleaved = p->interleaved;
    P.eps = p->eps;
    P.inv_d = 1.f / (float)p->head_dim;
    return P;
}

int operand(const char* name, Params& P, int k, const void* x, int64_t ts, int64_t hs, const float* w, void* out) {
    P.x[k] = x;
    P.ts[k] = ts;
    P.hs[k] = hs;
    P.w[k] = w;
    P.out[k] = out;
    if (P.heads[k] > 0 && !out) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
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
    if (int rc = qkn::operand(name, P, 0, q, q_ts, q_hs, q_weight, q_out)) return rc;
    if (int rc = qkn::operand(name, P, 1, k, k_ts, k_hs, k_weight, k_out)) return rc;
    if ((p->heads && !q) || (p->kv_heads && !k)) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    return qkn::dispatch(P, p, false, as_stream(stream));
}

extern "C" size_t concord_qk_norm_rope_bwd_workspace_bytes(const concord_qk_params* p) {
    if (qkn::check_params("concord_qk_norm_rope_bwd_workspace_bytes", p) || !p->norm || p->tokens == 0) return 0;
    return (size_t)qkn::MAX_BLOCKS * 2 * p->head_dim * sizeof(float);
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
    if (int rc = qkn::operand(name, P, 0, q, q_ts, q_hs, q_weight, dq)) return rc;
    if (int rc = qkn::operand(name, P, 1, k, k_ts, k_hs, k_weight, dk)) return rc;
    if ((p->heads && (!dq_out || (p->norm && !q))) || (p->kv_heads && (!dk_out || (p->norm && !k))))
        return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    if (dq_ts < 0 || dq_hs < 0 || dk_ts < 0 || dk_hs < 0) return fail(CONCORD_ESHAPE, std::string(name) + ": negative stride");
    P.dy[0] = dq_out;
    P.dts[0] = dq_ts;
    P.dhs[0] = dq_hs;
    P.dy[1] = dk_out;
    P.dts[1] = dk_ts;
    P.dhs[1] = dk_hs;
    if (weights) {
        if (!workspace || workspace_bytes < concord_qk_norm_rope_bwd_workspace_bytes(p))
            return fail(CONCORD_EWORKSPACE, std::string(name) + ": workspace too small");
        P.part = static_cast<float*>(workspace);
    }
    if (int rc = qkn::dispatch(P, p, true, st)) return rc;
    if (weights) {
        const bool vec = qkn::vec_of(P, p, true);
        const int lanes = qkn::lanes_of(P.D, vec), groups = qkn::THREADS / lanes;
        const int share = qkn::share_of(P.T, P.heads[0] > P.heads[1] ? P.heads[0] : P.heads[1], groups);
        qkn::sum_kernel<<<(2 * P.D + 7) / 8, 256, 0, st>>>(P.part, (int)qkn::blocks_of(P, lanes, share, true), P.D,
                                                           dq_weight, dk_weight);
        return check_launch(name);
    }
    return CONCORD_OK;
}
