// norm.cu — layer norm over the last dimension, forward and backward.
//
//   y  = (x - mean) rstd w + b,           rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)),  g = dy w, xh = (x - mean) rstd
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Bound by memory: the forward reads x and writes y once, the backward reads
// x and dy and writes dx once.  A row stays in the registers of the threads
// that own it (16 elements each: 32 threads up to 512 columns, 1024 at the
// largest width), so the variance is the mean of squared deviations from the
// finished mean and nothing is read twice.  The grid is one wave of resident
// blocks that walk the rows; each thread keeps its columns' weight, and in the
// backward its columns' sums of dy xh and dy, from row to row.  The blocks'
// sums are added in block order by a second kernel: no atomics, so the
// gradients are the same bits on every run of one device.
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
    const float2 s = lane < nw ? r[w0 + lane] : make_float2(0.f, 0.f);
    a = warp_sum(s.x);
    if (NB == 2) b = warp_sum(s.y);
}

template <typename TX, typename TY, int VEC>
__global__ void __launch_bounds__(1024)
    fwd_kernel(const TX* __restrict__ x, int64_t ldx, const float* __restrict__ w, const float* __restrict__ b,
               TY* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, int64_t N, int D, float eps,
               int tpr) {
    constexpr int NV = PER / VEC;
    __shared__ float2 red[64];
    int turn = 0;
    const int t = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const float inv = 1.0f / (float)D;
    float wv[PER], bv[PER];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * tpr + t) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            wv[i * VEC + j] = w && c + j < D ? w[c + j] : 1.0f;
            bv[i * VEC + j] = b && c + j < D ? b[c + j] : 0.0f;
        }
    }
    for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < N; r0 += (int64_t)gridDim.x * groups) {
        const int64_t row = r0 + group;
        const bool live = row < N;
        float v[PER];
        float sum = 0.f, none = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + t) * VEC;
            if (live && c < D) load_vec<VEC>(x + row * ldx + c, v + i * VEC);
            else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[i * VEC + j] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += v[i];
        row_sum<1>(sum, none, tpr, red, turn);
        const float mu = sum * inv;
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((i * tpr + t) * VEC < D) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    v[i * VEC + j] -= mu;
                    sq += v[i * VEC + j] * v[i * VEC + j];
                }
            }
        }
        row_sum<1>(sq, none, tpr, red, turn);
        const float rs = 1.0f / sqrtf(sq * inv + eps);
        if (live) {
            if (mean && t == 0) {
                mean[row] = mu;
                rstd[row] = rs;
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * tpr + t) * VEC;
                if (c < D) {
                    float o[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o[j] = v[i * VEC + j] * rs * wv[i * VEC + j] + bv[i * VEC + j];
                    store_vec<VEC>(y + row * D + c, o);
                }
            }
        }
    }
}

// dx, and this block's column sums to part[block][0: dy xh, 1: dy][D].  WIDE
// (above 8192 columns, 1024 threads of at most 64 registers): the column sums
// live in the thread's own shared-memory slots instead of its registers.
template <typename TX, typename TY, int VEC, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 1024 : 512)
    bwd_kernel(const TX* __restrict__ x, int64_t ldx, const TY* __restrict__ dy, int64_t lddy,
               const float* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
               TX* __restrict__ dx, float* __restrict__ part, int64_t N, int D, int tpr) {
    constexpr int NV = PER / VEC;
    extern __shared__ float dyn[];               // WIDE: 2 * PER * blockDim sums; else groups * D * 2 at the end
    __shared__ float2 red[64];
    int turn = 0;
    const int t = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const float inv = 1.0f / (float)D;
    float aw[WIDE ? 1 : PER], ab[WIDE ? 1 : PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if constexpr (WIDE) { dyn[i * 1024 + threadIdx.x] = 0.f; dyn[(PER + i) * 1024 + threadIdx.x] = 0.f; }
        else { aw[i] = 0.f; ab[i] = 0.f; }
    }
    for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < N; r0 += (int64_t)gridDim.x * groups) {
        const int64_t row = r0 + group;
        const bool live = row < N;
        const float mu = live ? mean[row] : 0.f, rs = live ? rstd[row] : 0.f;
        float xh[PER], g[PER];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + t) * VEC;
            if (live && c < D) {
                load_vec<VEC>(x + row * ldx + c, xh + i * VEC);
                load_vec<VEC>(dy + row * lddy + c, g + i * VEC);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) { xh[i * VEC + j] = mu; g[i * VEC + j] = 0.f; }
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + t) * VEC;
            float wv[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) wv[j] = 1.0f;
            if (w && c < D) load_vec<VEC>(w + c, wv);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int e = i * VEC + j;
                xh[e] = (xh[e] - mu) * rs;
                if constexpr (WIDE) {
                    dyn[e * 1024 + threadIdx.x] += g[e] * xh[e];
                    dyn[(PER + e) * 1024 + threadIdx.x] += g[e];
                } else {
                    aw[e] += g[e] * xh[e];
                    ab[e] += g[e];
                }
                g[e] *= wv[j];
                s1 += g[e];
                s2 += g[e] * xh[e];
            }
        }
        row_sum<2>(s1, s2, tpr, red, turn);
        s1 *= inv;
        s2 *= inv;
        if (live) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * tpr + t) * VEC;
                if (c < D) {
                    float o[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o[j] = rs * (g[i * VEC + j] - s1 - xh[i * VEC + j] * s2);
                    store_vec<VEC>(dx + row * D + c, o);
                }
            }
        }
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
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int c = ((e / VEC) * tpr + t) * VEC + e % VEC;
            if (c < D) { dyn[group * 2 * D + c] = aw[e]; dyn[group * 2 * D + D + c] = ab[e]; }
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

// blocks of the backward: one wave of 512 threads per SM (1024 where a row takes 1024)
int bwd_blocks(int64_t N, int64_t D, int* threads) {
    const int tpr = threads_per_row(D);
    *threads = tpr > 256 ? tpr : 256;
    const int64_t groups = *threads / tpr, need = (N + groups - 1) / groups;
    const int64_t wave = (int64_t)sm_count() * (*threads >= 512 ? 1 : 512 / *threads);
    return (int)(need < wave ? need : wave);
}

template <typename TX, typename TY>
int forward(const void* x, int64_t ldx, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t N,
            int64_t D, float eps, bool vec, cudaStream_t st) {
    const int tpr = threads_per_row(D), threads = tpr > 256 ? tpr : 256;
    const int64_t groups = threads / tpr, need = (N + groups - 1) / groups;
    const int64_t wave = (int64_t)sm_count() * (1024 / threads);
    const int grid = (int)(need < wave ? need : wave);
    auto k = vec ? fwd_kernel<TX, TY, 8> : fwd_kernel<TX, TY, 1>;
    k<<<grid, threads, 0, st>>>(static_cast<const TX*>(x), ldx, w, b, static_cast<TY*>(y), mean, rstd, N, (int)D, eps,
                                tpr);
    return check_launch("concord_layer_norm_fwd");
}

template <typename TX, typename TY>
int backward(const void* x, int64_t ldx, const void* dy, int64_t lddy, const float* w, const float* mean,
             const float* rstd, void* dx, float* dw, float* db, int64_t N, int64_t D, bool vec, float* part,
             cudaStream_t st) {
    int threads = 0;
    const int grid = bwd_blocks(N, D, &threads), tpr = threads_per_row(D);
    const bool wide = tpr == 1024;
    const size_t smem = wide ? 2 * PER * 1024 * sizeof(float) : (size_t)(threads / tpr) * 2 * D * sizeof(float);
    auto k = wide ? (vec ? bwd_kernel<TX, TY, 8, true> : bwd_kernel<TX, TY, 1, true>)
                  : (vec ? bwd_kernel<TX, TY, 8, false> : bwd_kernel<TX, TY, 1, false>);
    if (smem > 48 * 1024) {
        // 128 KB at most; set on every call that needs it (the attribute is per device and idempotent)
        cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail(CONCORD_ELAUNCH, std::string("concord_layer_norm_bwd: ") + cudaGetErrorString(e));
    }
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
    const bool vec = D % 8 == 0 && ldx * norm::esize(x_type) % 16 == 0 && aligned(x, 16) && aligned(y, 16);
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
                     aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16) && (!w || aligned(w, 16));
    NORM_TYPES(x_type, dy_type, norm::backward, x, ldx, dy, lddy, w, mean, rstd, dx, dw, db, N, D, vec,
               static_cast<float*>(workspace), st)
}
