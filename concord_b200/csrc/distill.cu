// distill.cu — distillation from a teacher's top logits: loss and gradient.
//
// Student logits z [N, V], the teacher's K best ids and logits t per row (an
// id outside [0, V) or a logit of -inf is an absent entry), hard labels y:
//   p    = softmax(t / T) over the entries present
//   KL_n = sum_k p_k (log p_k - z_k / T + lse(z / T)),  CE_n = lse(z) - z_y
//   loss = sum over the rows that count of (a T^2 KL_n + (1 - a) CE_n) [/ their number]
//   dz   = a T (softmax(z / T) - p) + (1 - a) (softmax(z) - e_y)      [/ their number]
// With labels a row counts where its label is in [0, V) and not the ignored
// one; without them, where the teacher has an entry.  A row that does not
// count has loss 0 and gradient 0, whatever its logits hold.
//
// Bound by memory, near the rate of the exponentials: a row is read once for
// its maximum and sums (one running maximum, one or two sums), and once more
// while it is still in the L2 to write dz, so the HBM sees z once and dz once.
// Where T is a power of two, exp(z) is exp(z / T) squared log2(T) times
// (relative error T times that of one exponential), which halves the
// exponentials.  A row belongs to 32 to 1024 threads of a block, by its
// length.  The K teacher entries and the label touch few places of dz: their
// owners write those again from fp32 after the dense pass, each from all
// entries with that id in entry order, so nothing is added atomically.
#include <float.h>
#include <math.h>

#include "common.cuh"
#include "vec.cuh"

namespace concord {
namespace distill {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_K = 512;
constexpr int COUNT_BLOCKS = 128;

struct Args {
    const void* z;
    int64_t ldz;
    const void* ids;
    const float* t;
    const void* labels;
    int64_t ignore;
    int ids64, labels64;
    int K;
    int64_t N;
    int64_t V;
    float temp, alpha, gscale;
    const float* gout;      // upstream gradient: one value (gout_stride 0) or one per row (1)
    int gout_stride;
    int mean;               // divide by the number of rows that count
    const int* counts;      // [COUNT_BLOCKS] partial counts (value and gradient in one pass)
    const float* number;    // the number of rows that count, from the forward (gradient alone)
    float* stats;           // [N, 3]: maximum, sum at 1/T, sum at 1
    float* row_loss;        // [N]
    float* row_counts;      // [N]: 1 where the row counts
    void* dz;
    int squarings;          // log2(T) where T = 2, 4, 8
    int tpr;
};

__device__ __forceinline__ int64_t entry(const void* p, int is64, int64_t i) {
    return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ bool label_counts(const Args& A, int64_t y) { return y != A.ignore && y >= 0 && y < A.V; }

__device__ __forceinline__ bool entry_counts(const Args& A, int64_t id, float t) {
    return id >= 0 && id < A.V && !(t == -INFINITY);
}

// rows that count, one partial number per block (whole numbers: any order gives the same)
__global__ void __launch_bounds__(256) count_kernel(const Args A, int* counts) {
    __shared__ int red[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int n = 0;
    if (A.labels) {
        for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < A.N; r += (int64_t)gridDim.x * 256)
            n += label_counts(A, entry(A.labels, A.labels64, r));
        n = __reduce_add_sync(0xffffffffu, n);
    } else {
        for (int64_t r = (int64_t)blockIdx.x * 8 + warp; r < A.N; r += (int64_t)gridDim.x * 8) {
            bool any = false;
            for (int k = lane; k < A.K && !any; k += 32)
                any = entry_counts(A, entry(A.ids, A.ids64, r * A.K + k), A.t[r * A.K + k]);
            n += __any_sync(0xffffffffu, any);
        }
    }
    if (lane == 0) red[warp] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        n = 0;
        for (int i = 0; i < 8; ++i) n += red[i];
        counts[blockIdx.x] = n;
    }
}

// the number of rows that count, known to every lane
__device__ __forceinline__ int total_count(const Args& A) {
    const int lane = threadIdx.x & 31;
    int n = 0;
#pragma unroll
    for (int i = 0; i < COUNT_BLOCKS / 32; ++i) n += A.counts[i * 32 + lane];
    return __reduce_add_sync(0xffffffffu, n);
}

// running maximum with the sums of exp((z - m) / T) and exp(z - m)
struct Run {
    float m, s, s1;
};

template <bool TWO>
__device__ __forceinline__ void merge(Run& a, float m, float s, float s1, float c, float c1) {
    const float top = fmaxf(a.m, m), ref = top == -INFINITY ? 0.f : top;
    a.s = a.s * ex2f((a.m - ref) * c) + s * ex2f((m - ref) * c);
    if (TWO) a.s1 = a.s1 * ex2f((a.m - ref) * c1) + s1 * ex2f((m - ref) * c1);
    a.m = top;
}

template <bool TWO> struct Exps {
    float c, c1;
    int squarings;
    // exp((z - m) / T) and exp(z - m); the difference first, so that rows of the
    // type's lowest value, or of 1e4 and more, lose nothing in a product
    __device__ __forceinline__ void at(float z, float m, float& e, float& e1) const {
        const float d = z - m;
        e = ex2f(d * c);
        if (TWO) {
            if (squarings) {
                e1 = e * e;
                if (squarings > 1) e1 *= e1;
                if (squarings > 2) e1 *= e1;
            } else e1 = ex2f(d * c1);
        }
    }
};

template <bool TWO, int NE>
__device__ __forceinline__ void take(Run& r, const float* v, const Exps<TWO>& X) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < NE; ++i) top = fmaxf(top, v[i]);
    if (top > r.m) {
        const float old = r.m;          // -inf at first: exp gives 0
        r.s *= ex2f((old - top) * X.c);
        if (TWO) r.s1 *= ex2f((old - top) * X.c1);
        r.m = top;
    }
    const float ref = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        float e, e1;
        X.at(v[i], ref, e, e1);
        r.s += e;
        if (TWO) r.s1 += e1;
    }
}

// T: logits' type; TWO: both temperatures are needed; MODE 1: statistics and
// loss, 2: gradient from given statistics, 3: both
template <typename T, bool TWO, int MODE>
__global__ void __launch_bounds__(1024) row_kernel(const Args A) {
    constexpr int W = Pack16<T>::N;
    extern __shared__ float dyn[];       // groups x (K probabilities, K ids)
    __shared__ float red[32][3];
    __shared__ float shared_row[32][4];
    const int tpr = A.tpr, t = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = tpr >> 5;
    float* prob = dyn + (size_t)group * 2 * A.K;
    int* pid = reinterpret_cast<int*>(prob + A.K);
    Exps<TWO> X;
    X.c = LOG2E / A.temp;
    X.c1 = LOG2E;
    X.squarings = A.squarings;
    float number = 1.f;
    if (MODE == 3 && A.mean) number = (float)max(1, total_count(A));
    if (MODE == 2 && A.mean) number = *A.number;

    auto sync = [&]() { if (tpr == 32) __syncwarp(); else __syncthreads(); };
    for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < A.N; r0 += (int64_t)gridDim.x * groups) {
        const int64_t row = r0 + group;
        const bool live = row < A.N;
        const int64_t V = A.V;
        const T* z = static_cast<const T*>(A.z) + (live ? row * A.ldz : 0);
        const int64_t y = live && A.labels ? entry(A.labels, A.labels64, row) : -1;
        // aligned body [head, head + body): 16-byte loads; the rest by element
        const int64_t head = min(V, (int64_t)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T)));
        const int64_t nvec = (V - head) / W, tail = head + nvec * W;
        bool counts = live && (!A.labels || label_counts(A, y));

        // ---- the teacher's distribution, by the row's first warp ----
        float has = 0.f, plogp = 0.f;
        if (t < 32) {
            float top = -INFINITY;
            bool any = false;
            for (int k = lane; counts && k < A.K; k += 32) {
                const float tk = A.t[row * A.K + k];
                const bool ok = entry_counts(A, entry(A.ids, A.ids64, row * A.K + k), tk);
                any |= ok;
                if (ok) top = fmaxf(top, tk);
            }
            any = __any_sync(0xffffffffu, any);
            top = warp_maxf(top);
            float sum = 0.f;
            for (int k = lane; k < A.K; k += 32) {
                float e = 0.f;
                int id = -1;
                if (counts) {
                    const float tk = A.t[row * A.K + k];
                    const int64_t i64 = entry(A.ids, A.ids64, row * A.K + k);
                    if (entry_counts(A, i64, tk)) {
                        id = (int)i64;
                        e = expf((tk - top) / A.temp);
                    }
                }
                prob[k] = e;
                pid[k] = id;
                sum += e;
            }
            sum = warp_sum(sum);
            for (int k = lane; k < A.K; k += 32) {
                const float p = any ? prob[k] / sum : 0.f;
                if ((MODE & 1) && pid[k] >= 0 && !(p == 0.f))
                    plogp += p * ((A.t[row * A.K + k] - top) / A.temp - logf(sum));
                prob[k] = p;
            }
            if (MODE & 1) plogp = warp_sum(plogp);
            has = any ? 1.f : 0.f;
            if (lane == 0) shared_row[group][0] = has;
        }
        sync();
        has = shared_row[group][0];
        if (!A.labels) counts = counts && has != 0.f;

        // ---- maximum and sums ----
        Run R = {-INFINITY, 0.f, 0.f};
        if (MODE & 1) {
            if (counts) {
                for (int64_t i = t; i < head + (V - tail); i += tpr) {
                    const float v = to_f32(z[i < head ? i : tail + (i - head)]);
                    take<TWO, 1>(R, &v, X);
                }
                const uint4* zv = reinterpret_cast<const uint4*>(z + head);
                for (int64_t i = t; i < nvec; i += tpr) {
                    float v[W];
                    Pack16<T>::unpack(zv[i], v);
                    take<TWO, W>(R, v, X);
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float m = __shfl_xor_sync(0xffffffffu, R.m, o), s = __shfl_xor_sync(0xffffffffu, R.s, o);
                const float s1 = TWO ? __shfl_xor_sync(0xffffffffu, R.s1, o) : 0.f;
                // the lower lane's values first on both sides: the same bits in every lane
                Run L = {R.m, R.s, R.s1};
                if (lane & o) { L = {m, s, s1}; merge<TWO>(L, R.m, R.s, R.s1, X.c, X.c1); }
                else merge<TWO>(L, m, s, s1, X.c, X.c1);
                R = L;
            }
            if (tpr > 32) {
                if (lane == 0) { red[warp][0] = R.m; red[warp][1] = R.s; red[warp][2] = R.s1; }
                __syncthreads();
                const int w0 = warp & ~(nw - 1);
                R = {red[w0][0], red[w0][1], red[w0][2]};
                for (int i = 1; i < nw; ++i) merge<TWO>(R, red[w0 + i][0], red[w0 + i][1], red[w0 + i][2], X.c, X.c1);
            }
            if (!TWO) R.s1 = R.s;
        } else if (counts) {
            R = {A.stats[row * 3], A.stats[row * 3 + 1], A.stats[row * 3 + 2]};
        }

        // ---- loss of the row, by its first warp ----
        if ((MODE & 1) && t < 32) {
            const float lse = R.m / A.temp + logf(R.s);
            float cross = 0.f;           // sum_k p_k (lse(z / T) - z_k / T)
            for (int k = lane; counts && k < A.K; k += 32)
                if (pid[k] >= 0 && !(prob[k] == 0.f)) cross += prob[k] * (lse - to_f32(z[pid[k]]) / A.temp);
            cross = warp_sum(cross);
            if (live && lane == 0) {
                float loss = 0.f;
                if (counts) {
                    if (has != 0.f) loss = A.alpha * A.temp * A.temp * (plogp + cross);
                    if (A.labels) loss += (1.f - A.alpha) * (R.m + logf(R.s1) - to_f32(z[y]));
                }
                A.row_loss[row] = loss;
                if (A.row_counts) A.row_counts[row] = counts ? 1.f : 0.f;
                if (A.stats) { A.stats[row * 3] = R.m; A.stats[row * 3 + 1] = R.s; A.stats[row * 3 + 2] = R.s1; }
            }
        }

        // ---- gradient ----
        if (MODE & 2) {
            T* dz = static_cast<T*>(A.dz) + (live ? row * V : 0);
            const bool same = (reinterpret_cast<uintptr_t>(dz) & 15) == (reinterpret_cast<uintptr_t>(z) & 15);
            const int64_t h = same ? head : V, n = same ? nvec : 0, tl = same ? tail : V;
            if (live && !counts) {
                const uint4 zero = make_uint4(0, 0, 0, 0);
                for (int64_t i = t; i < h + (V - tl); i += tpr) dz[i < h ? i : tl + (i - h)] = from_f32<T>(0.f);
                for (int64_t i = t; i < n; i += tpr) reinterpret_cast<uint4*>(dz + h)[i] = zero;
            } else if (live) {
                float g = A.gscale / number;
                if (A.gout) g *= A.gout[A.gout_stride * row];
                const float ga = g * A.alpha * A.temp * has, gb = A.labels ? g * (1.f - A.alpha) : 0.f;
                const float a = ga / R.s, b = TWO ? gb / R.s1 : 0.f;
                const float ref = R.m == -INFINITY ? 0.f : R.m;
                // one temperature: both terms share the exponential
                const float ab = TWO ? a : a + gb / R.s;
                auto dense = [&](float v) {
                    float e, e1 = 0.f;
                    X.at(v, ref, e, e1);
                    return TWO ? fmaf(b, e1, ab * e) : ab * e;
                };
                for (int64_t i = t; i < h + (V - tl); i += tpr) {
                    const int64_t c = i < h ? i : tl + (i - h);
                    dz[c] = from_f32<T>(dense(to_f32(z[c])));
                }
                const uint4* zv = reinterpret_cast<const uint4*>(z + h);
                uint4* dv = reinterpret_cast<uint4*>(dz + h);
                for (int64_t i = t; i < n; i += tpr) {
                    float v[W];
                    Pack16<T>::unpack(zv[i], v);
#pragma unroll
                    for (int j = 0; j < W; ++j) v[j] = dense(v[j]);
                    dv[i] = Pack16<T>::pack(v);
                }
                sync();
                for (int k = t; k <= A.K; k += tpr) {
                    const int id = k < A.K ? pid[k] : (A.labels ? (int)y : -1);
                    if (id < 0) continue;
                    float p = 0.f;
                    for (int j = 0; j < A.K; ++j) p += pid[j] == id ? prob[j] : 0.f;
                    float v = dense(to_f32(z[id])) - ga * p;
                    if (A.labels && id == (int)y) v -= gb;
                    dz[id] = from_f32<T>(v);
                }
            }
        }
        sync();          // prob / pid / red are written again by the next row
    }
}

// the rows' losses in a fixed order, divided by the number of rows that count
// (which the gradient reads); 64 bits: a sum of up to 2^24 whole numbers is exact
__global__ void __launch_bounds__(1024) total_kernel(const Args A, float* loss, float* number) {
    __shared__ double red[32][2];
    double s = 0.0, n = 0.0;
    for (int64_t r = threadIdx.x; r < A.N; r += 1024) {
        s += (double)A.row_loss[r];
        n += (double)A.row_counts[r];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        n += __shfl_xor_sync(0xffffffffu, n, o);
    }
    if ((threadIdx.x & 31) == 0) { red[threadIdx.x >> 5][0] = s; red[threadIdx.x >> 5][1] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = n = 0.0;
        for (int i = 0; i < 32; ++i) { s += red[i][0]; n += red[i][1]; }
        n = n > 1.0 ? n : 1.0;
        loss[0] = (float)(A.mean ? s / n : s);
        if (number) number[0] = (float)n;
    }
}

int sm_count() {
    int d = 0, n = 148;
    if (cudaGetDevice(&d) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d);
    return n;
}

template <typename T, bool TWO, int MODE>
void launch(Args& A, cudaStream_t st) {
    // threads of a row: a warp for short rows, a block otherwise
    A.tpr = A.V <= 1024 ? 32 : A.V <= 4096 ? 128 : A.V <= 65536 ? 256 : 1024;
    if (A.N < sm_count() && A.V > 4096) A.tpr = 1024;
    const int threads = A.tpr == 32 ? 256 : A.tpr, groups = threads / A.tpr;
    const int64_t need = (A.N + groups - 1) / groups, wave = (int64_t)sm_count() * (2048 / threads);
    const size_t smem = (size_t)groups * 2 * A.K * sizeof(float);
    row_kernel<T, TWO, MODE><<<(int)(need < wave ? need : wave), threads, smem, st>>>(A);
}

template <int MODE>
int run(Args& A, int32_t type, cudaStream_t st, const char* name) {
    const bool two = A.labels && A.temp != 1.0f;
    A.squarings = A.temp == 2.0f ? 1 : A.temp == 4.0f ? 2 : A.temp == 8.0f ? 3 : 0;
    if (type == 0) { if (two) launch<float, true, MODE>(A, st); else launch<float, false, MODE>(A, st); }
    else if (type == 1) {
        if (two) launch<__nv_bfloat16, true, MODE>(A, st); else launch<__nv_bfloat16, false, MODE>(A, st);
    } else { if (two) launch<__half, true, MODE>(A, st); else launch<__half, false, MODE>(A, st); }
    return check_launch(name);
}

int check(const char* name, const Args& A, int32_t type) {
    if (type < 0 || type > 2) return fail(CONCORD_EINVAL, std::string(name) + ": unknown element type");
    if (A.N < 0 || A.V <= 0 || A.K <= 0 || A.ldz < A.V || A.V > INT32_MAX)
        return fail(CONCORD_ESHAPE, std::string(name) + ": bad extents or row stride");
    if (A.K > MAX_K) return fail(CONCORD_ETOOBIG, std::string(name) + ": more than 512 teacher entries");
    if (!(A.temp > 0.f) || !(A.temp <= FLT_MAX)) return fail(CONCORD_EINVAL, std::string(name) + ": temperature must be positive");
    if (A.N > 0 && (!A.z || !A.ids || !A.t)) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    return CONCORD_OK;
}

Args make_args(const concord_distill_params* p, const void* z, int64_t ldz, const void* ids, const float* t,
               const void* labels, int64_t N, int64_t V, int64_t K) {
    Args A{};
    A.z = z; A.ldz = ldz; A.ids = ids; A.t = t; A.labels = labels;
    A.ignore = p->ignore_index; A.ids64 = p->ids64; A.labels64 = p->labels64;
    A.K = (int)K; A.N = N; A.V = V;
    A.temp = p->temperature; A.alpha = p->alpha; A.gscale = p->grad_scale; A.mean = p->mean;
    return A;
}

}  // namespace distill
}  // namespace concord

using namespace concord;

// workspace: the partial counts, the rows' losses, which rows count
extern "C" size_t concord_distill_workspace_bytes(int64_t N) {
    return distill::COUNT_BLOCKS * sizeof(int) + (N > 0 ? (size_t)N * 2 * sizeof(float) : 0);
}

extern "C" int concord_distill_loss(const concord_distill_params* p, const void* z, int32_t z_type, int64_t ldz,
                                    const void* ids, const float* t, const void* labels, float* loss,
                                    float* row_loss, float* stats, void* dz, int64_t N, int64_t V, int64_t K,
                                    void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "concord_distill_loss";
    if (!p || (!loss && !row_loss)) return fail(CONCORD_EINVAL, "concord_distill_loss: null pointer");
    distill::Args A = distill::make_args(p, z, ldz, ids, t, labels, N, V, K);
    if (int rc = distill::check(name, A, z_type)) return rc;
    if (!workspace || workspace_bytes < concord_distill_workspace_bytes(N))
        return fail(CONCORD_EWORKSPACE, "concord_distill_loss: workspace too small");
    cudaStream_t st = as_stream(stream);
    if (N == 0) {
        if (loss) cudaMemsetAsync(loss, 0, sizeof(float), st);
        return check_launch(name);
    }
    int* counts = static_cast<int*>(workspace);
    float* rows = reinterpret_cast<float*>(counts + distill::COUNT_BLOCKS);
    A.counts = counts;
    A.row_loss = row_loss ? row_loss : rows;
    A.row_counts = loss ? rows + N : nullptr;
    A.stats = stats;
    A.dz = dz;
    if (A.mean && dz) distill::count_kernel<<<distill::COUNT_BLOCKS, 256, 0, st>>>(A, counts);
    if (int rc = dz ? distill::run<3>(A, z_type, st, name) : distill::run<1>(A, z_type, st, name)) return rc;
    if (loss) distill::total_kernel<<<1, 1024, 0, st>>>(A, loss, stats ? stats + 3 * N : nullptr);
    return check_launch(name);
}

extern "C" int concord_distill_grad(const concord_distill_params* p, const void* z, int32_t z_type, int64_t ldz,
                                    const void* ids, const float* t, const void* labels, const float* stats,
                                    const float* grad_out, int32_t grad_out_per_row, void* dz, int64_t N, int64_t V,
                                    int64_t K, void* stream) {
    const char* name = "concord_distill_grad";
    if (!p || (N > 0 && (!stats || !dz))) return fail(CONCORD_EINVAL, "concord_distill_grad: null pointer");
    distill::Args A = distill::make_args(p, z, ldz, ids, t, labels, N, V, K);
    if (int rc = distill::check(name, A, z_type)) return rc;
    if (N == 0) return CONCORD_OK;
    A.stats = const_cast<float*>(stats);
    A.number = stats + 3 * N;
    A.gout = grad_out;
    A.gout_stride = grad_out_per_row ? 1 : 0;
    A.dz = dz;
    return distill::run<2>(A, z_type, as_stream(stream), name);
}
