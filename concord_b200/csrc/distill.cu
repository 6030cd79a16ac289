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
// 16384 x 32000 bf16, T = 2, value and gradient: 500 us, 4.2 TB/s, the
// special-function unit 64 % busy (256 threads a row, four 16-byte loads each on
// their way; 512 threads 729 us, 128 518, two loads 539).
// Where T is 2, 4 or 8, exp(z) is exp(z / T) squared log2(T) times
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
constexpr int MAX_V = INT32_MAX - 1024;      // a thread's column and the next one of its 1024 neighbours' fit 32 bits
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

// KIND of a kernel: 0: one temperature serves both terms (or there is one term
// only); 1: two exponentials; 1 + n: T = 2^n, the second is the first squared n times
// running maximum with the sums of exp((z - m) / T) and exp(z - m)
struct Run {
    float m, s, s1;
};

template <int KIND>
__device__ __forceinline__ void merge(Run& a, float m, float s, float s1, float c, float c1) {
    const float top = fmaxf(a.m, m), ref = top == -INFINITY ? 0.f : top;
    a.s = a.s * ex2f((a.m - ref) * c) + s * ex2f((m - ref) * c);
    if (KIND) a.s1 = a.s1 * ex2f((a.m - ref) * c1) + s1 * ex2f((m - ref) * c1);
    a.m = top;
}

template <int KIND> struct Exps {
    float c, c1;
    // exp((z - m) / T) and exp(z - m) of two logits; the difference first, so
    // that rows of the type's lowest value, or of 1e4 and more, lose nothing in
    // a product.  `neg`: -m twice.
    __device__ __forceinline__ void at(uint64_t z, uint64_t neg, uint64_t& e, uint64_t& e1) const {
        const uint64_t d = add2(z, neg);
        float a, b;
        unf2(mul2(d, f2(c, c)), a, b);
        e = f2(ex2f(a), ex2f(b));
        e1 = e;
        if (KIND == 1) {
            unf2(mul2(d, f2(c1, c1)), a, b);
            e1 = f2(ex2f(a), ex2f(b));
        }
#pragma unroll
        for (int i = 1; i < KIND; ++i) e1 = mul2(e1, e1);
    }
};

// NE logits (even) into a thread's running maximum and sums
template <int KIND, int NE>
__device__ __forceinline__ void take(Run& r, const float* v, const Exps<KIND>& X) {
    float top = fmaxf(v[0], v[1]);
#pragma unroll
    for (int i = 2; i < NE; i += 2) top = max3(top, v[i], v[i + 1]);
    if (top > r.m) {
        const float old = r.m;          // -inf at first: exp gives 0
        r.s *= ex2f((old - top) * X.c);
        if (KIND) r.s1 *= ex2f((old - top) * X.c1);
        r.m = top;
    }
    const float ref = r.m == -INFINITY ? 0.f : r.m;
    const uint64_t neg = f2(-ref, -ref);
    uint64_t s[2] = {0, 0}, s1 = 0;
#pragma unroll
    for (int i = 0; i < NE; i += 2) {
        uint64_t e, e1;
        X.at(f2(v[i], v[i + 1]), neg, e, e1);
        s[(i >> 1) & 1] = add2(s[(i >> 1) & 1], e);
        if (KIND) s1 = add2(s1, e1);
    }
    float a, b;
    unf2(add2(s[0], s[1]), a, b);
    r.s += a + b;
    if (KIND) {
        unf2(s1, a, b);
        r.s1 += a + b;
    }
}

// 16 bytes of -inf: what stands for the pieces beyond a row's end
template <typename T> __device__ __forceinline__ uint4 nothing() {
    const uint32_t u = sizeof(T) == 4 ? 0xff800000u : __is_same(T, __half) ? 0xfc00fc00u : 0xff80ff80u;
    return make_uint4(u, u, u, u);
}

constexpr int DEEP = 4;              // 16-byte loads of a thread on their way at a time

// T: logits' type; MODE 1: statistics and
// loss, 2: gradient from given statistics, 3: both
template <typename T, int KIND, int MODE>
__global__ void __launch_bounds__(1024) row_kernel(const Args A) {
    constexpr int W = Pack16<T>::N;
    extern __shared__ float dyn[];       // groups x (K probabilities, K ids, K logits at them)
    __shared__ float red[32][3];
    __shared__ float teacher[32];        // whether the group's teacher has an entry
    const int tpr = A.tpr, t = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = tpr >> 5;
    const int V = (int)A.V, K = A.K;
    float* prob = dyn + (size_t)group * 3 * K;
    int* pid = reinterpret_cast<int*>(prob + K);
    float* at_id = prob + 2 * K;
    Exps<KIND> X;
    X.c = LOG2E / A.temp;
    X.c1 = LOG2E;
    float number = 1.f;
    if (MODE == 3 && A.mean) number = (float)max(1, total_count(A));
    if (MODE == 2 && A.mean) number = *A.number;

    // (a block of more than a warp per row holds one row: its branches are uniform)
    auto sync = [&]() { if (tpr == 32) __syncwarp(); else __syncthreads(); };
    const int64_t row0 = (int64_t)blockIdx.x * groups + group;
    int64_t next_y = row0 < A.N && A.labels ? entry(A.labels, A.labels64, row0) : -1;      // a row ahead
    for (int64_t row = row0; row - group < A.N; row += (int64_t)gridDim.x * groups) {
        const bool live = row < A.N;
        const T* z = static_cast<const T*>(A.z) + (live ? row * A.ldz : 0);
        const int64_t y = next_y;
        const int64_t ahead = row + (int64_t)gridDim.x * groups;
        next_y = ahead < A.N && A.labels ? entry(A.labels, A.labels64, ahead) : -1;
        // aligned body [head, tail): 16-byte loads; the rest by element
        const int head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T)));
        const int nvec = (V - head) / W, tail = head + nvec * W;
        bool counts = live && (!A.labels || label_counts(A, y));
        float t0 = 0.f;
        int64_t id0 = -1;
        if (t < 32 && lane < K && live) {
            t0 = A.t[row * K + lane];
            id0 = entry(A.ids, A.ids64, row * K + lane);
        }

        // ---- maximum and sums (before the teacher's entries are known: a row
        // that turns out to have none is read for nothing) ----
        Run R = {-INFINITY, 0.f, 0.f};
        if ((MODE & 1) && counts) {
            for (int i = t; i < head + (V - tail); i += tpr) {
                const float v[2] = {to_f32(z[i < head ? i : tail + (i - head)]), -INFINITY};
                take<KIND, 2>(R, v, X);
            }
            const uint4* zv = reinterpret_cast<const uint4*>(z + head);
            uint4 u[DEEP];
            auto take_all = [&]() {
#pragma unroll
                for (int k = 0; k < DEEP; k += 2) {
                    float v[2 * W];
                    Pack16<T>::unpack(u[k], v);
                    Pack16<T>::unpack(u[k + 1], v + W);
                    take<KIND, 2 * W>(R, v, X);
                }
            };
            int i = t;
            for (; i + (DEEP - 1) * tpr < nvec; i += DEEP * tpr) {
#pragma unroll
                for (int k = 0; k < DEEP; ++k) u[k] = zv[i + k * tpr];
                take_all();
            }
            if (i < nvec) {
#pragma unroll
                for (int k = 0; k < DEEP; ++k) u[k] = i + k * tpr < nvec ? zv[i + k * tpr] : nothing<T>();
                take_all();
            }
        }

        // ---- the teacher's distribution, and the logits at its places, by the
        // row's first warp (its first 32 entries are on their way since before
        // the row was read) ----
        float plogp = 0.f, zy = 0.f;
        if (t < 32) {
            if ((MODE & 1) && A.labels && counts) zy = to_f32(z[y]);
            float top = -INFINITY;
            for (int k = lane; k < K; k += 32) {
                float tk = t0;
                int64_t id = id0;
                if (k >= 32 && counts) { tk = A.t[row * K + k]; id = entry(A.ids, A.ids64, row * K + k); }
                const bool ok = counts && entry_counts(A, id, tk);
                pid[k] = ok ? (int)id : -1;
                prob[k] = tk;
                if (ok) {
                    top = fmaxf(top, tk);
                    at_id[k] = to_f32(z[id]);
                }
            }
            bool any = false;
            for (int k = lane; k < K; k += 32) any |= pid[k] >= 0;
            any = __any_sync(0xffffffffu, any);
            top = warp_maxf(top);
            float sum = 0.f;
            for (int k = lane; k < K; k += 32) {
                const float d = (prob[k] - top) / A.temp, e = pid[k] >= 0 ? expf(d) : 0.f;
                if ((MODE & 1) && pid[k] >= 0 && !(e == 0.f)) plogp += e * d;
                prob[k] = e;
                sum += e;
            }
            sum = warp_sum(sum);
            if (any) {
                for (int k = lane; k < K; k += 32) prob[k] /= sum;
                // sum_k p_k log p_k
                if (MODE & 1) plogp = warp_sum(plogp) / sum - logf(sum);
            }
            if (lane == 0) teacher[group] = any ? 1.f : 0.f;
        }

        // ---- the row's statistics, the same bits in every thread ----
        if (MODE & 1) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float m = __shfl_xor_sync(0xffffffffu, R.m, o), s = __shfl_xor_sync(0xffffffffu, R.s, o);
                const float s1 = KIND ? __shfl_xor_sync(0xffffffffu, R.s1, o) : 0.f;
                Run L = {R.m, R.s, R.s1};                     // the lower lane's first on both sides
                if (lane & o) { L = {m, s, s1}; merge<KIND>(L, R.m, R.s, R.s1, X.c, X.c1); }
                else merge<KIND>(L, m, s, s1, X.c, X.c1);
                R = L;
            }
            if (lane == 0 && tpr > 32) { red[warp][0] = R.m; red[warp][1] = R.s; red[warp][2] = R.s1; }
        }
        sync();
        if (MODE & 1) {
            if (tpr > 32) {
                R = {red[0][0], red[0][1], red[0][2]};
                for (int i = 1; i < nw; ++i) merge<KIND>(R, red[i][0], red[i][1], red[i][2], X.c, X.c1);
            }
            if (!KIND) R.s1 = R.s;
        }
        const float has = teacher[group];
        if (!A.labels) counts = counts && has != 0.f;
        if (MODE == 2 && counts) R = {A.stats[row * 3], A.stats[row * 3 + 1], A.stats[row * 3 + 2]};

        // ---- loss of the row, by its first warp ----
        if ((MODE & 1) && t < 32) {
            // differences from the maximum first here too: added to log(sum), a
            // maximum of 1e4 would leave 1e-3 of a loss that may be no larger
            const float logs = logf(R.s);
            float cross = 0.f;           // sum_k p_k (lse(z / T) - z_k / T)
            for (int k = lane; counts && k < K; k += 32)
                if (pid[k] >= 0 && !(prob[k] == 0.f)) cross += prob[k] * (logs + (R.m - at_id[k]) / A.temp);
            cross = warp_sum(cross);
            if (live && lane == 0) {
                float loss = 0.f;
                if (counts) {
                    if (has != 0.f) loss = A.alpha * A.temp * A.temp * (plogp + cross);
                    if (A.labels) loss += (1.f - A.alpha) * (logf(R.s1) + (R.m - zy));
                }
                A.row_loss[row] = loss;
                if (A.row_counts) A.row_counts[row] = counts ? 1.f : 0.f;
                if (A.stats) { A.stats[row * 3] = R.m; A.stats[row * 3 + 1] = R.s; A.stats[row * 3 + 2] = R.s1; }
            }
        }

        // ---- gradient ----
        if (MODE & 2) {
            T* dz = static_cast<T*>(A.dz) + (live ? row * A.V : 0);
            const bool same = (reinterpret_cast<uintptr_t>(dz) & 15) == (reinterpret_cast<uintptr_t>(z) & 15);
            const int h = same ? head : V, n = same ? nvec : 0, tl = same ? tail : V;
            uint4* dv = reinterpret_cast<uint4*>(dz + h);
            if (live && !counts) {
                for (int i = t; i < h + (V - tl); i += tpr) dz[i < h ? i : tl + (i - h)] = from_f32<T>(0.f);
                for (int i = t; i < n; i += tpr) dv[i] = make_uint4(0, 0, 0, 0);
            } else if (live) {
                float g = A.gscale / number;
                if (A.gout) g *= A.gout[A.gout_stride * row];
                const float ga = g * A.alpha * A.temp * has, gb = A.labels ? g * (1.f - A.alpha) : 0.f;
                const float ref = R.m == -INFINITY ? 0.f : R.m;
                // one temperature: both terms share the exponential
                const float a = KIND ? ga / R.s : ga / R.s + gb / R.s, b = gb / R.s1;
                const uint64_t neg = f2(-ref, -ref), a2 = f2(a, a), b2 = f2(b, b);
                auto dense = [&](uint64_t v) -> uint64_t {
                    uint64_t e, e1;
                    X.at(v, neg, e, e1);
                    return KIND ? fma2(b2, e1, mul2(a2, e)) : mul2(a2, e);
                };
                auto dense1 = [&](float v) {
                    float p, q;
                    unf2(dense(f2(v, v)), p, q);
                    return p;
                };
                for (int i = t; i < h + (V - tl); i += tpr) {
                    const int c = i < h ? i : tl + (i - h);
                    dz[c] = from_f32<T>(dense1(to_f32(z[c])));
                }
                const uint4* zv = reinterpret_cast<const uint4*>(z + h);
                uint4 u[DEEP];
                auto put = [&](int at, const uint4& x) {
                    float v[W];
                    Pack16<T>::unpack(x, v);
#pragma unroll
                    for (int j = 0; j < W; j += 2) unf2(dense(f2(v[j], v[j + 1])), v[j], v[j + 1]);
                    __stcs(dv + at, Pack16<T>::pack(v));     // not read again here: the L2 is z's
                };
                int i = t;
                for (; i + (DEEP - 1) * tpr < n; i += DEEP * tpr) {
#pragma unroll
                    for (int k = 0; k < DEEP; ++k) u[k] = zv[i + k * tpr];
#pragma unroll
                    for (int k = 0; k < DEEP; ++k) put(i + k * tpr, u[k]);
                }
                for (; i < n; i += tpr) put(i, zv[i]);
                sync();
                for (int k = t; k <= K; k += tpr) {
                    const int id = k < K ? pid[k] : (A.labels ? (int)y : -1);
                    if (id < 0) continue;
                    float p = 0.f;
                    for (int j = 0; j < K; ++j) p += pid[j] == id ? prob[j] : 0.f;
                    float v = dense1(k < K ? at_id[k] : to_f32(z[id])) - ga * p;
                    if (A.labels && id == (int)y) v -= gb;
                    dz[id] = from_f32<T>(v);
                }
            }
        }
        sync();          // prob, pid and red are written again by the next row
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

template <typename T, int KIND, int MODE>
void launch(Args& A, cudaStream_t st) {
    // threads of a row: a warp for short rows, a block otherwise
    A.tpr = A.V <= 1024 ? 32 : A.V <= 4096 ? 128 : A.V <= 65536 ? 256 : 1024;
    if (A.N < sm_count() && A.V > 4096) A.tpr = 1024;
    const int threads = A.tpr > 32 ? A.tpr : A.K > 256 ? 128 : 256, groups = threads / A.tpr;
    const int64_t need = (A.N + groups - 1) / groups, wave = (int64_t)sm_count() * (2048 / threads);
    const size_t smem = (size_t)groups * 3 * A.K * sizeof(float);       // 24 KB at most
    row_kernel<T, KIND, MODE><<<(int)(need < wave ? need : wave), threads, smem, st>>>(A);
}

template <typename T, int MODE>
void launch_kind(Args& A, cudaStream_t st) {
    if (!A.labels || A.temp == 1.0f) launch<T, 0, MODE>(A, st);
    else if (A.temp == 2.0f) launch<T, 2, MODE>(A, st);
    else if (A.temp == 4.0f) launch<T, 3, MODE>(A, st);
    else if (A.temp == 8.0f) launch<T, 4, MODE>(A, st);
    else launch<T, 1, MODE>(A, st);
}

template <int MODE>
int run(Args& A, int32_t type, cudaStream_t st, const char* name) {
    if (type == 0) launch_kind<float, MODE>(A, st);
    else if (type == 1) launch_kind<__nv_bfloat16, MODE>(A, st);
    else launch_kind<__half, MODE>(A, st);
    return check_launch(name);
}

int check(const char* name, const Args& A, int32_t type) {
    if (type < 0 || type > 2) return fail(CONCORD_EINVAL, std::string(name) + ": unknown element type");
    if (A.N < 0 || A.V <= 0 || A.K <= 0 || A.ldz < A.V)
        return fail(CONCORD_ESHAPE, std::string(name) + ": bad extents or row stride");
    if (A.V > MAX_V) return fail(CONCORD_ETOOBIG, std::string(name) + ": more than 2^31 - 1025 columns");
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
    // (a tensor of no rows has no address)
    if (!p || (!loss && !row_loss && N != 0)) return fail(CONCORD_EINVAL, "concord_distill_loss: null pointer");
    distill::Args A = distill::make_args(p, z, ldz, ids, t, labels, N, V, K);
    if (int rc = distill::check(name, A, z_type)) return rc;
    if (!workspace || workspace_bytes < concord_distill_workspace_bytes(N))
        return fail(CONCORD_EWORKSPACE, "concord_distill_loss: workspace too small");
    cudaStream_t st = as_stream(stream);
    if (N == 0) {
        if (!loss) return CONCORD_OK;
        cudaMemsetAsync(loss, 0, sizeof(float), st);
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
