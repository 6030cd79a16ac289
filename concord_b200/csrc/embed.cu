// embed.cu — embedding lookup with scaling, and the table's gradient.
//
//   y[t]  = scale W[ids[t]]                       (0 where ids[t] is outside [0, V))
//   dW[v] = scale sum over t with ids[t] = v of dy[t]      (0 for the padding row)
//
// Bound by memory: the forward reads a row and writes one, the backward reads
// dy once and writes the whole table once (rows of no token are zeros).
//
// The gradient goes by sorted tokens: a stable radix sort of (id, token) gives
// every row of the table its tokens in order, so that sums are fp32 in token
// order, without atomics on them: the same bits on every run.  A row of up to
// SEG tokens is summed by the threads that own it.  A longer one (every symbol
// of a small vocabulary) is cut where the sorted tokens pass a multiple of SEG;
// the pieces are summed side by side and joined in order by a second kernel.
#include "common.cuh"
#include "vec.cuh"

namespace concord {
namespace embed {

constexpr int SEG = 64;                    // tokens that one owner sums
constexpr int DIGIT = 9, BINS = 1 << DIGIT;
constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32;
constexpr int64_t SORT_CHUNK = 4096;       // tokens of a sorting block, and more where blocks would pass
constexpr int64_t SORT_BLOCKS = 512;       // this number: each of them reads all blocks' counts

// ---------------------------------------------------------------- forward
// A thread holds VEC columns of ROWS rows.
template <typename TW, typename TY, int VEC, int ROWS>
__global__ void __launch_bounds__(256)
    fwd_kernel(const void* ids, int ids64, const TW* w, int64_t ldw, TY* y, int64_t T, int64_t V, int D, float scale) {
    const int col = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    const int64_t t0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * ROWS;
    if (col >= D || t0 >= T) return;
    int64_t id[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        id[r] = -1;
        if (t0 + r < T)
            id[r] = ids64 ? static_cast<const int64_t*>(ids)[t0 + r] : (int64_t)static_cast<const int32_t*>(ids)[t0 + r];
    }
    float v[ROWS][VEC];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (id[r] >= 0 && id[r] < V) load_vec<VEC>(w + id[r] * ldw + col, v[r]);
        else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[r][j] = 0.f;
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (t0 + r >= T) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[r][j] *= scale;
        store_vec<VEC>(y + (t0 + r) * D + col, v[r]);
    }
}

// ---------------------------------------------------------------- sort
// Token t's key: its id; V where it counts for no row.
__device__ __forceinline__ uint32_t key_of(const void* ids, int ids64, int64_t t, int64_t V, int64_t padding) {
    const int64_t id =
        ids64 ? static_cast<const int64_t*>(ids)[t] : (int64_t)static_cast<const int32_t*>(ids)[t];
    return id < 0 || id >= V || id == padding ? (uint32_t)V : (uint32_t)id;
}

struct Pass {
    const void* ids;          // first pass: the call's ids
    int ids64;
    const uint2* from;        // later ones: (key, token) as the pass before left them
    uint2* to;
    uint32_t* counts;         // [blocks][BINS]
    int64_t T, V, padding, chunk;
    int shift;
};

__device__ __forceinline__ uint2 item(const Pass& P, int64_t t) {
    return P.from ? P.from[t] : make_uint2(key_of(P.ids, P.ids64, t, P.V, P.padding), (uint32_t)t);
}

__global__ void __launch_bounds__(SORT_THREADS) count_kernel(const __grid_constant__ Pass P) {
    __shared__ uint32_t n[BINS];
    for (int b = threadIdx.x; b < BINS; b += SORT_THREADS) n[b] = 0;
    __syncthreads();
    const int64_t t0 = blockIdx.x * P.chunk, t1 = min(t0 + P.chunk, P.T);
    for (int64_t t = t0 + threadIdx.x; t < t1; t += SORT_THREADS)
        atomicAdd(&n[(item(P, t).x >> P.shift) & (BINS - 1)], 1u);          // whole numbers: any order
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += SORT_THREADS) P.counts[blockIdx.x * (int64_t)BINS + b] = n[b];
}

// Each warp owns a run of the block's tokens: it counts their digits, and, once
// the places before them are known, puts them there in order.
__global__ void __launch_bounds__(SORT_THREADS) place_kernel(const __grid_constant__ Pass P) {
    __shared__ uint32_t at[SORT_WARPS][BINS];      // the warp's next place for each digit
    __shared__ uint32_t sums[SORT_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < SORT_WARPS * BINS; i += SORT_THREADS) (&at[0][0])[i] = 0;
    __syncthreads();
    const int64_t run = P.chunk / SORT_WARPS, t0 = blockIdx.x * P.chunk + warp * run, t1 = min(t0 + run, P.T);
    for (int64_t t = t0; t < t1; t += 32) {
        const bool have = t + lane < t1;
        const uint32_t d = have ? (item(P, t + lane).x >> P.shift) & (BINS - 1) : BINS;
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        if (have && lane == __ffs(same) - 1) at[warp][d] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    // places before this block: all tokens of smaller digits, earlier blocks' of the same
    static_assert(BINS == SORT_THREADS, "a thread a digit");
    uint32_t all = 0, before = 0;
#pragma unroll 8
    for (int b = 0; b < gridDim.x; ++b) {
        const uint32_t n = P.counts[b * (int64_t)BINS + threadIdx.x];
        all += n;
        before += b < blockIdx.x ? n : 0;
    }
    uint32_t incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    uint32_t base = incl - all + before;
    for (int w = 0; w < warp; ++w) base += sums[w];
    for (int w = 0; w < SORT_WARPS; ++w) {
        const uint32_t n = at[w][threadIdx.x];
        at[w][threadIdx.x] = base;
        base += n;
    }
    __syncthreads();
    for (int64_t t = t0; t < t1; t += 32) {
        const bool have = t + lane < t1;
        const uint2 it = have ? item(P, t + lane) : make_uint2(0, 0);
        const uint32_t d = have ? (it.x >> P.shift) & (BINS - 1) : BINS;
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        if (have) P.to[at[warp][d] + __popc(same & ((1u << lane) - 1))] = it;
        __syncwarp();
        if (have && lane == __ffs(same) - 1) at[warp][d] += __popc(same);
        __syncwarp();
    }
}

// first[v]: the first sorted place of a key of v or more, v = 0 .. V
__global__ void __launch_bounds__(256) first_kernel(const uint2* sorted, uint32_t* first, int64_t T, int64_t V) {
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (v > V) return;
    uint32_t lo = 0, hi = (uint32_t)T;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (sorted[mid].x < v) lo = mid + 1;
        else hi = mid;
    }
    first[v] = lo;
}

// ---------------------------------------------------------------- sums
struct Sums {
    const uint2* sorted;
    const uint32_t* first;
    float* part;              // [chunks][2][D]: pieces of the long rows
    int64_t T, V, lddy;
    int64_t chunks;
    int D;
    float scale;
};

// acc += the rows of tokens [a, b) of the sorted ones, in order, four loads on their way
template <typename TY, int VEC>
__device__ __forceinline__ void add_rows(const Sums& P, const TY* dy, uint32_t a, uint32_t b, int col, float* acc) {
    constexpr int AHEAD = 4;
    uint32_t p = a;
    for (; p + AHEAD <= b; p += AHEAD) {
        float v[AHEAD][VEC];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) load_vec<VEC>(dy + P.sorted[p + i].y * P.lddy + col, v[i]);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += v[i][j];
    }
    for (; p < b; ++p) {
        float v[VEC];
        load_vec<VEC>(dy + P.sorted[p].y * P.lddy + col, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += v[j];
    }
}

// The first `chunks` rows of threads take the pieces of long rows, the others a
// row of the table each.
template <typename TY, typename TW, int VEC>
__global__ void __launch_bounds__(256) sum_kernel(const TY* dy, TW* dw, const __grid_constant__ Sums P) {
    const int col = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    const int64_t i = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (col >= P.D || i >= P.chunks + P.V) return;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (i >= P.chunks) {
        const int64_t v = i - P.chunks;
        const uint32_t a = P.first[v], b = P.first[v + 1];
        if (b - a > SEG) return;
        add_rows<TY, VEC>(P, dy, a, b, col, acc);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] *= P.scale;
        store_vec<VEC>(dw + v * P.D + col, acc);
        return;
    }
    const uint32_t p0 = (uint32_t)i * SEG, p1 = min(p0 + SEG, P.first[P.V]);
    if (p0 >= p1) return;
    const uint32_t v0 = P.sorted[p0].x, v1 = P.sorted[p1 - 1].x;
    const uint32_t e0 = P.first[v0 + 1], a1 = P.first[v1];
    if (e0 - P.first[v0] > SEG) {
        add_rows<TY, VEC>(P, dy, p0, min(e0, p1), col, acc);
        store_vec<VEC>(P.part + (2 * i) * P.D + col, acc);
    }
    if (v1 != v0 && P.first[v1 + 1] - a1 > SEG) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        add_rows<TY, VEC>(P, dy, a1, p1, col, acc);
        store_vec<VEC>(P.part + (2 * i + 1) * P.D + col, acc);
    }
}

// One long row at most begins in each chunk: its pieces, in order.
template <typename TW, int VEC>
__global__ void __launch_bounds__(256) join_kernel(TW* dw, const __grid_constant__ Sums P) {
    const int col = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    const int64_t i = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (col >= P.D || i >= P.chunks) return;
    const uint32_t p0 = (uint32_t)i * SEG, p1 = min(p0 + SEG, P.first[P.V]);
    if (p0 >= p1) return;
    const uint32_t v = P.sorted[p1 - 1].x, a = P.first[v], b = P.first[v + 1];
    if (b - a <= SEG || a < p0) return;
    const int64_t last = (b - 1) / SEG;
    float acc[VEC];
    load_vec<VEC>(P.part + (2 * i + (a != p0)) * P.D + col, acc);
#pragma unroll 8
    for (int64_t c = i + 1; c <= last; ++c) {
        float x[VEC];
        load_vec<VEC>(P.part + 2 * c * P.D + col, x);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += x[j];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] *= P.scale;
    store_vec<VEC>(dw + (int64_t)v * P.D + col, acc);
}

// ---------------------------------------------------------------- host side
// threads of a block along the columns (any number: no kernel here shares within a warp), and blocks along them
void shape(int64_t D, int vec, dim3* threads, int* across) {
    const int64_t pieces = (D + vec - 1) / vec, x = pieces < 256 ? pieces : 256;
    *threads = dim3((unsigned)x, (unsigned)(256 / x), 1);
    *across = (int)((pieces + x - 1) / x);
}

template <typename TW, typename TY>
int forward(const void* ids, int ids64, const void* w, int64_t ldw, void* y, int64_t T, int64_t V, int64_t D,
            float scale, bool vec, cudaStream_t st) {
    dim3 threads;
    int across;
    shape(D, vec ? 8 : 1, &threads, &across);
    // four rows a thread once that still fills the GPU twice over
    const bool many = vec && T * D / 8 / 4 >= 2 * 148 * 2048;
    const int64_t rows = (many ? 4 : 1) * (int64_t)threads.y, blocks = (T + rows - 1) / rows;
    const dim3 grid((unsigned)blocks, across, 1);
    auto k = !vec ? fwd_kernel<TW, TY, 1, 1> : many ? fwd_kernel<TW, TY, 8, 4> : fwd_kernel<TW, TY, 8, 1>;
    k<<<grid, threads, 0, st>>>(ids, ids64, static_cast<const TW*>(w), ldw, static_cast<TY*>(y), T, V, (int)D, scale);
    return check_launch("concord_embedding_fwd");
}

struct Layout {
    int64_t chunk, blocks, chunks;
    size_t second, counts, first, part, total;        // offsets (the first list stands at 0)
};
Layout layout(int64_t T, int64_t V, int64_t D) {
    Layout L;
    L.chunk = SORT_CHUNK;
    while ((T + L.chunk - 1) / L.chunk > SORT_BLOCKS) L.chunk *= 2;
    L.blocks = (T + L.chunk - 1) / L.chunk;
    L.chunks = (T + SEG - 1) / SEG;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    L.second = up(T * sizeof(uint2));
    L.counts = L.second + up(T * sizeof(uint2));
    L.first = L.counts + up(L.blocks * BINS * sizeof(uint32_t));
    L.part = L.first + up((V + 1) * sizeof(uint32_t));
    L.total = L.part + up((size_t)L.chunks * 2 * D * sizeof(float));
    return L;
}

template <typename TY, typename TW>
int backward(const void* ids, int ids64, const void* dy, int64_t lddy, void* dw, int64_t T, int64_t V, int64_t D,
             float scale, int64_t padding, char* ws, bool vec, cudaStream_t st) {
    const Layout L = layout(T, V, D);
    uint2 *list[2] = {reinterpret_cast<uint2*>(ws), reinterpret_cast<uint2*>(ws + L.second)};
    uint32_t* first = reinterpret_cast<uint32_t*>(ws + L.first);
    Pass P{ids, ids64, nullptr, list[0], reinterpret_cast<uint32_t*>(ws + L.counts), T, V, padding, L.chunk, 0};
    int turn = 0;
    for (int shift = 0; shift == 0 || V >> shift; shift += DIGIT) {
        P.shift = shift;
        P.to = list[turn];
        count_kernel<<<(int)L.blocks, SORT_THREADS, 0, st>>>(P);
        place_kernel<<<(int)L.blocks, SORT_THREADS, 0, st>>>(P);
        P.from = list[turn];
        turn ^= 1;
    }
    first_kernel<<<(int)(V / 256 + 1), 256, 0, st>>>(P.from, first, T, V);
    const Sums S{P.from, first, reinterpret_cast<float*>(ws + L.part), T, V, lddy, L.chunks, (int)D, scale};
    dim3 threads;
    int across;
    shape(D, vec ? 8 : 1, &threads, &across);
    const dim3 grid((unsigned)((L.chunks + V + threads.y - 1) / threads.y), across, 1);
    auto k = vec ? sum_kernel<TY, TW, 8> : sum_kernel<TY, TW, 1>;
    k<<<grid, threads, 0, st>>>(static_cast<const TY*>(dy), static_cast<TW*>(dw), S);
    auto j = vec ? join_kernel<TW, 8> : join_kernel<TW, 1>;
    j<<<dim3((unsigned)((L.chunks + threads.y - 1) / threads.y), across, 1), threads, 0, st>>>(static_cast<TW*>(dw), S);
    return check_launch("concord_embedding_bwd");
}

int check_shape(const char* name, int32_t ta, int32_t tb, int64_t T, int64_t V, int64_t D, int64_t ld) {
    if (ta < 0 || ta > 2 || tb < 0 || tb > 2) return fail(CONCORD_EINVAL, std::string(name) + ": unknown element type");
    if (T < 0 || V <= 0 || D <= 0 || ld < D) return fail(CONCORD_ESHAPE, std::string(name) + ": bad extents or row stride");
    if (T > (1 << 30) || V > (1 << 30) || D > (1 << 20))
        return fail(CONCORD_ETOOBIG, std::string(name) + ": more than 2^30 tokens or rows, or 2^20 columns");
    return CONCORD_OK;
}

size_t esize(int32_t t) { return t == CONCORD_F32 ? 4 : 2; }

// calls F<A, B> for the two type codes
#define EMBED_TYPES(ta, tb, F, ...)                                                             \
    switch ((ta) * 3 + (tb)) {                                                                  \
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

}  // namespace embed
}  // namespace concord

using namespace concord;

extern "C" int concord_embedding_fwd(const void* ids, int32_t ids64, const void* w, int32_t w_type, int64_t ldw,
                                     void* y, int32_t y_type, int64_t T, int64_t V, int64_t D, float scale,
                                     void* stream) {
    if (int rc = embed::check_shape("concord_embedding_fwd", w_type, y_type, T, V, D, ldw)) return rc;
    if (T == 0) return CONCORD_OK;
    if (!ids || !w || !y) return fail(CONCORD_EINVAL, "concord_embedding_fwd: null pointer");
    const bool vec = D % 8 == 0 && ldw * embed::esize(w_type) % 16 == 0 && aligned(w, 16) && aligned(y, 16);
    EMBED_TYPES(w_type, y_type, embed::forward, ids, ids64, w, ldw, y, T, V, D, scale, vec, as_stream(stream))
}

extern "C" size_t concord_embedding_bwd_workspace_bytes(int64_t T, int64_t V, int64_t D) {
    if (T <= 0 || V <= 0 || D <= 0 || T > (1 << 30) || V > (1 << 30) || D > (1 << 20)) return 0;
    return embed::layout(T, V, D).total;
}

extern "C" int concord_embedding_bwd(const void* ids, int32_t ids64, const void* dy, int32_t dy_type, int64_t lddy,
                                     void* dw, int32_t dw_type, int64_t T, int64_t V, int64_t D, float scale,
                                     int64_t padding, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = embed::check_shape("concord_embedding_bwd", dy_type, dw_type, T, V, D, lddy)) return rc;
    if (!dw) return fail(CONCORD_EINVAL, "concord_embedding_bwd: null pointer");
    cudaStream_t st = as_stream(stream);
    if (T == 0) {
        cudaMemsetAsync(dw, 0, (size_t)V * D * embed::esize(dw_type), st);
        return check_launch("concord_embedding_bwd");
    }
    if (!ids || !dy) return fail(CONCORD_EINVAL, "concord_embedding_bwd: null pointer");
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < concord_embedding_bwd_workspace_bytes(T, V, D))
        return fail(CONCORD_EWORKSPACE, "concord_embedding_bwd: workspace too small, or not 16-byte aligned");
    const bool vec = D % 8 == 0 && lddy * embed::esize(dy_type) % 16 == 0 && aligned(dy, 16) && aligned(dw, 16);
    EMBED_TYPES(dy_type, dw_type, embed::backward, ids, ids64, dy, lddy, dw, T, V, D, scale, padding,
                static_cast<char*>(workspace), vec, st)
}
