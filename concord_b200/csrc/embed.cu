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
// order, without atomics on them: the same bits on every run.  Up to 65,536 tokens
// are sorted by one cluster of 8 blocks in its shared memory, in one launch;
// more go through memory, two launches a digit.  The sorted tokens are cut into
// chunks of 32, summed side by side, each chunk's rows in order; a row that begins and
// ends in one is finished there, the pieces of the others are joined in order
// by a second kernel.  Rows of no token, which the sort's bit of each row tells, are cleared by the same launch's other blocks.
#include <cooperative_groups.h>

#include "common.cuh"
#include "vec.cuh"

namespace concord {
namespace embed {

constexpr int SEG = 32;                    // sorted tokens of a chunk
constexpr int DIGIT = 9, BINS = 1 << DIGIT;
constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32;
constexpr int64_t SORT_CHUNK = 4096;       // tokens of a sorting block, and more where blocks would pass
constexpr int64_t SORT_BLOCKS = 512;       // this number: each of them reads all blocks' counts

// The columns that a thread holds: 8 neighbours (VEC), or 4 that are `step` apart,
// for rows that do not start on 16 bytes (a column that is not there reads the last one).
template <bool VEC> struct Cols {
    static constexpr int N = VEC ? 8 : 4;
    int at[VEC ? 1 : N];
    int count;                            // that are there
    __device__ __forceinline__ Cols(int block, int thread, int step, int D) {
        if constexpr (VEC) {
            at[0] = (block * step + thread) * 8;
            count = at[0] < D ? 8 : 0;
        } else {
            const int first = block * step * N + thread;
            count = 0;
#pragma unroll
            for (int c = 0; c < N; ++c) {
                at[c] = min(first + c * step, D - 1);
                count += first + c * step < D;
            }
        }
    }
};
// a row's columns as they come from memory
template <typename T, bool VEC> struct Raw {
    static constexpr int N = Cols<VEC>::N, W = VEC ? 8 * (int)sizeof(T) / 4 : N;
    uint32_t v[W];
    __device__ __forceinline__ void load(const T* row, const Cols<VEC>& C) {
        if constexpr (VEC) {
            uint4 a, b;
            if constexpr (sizeof(T) == 4) load32(row + C.at[0], a, b);
            else a = *reinterpret_cast<const uint4*>(row + C.at[0]);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            if constexpr (sizeof(T) == 4) { v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w; }
        } else {
#pragma unroll
            for (int c = 0; c < N; ++c) v[c] = __float_as_uint(to_f32(row[C.at[c]]));
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (!VEC || sizeof(T) == 4) return __uint_as_float(v[i]);
        else {
            const float2 f = unpack2(v[i / 2], T());
            return i & 1 ? f.y : f.x;
        }
    }
};
template <typename T, bool VEC> __device__ __forceinline__ void store_cols(T* row, const Cols<VEC>& C, const float* v) {
    if constexpr (VEC && sizeof(T) == 4) store32(row + C.at[0], Pack16<T>::pack(v), Pack16<T>::pack(v + 4));
    else if constexpr (VEC) store_vec<8>(row + C.at[0], v);
    else {
#pragma unroll
        for (int c = 0; c < Cols<VEC>::N; ++c)
            if (c < C.count) row[C.at[c]] = from_f32<T>(v[c]);
    }
}

// ---------------------------------------------------------------- forward
// A thread holds its columns of ROWS rows.
template <typename TW, typename TY, bool VEC, int ROWS>
__global__ void __launch_bounds__(256)
    fwd_kernel(const void* ids, int ids64, const TW* w, int64_t ldw, TY* y, int64_t T, int64_t V, int D, float scale) {
    const Cols<VEC> C(blockIdx.y, threadIdx.x, blockDim.x, D);
    const int64_t t0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * ROWS;
    if (C.count == 0 || t0 >= T) return;
    int64_t id[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        id[r] = -1;
        if (t0 + r < T)
            id[r] = ids64 ? static_cast<const int64_t*>(ids)[t0 + r] : (int64_t)static_cast<const int32_t*>(ids)[t0 + r];
    }
    Raw<TW, VEC> raw[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (id[r] >= 0 && id[r] < V) raw[r].load(w + id[r] * ldw, C);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (t0 + r >= T) continue;
        const bool there = id[r] >= 0 && id[r] < V;
        float v[Cols<VEC>::N];
#pragma unroll
        for (int j = 0; j < Cols<VEC>::N; ++j) v[j] = there ? raw[r].get(j) * scale : 0.f;
        store_cols<TY, VEC>(y + (t0 + r) * D, C, v);
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

// The whole sort by one cluster: block r holds places [r n, (r + 1) n)
// of the list, n a power of two.  A digit takes two exchanges: the blocks' counts,
// and the items, stored straight into the shared memory of the block that owns their place.
constexpr int CLUSTER = 8, CT = 1024, CW = CT / 32;
constexpr int64_t CLUSTER_MOST = 8192;                       // items of a block
struct ClusterSort {
    const void* ids;
    int ids64;
    int64_t V, padding;
    int T, n, log_n, passes, digit;       // digit: bits of a pass, up to 9
    uint2* sorted;
    uint32_t* end;                                // places of rows; behind them what counts for none
    uint32_t* some;                               // a bit a row: it has tokens
};
// One place of the sorted list, its neighbours' keys beside it: the row's bit, and where rows end.
__device__ __forceinline__ void mark(uint32_t* some, uint32_t* end, int64_t V, int64_t T, int64_t i, uint32_t before, uint32_t key, uint32_t after) {
    if (key >= V) {
        if (i == 0) *end = 0;
        return;
    }
    if (before != key) atomicOr(&some[key / 32], 1u << (key % 32));
    if (i + 1 == T || after >= V) *end = (uint32_t)(i + 1);
}
__global__ void __launch_bounds__(256) mark_kernel(const uint2* sorted, uint32_t* some, uint32_t* end, int64_t T, int64_t V) {
    const int64_t i = blockIdx.x * 256ll + threadIdx.x;
    if (i < T) mark(some, end, V, T, i, i ? sorted[i - 1].x : ~0u, sorted[i].x, i + 1 < T ? sorted[i + 1].x : ~0u);
}
size_t cluster_smem(int n) { return (size_t)2 * n * sizeof(uint2) + CW * BINS * sizeof(uint16_t) + 2 * BINS * sizeof(uint32_t); }

__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(CT) cluster_sort_kernel(const __grid_constant__ ClusterSort P) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ uint32_t sums[CW];
    uint2* list[2] = {reinterpret_cast<uint2*>(raw), reinterpret_cast<uint2*>(raw) + P.n};
    uint16_t* run_at = reinterpret_cast<uint16_t*>(list[1] + P.n);         // [warp][digit]
    uint32_t* mine = reinterpret_cast<uint32_t*>(run_at + CW * BINS);      // this block's counts
    uint32_t* base = mine + BINS;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int begin = rank * P.n, have = max(0, min(P.n, P.T - begin));    // places of this block, and items in them
    const int run = max(32, P.n / CW), r0 = min(warp * run, have), r1 = min(r0 + run, have);
    for (int i = threadIdx.x; i < have; i += CT)
        list[0][i] = make_uint2(key_of(P.ids, P.ids64, begin + i, P.V, P.padding), (uint32_t)(begin + i));
    for (int64_t i = rank * CT + threadIdx.x; i < (P.V + 31) / 32; i += CLUSTER * CT) P.some[i] = 0;
    const int bins = 1 << P.digit;
    for (int pass = 0; pass < P.passes; ++pass) {
        const uint2* from = list[pass & 1];
        const int shift = pass * P.digit;
        for (int i = threadIdx.x; i < CW * bins / 8; i += CT) reinterpret_cast<uint4*>(run_at)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        uint16_t* at = run_at + warp * bins;
        for (int t = r0; t < r1; t += 32) {
            const bool is = t + lane < r1;
            const uint32_t d = is ? (from[t + lane].x >> shift) & (bins - 1) : BINS;
            const uint32_t same = __match_any_sync(0xffffffffu, d);
            if (is && lane == __ffs(same) - 1) at[d] += (uint16_t)__popc(same);
            __syncwarp();
        }
        __syncthreads();
        if (threadIdx.x < bins) {                 // each run's first place among the block's of this digit
            uint32_t c[CW], n = 0;
#pragma unroll
            for (int w = 0; w < CW; ++w) c[w] = run_at[w * bins + threadIdx.x];
#pragma unroll
            for (int w = 0; w < CW; ++w) {
                run_at[w * bins + threadIdx.x] = (uint16_t)n;
                n += c[w];
            }
            mine[threadIdx.x] = n;
        }
        cluster.sync();
        uint32_t all = 0, before = 0;
        if (threadIdx.x < bins) {
#pragma unroll
            for (int r = 0; r < CLUSTER; ++r) {
                const uint32_t c = cluster.map_shared_rank(mine, r)[threadIdx.x];
                all += c;
                before += r < rank ? c : 0;
            }
        }
        uint32_t incl = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        if (threadIdx.x < bins) {
            uint32_t b = incl - all + before;
#pragma unroll
            for (int w = 0; w < BINS / 32; ++w) b += w < warp ? sums[w] : 0;
            base[threadIdx.x] = b;
        }
        __syncthreads();
        uint2* to = list[(pass + 1) & 1];
        for (int t = r0; t < r1; t += 32) {
            const bool is = t + lane < r1;
            const uint2 it = is ? from[t + lane] : make_uint2(0, 0);
            const uint32_t d = is ? (it.x >> shift) & (bins - 1) : BINS;
            const uint32_t same = __match_any_sync(0xffffffffu, d);
            if (is) {
                const uint32_t p = base[d] + at[d] + __popc(same & ((1u << lane) - 1));
                cluster.map_shared_rank(to, p >> P.log_n)[p & (P.n - 1)] = it;
            }
            __syncwarp();
            if (is && lane == __ffs(same) - 1) at[d] += (uint16_t)__popc(same);
            __syncwarp();
        }
        cluster.sync();
    }
    const uint2* done = list[P.passes & 1];
    for (int i = threadIdx.x; i < have; i += CT) {
        const uint2 it = done[i];
        P.sorted[begin + i] = it;
        const int n = begin + i + 1;
        const uint32_t after = n == P.T ? ~0u : i + 1 < have ? done[i + 1].x : cluster.map_shared_rank(const_cast<uint2*>(done), rank + 1)[0].x;
        mark(P.some, P.end, P.V, P.T, begin + i, i > 0 ? done[i - 1].x : ~0u, it.x, after);
    }
    cluster.sync();                               // nobody leaves while its list is read
}

// ---------------------------------------------------------------- sums
struct Sums {
    const uint2* sorted;
    const uint32_t *end, *some;
    float* part;              // [chunks][2][D]: a row's piece that goes on from the chunk before, one that begins here and goes on
    int64_t T, V, lddy;
    int64_t chunks;
    int D;
    float scale;
};

// Blocks of two kinds: chunks, one a row of threads (their loads run AHEAD
// tokens before their sums), then rows of no token to clear, CLEAR a thread.  Chunks
// first, as they wait for memory and the others only fill it (16384 tokens, 32000 x 2048
// fp32: 49 us, 6.7 TB/s; both kinds mixed 56; with 16 bytes a store, which leave half a sector
// of 8 columns of fp32 to the next one, 67).
constexpr int CLEAR = 8;
template <typename TY, typename TW, bool VEC>
__global__ void __launch_bounds__(256, 3) sum_kernel(const TY* dy, TW* dw, const __grid_constant__ Sums P, int chunk_blocks) {
    constexpr int N = Cols<VEC>::N;
    const Cols<VEC> C(blockIdx.y, threadIdx.x, blockDim.x, P.D);
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    if (C.count == 0) return;
    if (blockIdx.x >= chunk_blocks) {
        const int64_t v0 = (blockIdx.x - chunk_blocks) * (int64_t)(CLEAR * blockDim.y) + threadIdx.y;
        bool none[CLEAR];
#pragma unroll
        for (int r = 0; r < CLEAR; ++r) {
            const int64_t v = v0 + r * blockDim.y;
            none[r] = v < P.V && !(P.some[v / 32] >> (v % 32) & 1);
        }
#pragma unroll
        for (int r = 0; r < CLEAR; ++r)
            if (none[r]) store_cols<TW, VEC>(dw + (v0 + r * blockDim.y) * P.D, C, acc);
        return;
    }
    constexpr int AHEAD = !VEC || sizeof(TY) == 2 ? 8 : 4;
    const int64_t i = blockIdx.x * (int64_t)blockDim.y + threadIdx.y;
    const uint32_t end = *P.end;
    if (i >= P.chunks || (uint32_t)i * SEG >= end) return;
    const uint32_t p0 = (uint32_t)i * SEG, p1 = min(p0 + SEG, end);
    const uint2* at = P.sorted;
    Raw<TY, VEC> ring[AHEAD];
    uint32_t key[AHEAD];                                  // their rows
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
        const uint2 it = at[min(p0 + k, p1 - 1)];
        key[k] = it.x;
        ring[k].load(dy + it.y * P.lddy, C);
    }
    bool before = p0 > 0 && at[p0 - 1].x == key[0];       // the row goes on from the chunk before
    const uint32_t after = p1 < end ? at[p1].x : (uint32_t)P.V;
    for (uint32_t p = p0; p < p1; p += AHEAD) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (p + k >= p1) break;
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] += ring[k].get(j);
            const uint32_t v = key[k];
            const uint2 it = at[min(p + k + AHEAD, p1 - 1)];      // (the last one again where there are no more)
            key[k] = it.x;
            ring[k].load(dy + it.y * P.lddy, C);
            const bool last = p + k + 1 == p1;
            const uint32_t next = last ? after : key[(k + 1) % AHEAD];
            if (next == v && !last) continue;
            if (!before && next != v) {
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] *= P.scale;
                store_cols<TW, VEC>(dw + (int64_t)v * P.D, C, acc);
            } else {
                store_cols<float, VEC>(P.part + (2 * i + !before) * P.D, C, acc);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = 0.f;
            before = false;
        }
    }
}

// How many of the chunks behind i, below `chunks`, begin with row v, by a whole warp: the next
// 32, then 32 places of what is left at once.
__device__ __forceinline__ int64_t going_on(const uint2* sorted, int64_t i, int64_t chunks, uint32_t v) {
    int64_t known = 0, len = chunks - i - 1, step = 1;          // the answer is in [known, known + len]
    uint32_t lane;                                              // (blocks have two dimensions)
    asm("mov.u32 %0, %%laneid;" : "=r"(lane));
    while (len > 0) {
        const int64_t at = lane * step;
        const bool on = at < len && sorted[(i + 1 + known + at) * SEG].x == v;
        const int64_t k = __popc(__ballot_sync(0xffffffffu, on));          // lanes 0 .. k - 1
        if (k == 0) break;
        const int64_t from = (k - 1) * step + 1;
        len = k < 32 ? min(step - 1, len - from) : len - from;
        known += from;
        step = (len + 31) / 32;
    }
    return known;
}

// One row at most begins in a chunk and goes on: its pieces in order, eight runs of
// them side by side, the runs' sums in order again.  Most blocks find nothing to
// do, so that what counts is how many fit (eight an SM, two pieces at once: 9.9 us for 16384
// tokens and 2048 columns; four and four 12.4).
constexpr int JOIN = 8;
template <typename TW, bool VEC>
__global__ void __launch_bounds__(256, 8) join_kernel(TW* dw, const __grid_constant__ Sums P) {
    constexpr int N = Cols<VEC>::N;
    __shared__ float runs[JOIN][32][N];
    const int64_t i = blockIdx.x;
    const uint32_t end = *P.end, p0 = (uint32_t)i * SEG, p1 = p0 + SEG;       // (p1 is below T: the last chunk has no block)
    const uint32_t v = P.sorted[p1 - 1].x, next = P.sorted[p1].x, before = P.sorted[max(p0, 1u) - 1].x;
    if (p1 >= end || next != v || (p0 > 0 && before == v)) return;            // nothing goes on, or it began before
    const int64_t pieces = going_on(P.sorted, i, min(P.chunks, ((int64_t)end + SEG - 1) / SEG), v);
    const Cols<VEC> C(blockIdx.y, threadIdx.x, 32, P.D);
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    if (C.count > 0) {
        const int64_t c0 = i + 1 + pieces * threadIdx.y / JOIN, c1 = i + 1 + pieces * (threadIdx.y + 1) / JOIN;
        if (threadIdx.y == 0) {
            Raw<float, VEC> x;
            x.load(P.part + (2 * i + 1) * P.D, C);
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = x.get(j);
        }
#pragma unroll 2
        for (int64_t c = c0; c < c1; ++c) {
            Raw<float, VEC> x;
            x.load(P.part + 2 * c * P.D, C);
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] += x.get(j);
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) runs[threadIdx.y][threadIdx.x][j] = acc[j];
    __syncthreads();
    if (threadIdx.y == 0 && C.count > 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            for (int k = 1; k < JOIN; ++k) acc[j] += runs[k][threadIdx.x][j];
            acc[j] *= P.scale;
        }
        store_cols<TW, VEC>(dw + (int64_t)v * P.D, C, acc);
    }
}

// ---------------------------------------------------------------- host side
// threads of a block along the columns, and blocks along them
void shape(int64_t D, int each, dim3* threads, int* across) {
    const int64_t pieces = (D + each - 1) / each, x = pieces < 256 ? pieces : 256;
    *threads = dim3((unsigned)x, (unsigned)(256 / x), 1);
    *across = (int)((pieces + x - 1) / x);
}

template <typename TW, typename TY>
int forward(const void* ids, int ids64, const void* w, int64_t ldw, void* y, int64_t T, int64_t V, int64_t D,
            float scale, bool vec, cudaStream_t st) {
    dim3 threads;
    int across;
    shape(D, vec ? 8 : 4, &threads, &across);
    // four rows a thread once that still fills the GPU twice over
    const bool many = T * D / (vec ? 8 : 4) / 4 >= 2 * 148 * 2048;
    const int64_t rows = (many ? 4 : 1) * (int64_t)threads.y, blocks = (T + rows - 1) / rows;
    const dim3 grid((unsigned)blocks, across, 1);
    auto k = vec ? (many ? fwd_kernel<TW, TY, true, 4> : fwd_kernel<TW, TY, true, 1>)
                 : (many ? fwd_kernel<TW, TY, false, 4> : fwd_kernel<TW, TY, false, 1>);
    k<<<grid, threads, 0, st>>>(ids, ids64, static_cast<const TW*>(w), ldw, static_cast<TY*>(y), T, V, (int)D, scale);
    return check_launch("concord_embedding_fwd");
}

struct Layout {
    int64_t chunk, blocks, chunks;
    size_t second, counts, end, some, part, total;        // offsets (the first list stands at 0)
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
    L.end = L.counts + up(L.blocks * BINS * sizeof(uint32_t));
    L.some = L.end + up(sizeof(uint32_t));
    L.part = L.some + up((V + 31) / 32 * sizeof(uint32_t));
    L.total = L.part + up((size_t)L.chunks * 2 * D * sizeof(float));
    return L;
}

template <typename TY, typename TW>
int backward(const void* ids, int ids64, const void* dy, int64_t lddy, void* dw, int64_t T, int64_t V, int64_t D,
             float scale, int64_t padding, char* ws, bool vec, cudaStream_t st) {
    const Layout L = layout(T, V, D);
    uint2 *list[2] = {reinterpret_cast<uint2*>(ws), reinterpret_cast<uint2*>(ws + L.second)};
    uint32_t *end = reinterpret_cast<uint32_t*>(ws + L.end), *some = reinterpret_cast<uint32_t*>(ws + L.some);
    const uint2* sorted = list[0];
    int passes = 1;
    while (V >> (passes * DIGIT)) ++passes;
    if (T <= CLUSTER * CLUSTER_MOST) {
        int bits = 1;
        while (V >> bits) ++bits;
        ClusterSort C{ids, ids64, V, padding, (int)T, 32, 5, passes, (bits + passes - 1) / passes, list[0], end, some};
        if (C.digit < 3) C.digit = 3;             // (whole 16-byte pieces of counts)
        while ((int64_t)C.n * CLUSTER < T) {
            C.n *= 2;
            ++C.log_n;
        }
        const size_t smem = cluster_smem(C.n);
        cudaError_t e = cudaFuncSetAttribute(cluster_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)cluster_smem(CLUSTER_MOST));
        if (e != cudaSuccess) return fail(CONCORD_ELAUNCH, std::string("concord_embedding_bwd: ") + cudaGetErrorString(e));
        cluster_sort_kernel<<<CLUSTER, CT, smem, st>>>(C);
    } else {
        Pass P{ids, ids64, nullptr, list[0], reinterpret_cast<uint32_t*>(ws + L.counts), T, V, padding, L.chunk, 0};
        for (int pass = 0; pass < passes; ++pass) {
            P.shift = pass * DIGIT;
            P.to = list[pass & 1];
            count_kernel<<<(int)L.blocks, SORT_THREADS, 0, st>>>(P);
            place_kernel<<<(int)L.blocks, SORT_THREADS, 0, st>>>(P);
            P.from = P.to;
        }
        sorted = P.from;
        cudaMemsetAsync(some, 0, (V + 31) / 32 * sizeof(uint32_t), st);
        mark_kernel<<<(unsigned)((T + 255) / 256), 256, 0, st>>>(sorted, some, end, T, V);
    }
    const Sums S{sorted, end, some, reinterpret_cast<float*>(ws + L.part), T, V, lddy, L.chunks, (int)D, scale};
    dim3 threads;
    int across;
    shape(D, vec ? 8 : 4, &threads, &across);
    const int chunk_blocks = (int)((L.chunks + threads.y - 1) / threads.y);
    const int clear_blocks = (int)((V + CLEAR * threads.y - 1) / (CLEAR * threads.y));
    auto k = vec ? sum_kernel<TY, TW, true> : sum_kernel<TY, TW, false>;
    k<<<dim3((unsigned)(chunk_blocks + clear_blocks), across, 1), threads, 0, st>>>(
        static_cast<const TY*>(dy), static_cast<TW*>(dw), S, chunk_blocks);
    if (L.chunks > 1) {
        auto j = vec ? join_kernel<TW, true> : join_kernel<TW, false>;
        const int wide = 32 * (vec ? 8 : 4);
        j<<<dim3((unsigned)(L.chunks - 1), (unsigned)((D + wide - 1) / wide), 1), dim3(32, JOIN, 1), 0, st>>>(
            static_cast<TW*>(dw), S);
    }
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
// whether rows are runs of 8 columns, each a whole access
bool runs(const void* p, int32_t t, int64_t ld) { return ld % 8 == 0 && aligned(p, 8 * esize(t)); }

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
    const bool vec = embed::runs(w, w_type, ldw) && embed::runs(y, y_type, D);
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
    const bool vec = embed::runs(dy, dy_type, lddy) && embed::runs(dw, dw_type, D) && aligned(workspace, 32);
    EMBED_TYPES(dy_type, dw_type, embed::backward, ids, ids64, dy, lddy, dw, T, V, D, scale, padding,
                static_cast<char*>(workspace), vec, st)
}
