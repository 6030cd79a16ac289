// attention.cu — attention over packed sequences of different lengths, with
// grouped heads, causal or not, forward and backward.
//
//   s_ij = scale q_i . k_j           (j <= i + Lk - Lq where causal)
//   o_i  = sum_j exp(s_ij - m_i) v_j / l_i,  lse_i = m_i + log l_i
//   p_ij = exp(s_ij - lse_i),  delta_i = do_i . o_i
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// (sums over i also run over the query heads that share the key head).
//
// Every product runs on tcgen05 (bf16 or fp16 operands, fp32 accumulators in
// tensor memory); tiles are 128 rows of up to 128 columns, loaded by TMA.  A
// head dimension below 64 or 128 is filled up with zeros by the loads.  p and
// ds are rounded to the operands' type for their second product, as the tensor
// cores read 16 bits; maxima, sums, lse and delta stay in fp32.
//
// Warp roles: warp 0 loads, warp 1 issues the products (and zeroes the rows of
// a tile that lie beyond its sequence: they belong to another sequence, or to
// nobody, and 0 * NaN is NaN), warps 4-11 do the softmax arithmetic, one row
// of 128 a thread in the forward, half a row in the backward.  Every wait on a
// barrier is bounded (2 s, see tc.cuh).  Where one runs out the loads and the
// products stop; the softmax warps go on through their loop on whatever is there
// (they never branch on a wait: their tcgen05 instructions want whole warps),
// and the block waits (bounded again) for its loads and products in flight,
// fills its results with NaN, frees its tensor memory and returns.  The next
// call finds the host's error word and fails.
//
// The backward is two kernels without atomics, so gradients are the same bits
// on every run: one owns 128 rows of q and walks the keys (dq, and delta), the
// other owns 128 keys and walks the queries of every head that shares them (dk,
// dv).  Both compute s and do . v, seven products in place of five; the
// alternative adds dq atomically into an fp32 buffer, which is another order of
// the sums on every run, and a pass to clear and one to round it.
#include <cuda.h>
#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "tc.cuh"
#include "vec.cuh"

namespace concord {
int bind_current_context(const char* name);

namespace attn {

using namespace tc;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 384;

struct Params {
    const int* cuq;       // [B + 1] first rows of the sequences (queries)
    const int* cuk;       // [B + 1] (keys)
    int B;
    int Tq, Tk;
    int H, G;             // query heads, query heads of one key head
    int D;
    int causal;
    float scale, scale2;  // scale, scale * log2(e)
    void* o;              // [Tq, H, D]
    void* rest;           // [Tq, H, D]: what o's rounding left over, for delta (NULL: not kept)
    float* lse;           // [H, Tq]
    const void* dout;     // row strides of dout in elements
    int64_t do_ts, do_hs;
    float* delta;         // [H, Tq]
    void *dq, *dk, *dv;
    float* part;          // splits > 1: [splits][dk, dv][Tk, key heads, D] in fp32
    int splits, per;      // parts of a key head's query heads, and heads of a part
    // fp16 backward (see lift): v, the largest |v| of each part of a sequence's keys
    // [B][key heads][chunks], and the largest sum of |dout| of a row [B][H]
    const void* v;
    int64_t v_ts, v_hs;
    float* vmax;
    int chunks;
    int* dmax;            // (fp32 of no sign, ordered as whole numbers)
    int* err;             // error word of the device, and the host's
    int* err_host;
};

// a block's work: sequence bounds (clamped to the tensors) and tile
struct Work {
    int q0, lq, k0, lk;   // first row and length of the sequence
    int tile;             // -1: none left; then `spare` of `spares` blocks zero the rows of no sequence
    int spare, spares;
    int first, last;      // rows [0, first) and [last, T) belong to no sequence
    int seq;              // its number
};

// The t-th tile of `rows` rows, sequences in order, a sequence's last tile
// first where `back` (causal queries: the longest first).  Whole warp, four
// sequences a lane.
__device__ __forceinline__ void find_tile(const Params& P, bool keys, int t, int tiles_bound, int rows, bool back,
                                          Work* w) {
    constexpr int EACH = 4;
    const int lane = threadIdx.x & 31;
    const int* cu = keys ? P.cuk : P.cuq;
    const int T = keys ? P.Tk : P.Tq;
    int before = 0;
    for (int b0 = 0; b0 < P.B; b0 += 32 * EACH) {
        const int b = b0 + lane * EACH;
        int at[EACH + 1], n[EACH], sum = 0;
#pragma unroll
        for (int k = 0; k <= EACH; ++k) at[k] = min(max(b + k <= P.B ? cu[b + k] : INT_MAX, 0), T);
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            n[k] = b + k < P.B ? (max(at[k + 1] - at[k], 0) + rows - 1) / rows : 0;
            sum += n[k];
        }
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        int lo = before + incl - sum;
        const bool mine = t >= lo && t < lo + sum;
        if (mine) {
            const int* other = keys ? P.cuq : P.cuk;
            const int To = keys ? P.Tq : P.Tk;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                if (t >= lo && t < lo + n[k]) {
                    const int s = at[k], len = max(at[k + 1] - s, 0);
                    const int so = min(max(other[b + k], 0), To), lo2 = max(min(max(other[b + k + 1], 0), To) - so, 0);
                    w->q0 = keys ? so : s;
                    w->lq = keys ? lo2 : len;
                    w->k0 = keys ? s : so;
                    w->lk = keys ? len : lo2;
                    w->seq = b + k;
                    w->tile = back ? n[k] - 1 - (t - lo) : t - lo;
                }
                lo += n[k];
            }
        }
        if (__any_sync(0xffffffffu, mine)) return;
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
        w->tile = -1;
        w->spare = t - before;
        w->spares = tiles_bound - before;
        w->first = min(max(cu[0], 0), T);
        w->last = min(max(cu[P.B], w->first), T);
    }
}

// zero out[row, head, :] for the rows of no sequence (16-byte stores)
__device__ __forceinline__ void zero_uncovered(void* out, const Work& w, int T, int heads, int head, int D) {
    const int chunks = D / 8, rows = w.first + (T - w.last);
    for (int64_t i = (int64_t)w.spare * blockDim.x + threadIdx.x; i < (int64_t)rows * chunks;
         i += (int64_t)w.spares * blockDim.x) {
        const int r = (int)(i / chunks), c = (int)(i % chunks);
        const int64_t row = r < w.first ? r : w.last + (r - w.first);
        reinterpret_cast<uint4*>(out)[(row * heads + head) * chunks + c] = make_uint4(0, 0, 0, 0);
    }
}

__device__ __forceinline__ uint8_t* align1024(uint8_t* p) {
    return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~(uintptr_t)1023);
}

// Behind the barriers: the tensor memory's address, and 12 bytes on the block's
// work, which is then read word by word: read in vectors its fields take
// neighbouring registers (8 x 2048: forward 174 -> 191 us, dq 229 -> 240).
__device__ __forceinline__ uint32_t* slot_of(uint64_t* bars, int n) { return reinterpret_cast<uint32_t*>(bars + n); }
__device__ __forceinline__ Work* work_of(uint64_t* bars, int n) { return reinterpret_cast<Work*>(slot_of(bars, n) + 3); }

// `rows` rows of `bytes`, the first of them the `row`-th such, `step` of them apart
__device__ __forceinline__ void spoil(void* out, int64_t row, int rows, int64_t step, int bytes) {
    const int words = bytes / 4;
    uint32_t* at = static_cast<uint32_t*>(out) + row * words;
#pragma unroll 1
    for (int64_t i = threadIdx.x & 31; i < (int64_t)rows * words; i += 32) at[i / words * step * words + i % words] = 0x7fff7fffu;
}
// What the product warp does at the end of a block whose waits ran out (looked
// for by all warps it cost the forward of 64 x 256 tokens 2 us of 32): the host
// is told, the products in flight end (bounded), and NaN (of any type) takes the results'
// place.  KIND 0: forward, 1: dq, 2: dk and dv; BARS: where its NBARS barriers
// stand, the last one for this (nothing of the kernel's is kept in registers for it).
template <int KIND, int BARS, int NBARS> __device__ __noinline__ void spoil_block(const Params& P) {
    extern __shared__ uint8_t raw[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(align1024(raw) + BARS);
    const Work* work = work_of(bars, NBARS);
    const uint32_t drained = smem_u32(bars + NBARS - 1);
    if ((threadIdx.x & 31) == 0) {
        *reinterpret_cast<volatile int*>(P.err_host) = *reinterpret_cast<volatile int*>(P.err);
        __threadfence_system();
    }
    __syncwarp();
    mma_commit(drained, elect_one());
    Patience patience;
    while (!__all_sync(0xffffffffu, mbar_try(drained, 0)) && !__any_sync(0xffffffffu, patience.over(P.err))) {}
    const Work w = *work;
    if (KIND < 2) {
        const int r0 = w.tile * (KIND ? 128 : 256), rows = min(KIND ? 128 : 256, w.lq - r0), head = blockIdx.x % P.H;
        const int64_t first = (int64_t)w.q0 + r0, row = first * P.H + head;
        spoil(KIND ? P.dq : P.o, row, rows, P.H, P.D * 2);
        if (!KIND && P.rest) spoil(P.rest, row, rows, P.H, P.D * 2);
        spoil(KIND ? P.delta : P.lse, (int64_t)head * P.Tq + first, rows, 1, 4);
    } else {
        const int HK = P.H / P.G, k0 = w.tile * 128, rows = min(128, w.lk - k0);
        const int64_t row = ((int64_t)w.k0 + k0) * HK + blockIdx.x % HK, all = (int64_t)P.Tk * HK * P.D;
        float* part = P.part + 2 * all * (blockIdx.x / HK % P.splits);
        const bool parts = P.splits > 1;
        spoil(parts ? part : P.dk, row, rows, HK, P.D * (parts ? 4 : 2));
        spoil(parts ? part + all : P.dv, row, rows, HK, P.D * (parts ? 4 : 2));
    }
}

// COLS columns of the warp's 32 rows in tensor memory, times f (one factor a
// row), to `rows` rows of `out` (row stride in elements), as columns col0 .. of
// D.  A lane holds a row, so stores straight from the registers touch 32 rows
// each (measured 6500 cycles a tile); the rows go through the warp's own part
// `stage` of a tile that no product reads any more, 16-byte pieces exchanged so
// that neither direction meets a bank twice, and leave as whole lines.  With
// REST also what the rounding left over, to `rest` (unless null).
template <typename T, int COLS, bool REST = false>
__device__ __forceinline__ void store_rows(uint32_t tm, uint32_t stage, float f, T* out, int64_t stride, int col0,
                                           int D, int rows, T* rest = nullptr) {
    constexpr int E = Pack16<T>::N, CH = COLS / E;             // elements of 16 bytes, such pieces of a row
    const int lane = threadIdx.x & 31;
    auto place = [](int row, int c) -> uint32_t { return (row * CH + (c ^ (CH >= 8 ? row & 7 : (row >> 1) & 3))) * 16; };
#pragma unroll
    for (int pass = 0; pass < (REST ? 2 : 1); ++pass) {
        if (pass && !rest) break;
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
            uint32_t r[32];
            ld32(tm + c, r);
            wait_ld();
#pragma unroll
            for (int k = 0; k < 32 / E; ++k) {
                float v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = __uint_as_float(r[k * E + e]) * f;
                uint4 o = Pack16<T>::pack(v);
                if (pass) {
                    float h[E];
                    Pack16<T>::unpack(o, h);
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] -= h[e];
                    o = Pack16<T>::pack(v);
                }
                sts16(stage + place(lane, c / E + k), o);
            }
        }
        __syncwarp();
        T* dst = pass ? rest : out;
#pragma unroll
        for (int i = 0; i < CH; i += 4) {          // four loads on their way at a time
            uint4 o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = (i + k) * 32 + lane;
                o[k] = lds16(stage + place(at / CH, at % CH));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = (i + k) * 32 + lane, row = at / CH, col = col0 + at % CH * E;
                if (row < rows && col < D) *reinterpret_cast<uint4*>(dst + row * stride + col) = o[k];
            }
        }
        __syncwarp();
    }
}

// ---------------------------------------------------------------- forward
// A block owns 256 query rows (two tiles, one softmax warpgroup each) of one
// head; K and V tiles go through one ring and serve both.  Tensor memory: S_0,
// S_1 (128 columns each), O_0, O_1 and, with heads up to 64, P_0, P_1 (16-bit
// pairs): the next S is then computed as soon as the present one is read.  With
// 128 there is no room, P_i takes the first 64 columns of S_i once they have
// been read, and the next S waits for P V.  The product P V begins with the
// first 64 keys while the exponentials of the others still run.
// Bound by the chain of a tile, S -> softmax -> P V -> next S, of which two run
// against each other (2900 cycles a pair of 128 x 128 blocks, 2048 of products);
// short sequences by a block's start and end.  8 x 2048 tokens, 16 heads of 128,
// causal: 166 us, 828 TFLOP/s; one sequence of 8191: 241 us, 1140 TFLOP/s.
template <int DP> struct Fwd {
    static constexpr int TILE = 256 * DP;               // bytes of 128 rows
    static constexpr int ST = DP == 128 ? 5 : 8;        // ring of K and V tiles
    static constexpr int RING = 2 * TILE;
    static constexpr int BARS = RING + ST * TILE;
    static constexpr size_t SMEM = BARS + BARRIERS + 1024;
};

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1)
    fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
               const __grid_constant__ CUtensorMap mv, const __grid_constant__ Params P) {
    using C = Fwd<DP>;
    constexpr int ST = C::ST, TILE = C::TILE;
    constexpr int BF = sizeof(T) == 2 && !__is_same(T, __half);
    extern __shared__ uint8_t raw[];
    uint8_t* smem = align1024(raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BARS);
    constexpr int NBARS = 2 * ST + 13;
    uint32_t* slot = slot_of(bars, NBARS);
    Work* work = work_of(bars, NBARS);
    const uint32_t base = smem_u32(smem), bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (ST + s); };
    auto q_full = [&](int i) { return bar0 + 8u * (2 * ST + i); };
    auto s_full = [&](int i) { return bar0 + 8u * (2 * ST + 2 + i); };
    auto p_full = [&](int i) { return bar0 + 8u * (2 * ST + 4 + i); };
    auto pv_done = [&](int i) { return bar0 + 8u * (2 * ST + 6 + i); };
    auto p_half = [&](int i) { return bar0 + 8u * (2 * ST + 8 + i); };
    auto s_free = [&](int i) { return bar0 + 8u * (2 * ST + 10 + i); };
    const uint32_t drained = bar0 + 8u * (2 * ST + 12);
    constexpr bool APART = DP == 64;             // P has columns of its own
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.x % P.H, t = blockIdx.x / P.H, kvh = head / P.G;

    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < ST; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
            for (int i = 0; i < 2; ++i) {
                mbar_init(q_full(i), 1); mbar_init(s_full(i), 1); mbar_init(p_full(i), 128); mbar_init(pv_done(i), 1);
                mbar_init(p_half(i), 128); mbar_init(s_free(i), 128);
            }
            mbar_init(drained, 1);
            set_gave_up(bar0, 0);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        find_tile(P, false, t, gridDim.x / P.H, 256, P.causal, work);
    }
    if (warp == 1) tmem_alloc<512>(smem_u32(slot));
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *slot;
    const Work w = *work;
    T* out = static_cast<T*>(P.o);

    // key blocks of the two tiles
    const int off = w.lk - w.lq;
    int n[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r0 = w.tile * 256 + i * 128;
        const int last = min(r0 + 127, w.lq - 1);
        const int keys = w.tile < 0 || r0 >= w.lq ? 0 : P.causal ? min(w.lk, last + off + 1) : w.lk;
        n[i] = keys > 0 ? (keys + 127) / 128 : 0;
    }
    const int nmax = max(n[0], n[1]);
    const uint32_t ring = base + C::RING;

    if (w.tile < 0) {
        const int rows = w.first + (P.Tq - w.last);
        if (rows > 0) {
            zero_uncovered(out, w, P.Tq, P.H, head, P.D);
            for (int64_t r = (int64_t)w.spare * blockDim.x + threadIdx.x; r < rows; r += (int64_t)w.spares * blockDim.x)
                P.lse[(int64_t)head * P.Tq + (r < w.first ? r : w.last + (r - w.first))] = 0.f;
        }
    } else if (warp == 0) {
        // ---- loads ----
        if (lane == 0 && nmax > 0) {
            auto load = [&](uint32_t dst, const CUtensorMap* m, uint32_t bar, int h, int row) {
                mbar_expect(bar, TILE);
                for (int b = 0; b < DP / 64; ++b) tma_load(dst + b * BOX, m, bar, b * 64, h, row);
            };
            auto load_q = [&](int i) {
                if (n[i] > 0) load(base + i * TILE, &mq, q_full(i), head, w.q0 + w.tile * 256 + i * 128);
            };
            load_q(0);
            int s = 0, sent = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (; sent < 2 * nmax; ++sent) {         // K_0, V_0, K_1, V_1, ...
                if (!(ok = mbar_wait(empty(s), ph ^ 1, P.err, 1))) break;
                load(ring + s * TILE, sent & 1 ? &mv : &mk, full(s), kvh, w.k0 + (sent >> 1) * 128);
                if (sent == 0) load_q(1);
                if (++s == ST) { s = 0; ph ^= 1; }
            }
            // the last use of every slot: nothing arrives on these barriers after the block has left
            for (int x = 0; ok && x < ST && x < 2 * nmax; ++x) {
                const int y = 2 * nmax - 1 - x;
                ok = mbar_wait(empty(y % ST), (y / ST) & 1, P.err, 2);
            }
            if (!ok) {
                if ((n[0] == 0 || ring_landed(q_full(0), 1, 1, P.err)) &&
                    (n[1] == 0 || sent == 0 || ring_landed(q_full(1), 1, 1, P.err)))
                    ring_landed(full(0), ST, sent, P.err);
                goto done;
            }
        }
    } else if (warp == 1) {
        // ---- products (the whole warp, one value of everything) ----
        constexpr uint32_t ID_S = instr_desc(BF, 128, 0), ID_O = instr_desc(BF, DP, 1);
        const uint32_t one = elect_one(), tm = uniform(tmem), sm = uniform(base);
        const int nu[2] = {uniform(n[0]), uniform(n[1])}, nm = max(nu[0], nu[1]), lk = uniform(w.lk);
        const uint64_t dq = desc_k(sm), dk = desc_k(sm + C::RING), dv = desc_mn(sm + C::RING);
        auto mma_s = [&](int i, int s) {
            const uint64_t a = dq + i * (TILE >> 4), b = dk + s * (TILE >> 4);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) mma_ss(tm + i * 128, a + step_k(kk), b + step_k(kk), ID_S, kk != 0, one);
            mma_commit(s_full(i), one);
        };
        if (nm > 0) {
            if (!warp_wait(full(0), 0, P.err, 3)) goto done;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (nu[i] == 0) continue;
                if (!warp_wait(q_full(i), 0, P.err, 4)) goto done;
                fence_after();
                mma_s(i, 0);
            }
            mma_commit(empty(0), one);
        }
        int sv = 1, sk = 2;
        uint32_t pv = 0, pk = 0;                  // phases of their barriers
        for (int j = 0; j < nm; ++j) {
            const bool more = j + 1 < nm;
            if (!warp_wait(full(sv), pv, P.err, 5)) goto done;
            if (lk - j * 128 < 128) zero_rows<DP>(smem + C::RING + sv * TILE, lk - j * 128);
            if (more && !warp_wait(full(sk), pk, P.err, 6)) goto done;
            const uint64_t b = dv + sv * (TILE >> 4);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (j >= nu[i]) continue;
                if (APART && j + 1 < nu[i]) {
                    if (!warp_wait(s_free(i), j & 1, P.err, 11)) goto done;
                    fence_after();
                    mma_s(i, sk);
                }
                const uint32_t p = APART ? tm + 384 + i * 64 : tm + i * 128;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!warp_wait(h ? p_full(i) : p_half(i), j & 1, P.err, 7)) goto done;
                    fence_after();
#pragma unroll
                    for (int kk = h * 4; kk < h * 4 + 4; ++kk)
                        mma_ts(tm + 256 + i * DP, p + kk * 8, b + step_mn(kk), ID_O, (j | kk) != 0, one);
                }
                mma_commit(pv_done(i), one);
                if (!APART && j + 1 < nu[i]) {    // S_i takes P_i's place: only after the product that reads P_i
                    if (!warp_wait(pv_done(i), j & 1, P.err, 8)) goto done;
                    fence_after();
                    mma_s(i, sk);
                }
            }
            mma_commit(empty(sv), one);
            if (more) mma_commit(empty(sk), one);
            sv += 2; if (sv >= ST) { sv -= ST; pv ^= 1; }
            sk += 2; if (sk >= ST) { sk -= ST; pk ^= 1; }
        }
    } else if (warp >= 4) {
        // ---- softmax: one row a thread ----
        const int i = (warp - 4) >> 2, q = warp & 3;
        const int ni = i ? n[1] : n[0];
        const int row = w.tile * 256 + i * 128 + q * 32 + lane;      // in the sequence
        const bool live = row < w.lq;
        const uint32_t ts = tmem + ((uint32_t)(q * 32) << 16) + i * 128;
        const uint32_t to = tmem + ((uint32_t)(q * 32) << 16) + 256 + i * DP;
        const uint32_t tp = APART ? tmem + ((uint32_t)(q * 32) << 16) + 384 + i * 64 : ts;
        const float c = P.scale2, slack = 8.0f / c;
        // keys this row sees; and those every row of the tile sees
        const int mine = P.causal ? min(w.lk, row + off + 1) : w.lk;
        const int every = P.causal ? min(w.lk, w.tile * 256 + i * 128 + off + 1) : w.lk;
        float m = -INFINITY, l = 0.f;
        for (int j = 0; j < ni; ++j) {
            mbar_wait(s_full(i), j & 1, P.err, 9);
            fence_after();
            // 32 scores at a time: the second half first, for the maximum alone;
            // the first half stays in registers for the exponentials
            const bool masked = (j + 1) * 128 > every;
            uint32_t x[32], y[32];
            auto load = [&](int at) {
                ld32(ts + at, x);
                ld32(ts + at + 32, y);
                wait_ld();
                if (masked) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        if (j * 128 + at + k >= mine) x[k] = 0xff800000u;          // -inf
                        if (j * 128 + at + 32 + k >= mine) y[k] = 0xff800000u;
                    }
                }
            };
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            auto largest = [&]() {
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    tops[0] = max3_nan(tops[0], __uint_as_float(x[k]), __uint_as_float(x[k + 1]));
                    tops[1] = max3_nan(tops[1], __uint_as_float(x[k + 2]), __uint_as_float(x[k + 3]));
                    tops[2] = max3_nan(tops[2], __uint_as_float(y[k]), __uint_as_float(y[k + 1]));
                    tops[3] = max3_nan(tops[3], __uint_as_float(y[k + 2]), __uint_as_float(y[k + 3]));
                }
            };
            load(64);
            largest();
            load(0);
            largest();
            const float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]);
            // the reference maximum follows only where it has fallen 2^8 behind:
            // p up to 256 is as exact, and O is rescaled a few times in all
            // (a NaN score, or one of +inf, makes the row NaN here: the exponentials
            // on the fma pipe would hide it)
            if (APART && j > 0) mbar_wait(pv_done(i), (j - 1) & 1, P.err, 12);     // O and P are free
            const bool up = !(top <= m + slack);
            if (__any_sync(0xffffffffu, up)) {
                float to_m = up ? max3_nan(m, top, top) : m;     // a row moves by its own scores alone
                if (to_m == INFINITY) to_m = NAN;
                const float f = m == to_m ? 1.0f : ex2f((m - to_m) * c);
                m = to_m;
                l *= f;
                if (j > 0) {            // P_i V of block j - 1 is complete
#pragma unroll
                    for (int k = 0; k < DP; k += 32) {
                        uint32_t o[32];
                        ld32(to + k, o);
                        wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        st32(to + k, o);
                    }
                }
            }
            const float mc = m == -INFINITY ? 0.f : -m * c;
            const uint64_t c2 = f2(c, c), mc2 = f2(mc, mc);
            uint64_t sum[2] = {0, 0};
            auto weigh = [&](const uint32_t* v, int at, auto fma_pipe) {       // P of 32 columns
                uint32_t w16[16];
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    float a, b;
                    const uint64_t x2 = fma2(f2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), c2, mc2);
                    // every fourth pair on the fma pipe (where nothing is masked: it has no exact 0)
                    if (decltype(fma_pipe)::value && k % 8 == 6) ex2_fma2(x2, a, b);
                    else {
                        unf2(x2, a, b);
                        a = ex2f(a);
                        b = ex2f(b);
                    }
                    sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], f2(a, b));
                    w16[k >> 1] = pack2(a, b, T());
                }
                st16(tp + at, w16);
            };
            auto block = [&](auto fma_pipe) {
                weigh(x, 0, fma_pipe);
                weigh(y, 16, fma_pipe);
                wait_st();
                fence_before();
                mbar_arrive(p_half(i));
                load(64);
                if (APART) {
                    fence_before();
                    mbar_arrive(s_free(i));
                }
                weigh(x, 32, fma_pipe);
                weigh(y, 48, fma_pipe);
            };
            if (masked) block(std::false_type());
            else block(std::true_type());
            float sa, sb;
            unf2(add2(sum[0], sum[1]), sa, sb);
            l += sa + sb;
            wait_st();
            fence_before();
            mbar_arrive(p_full(i));
        }
        const int64_t trow = (int64_t)w.q0 + row;
        const int64_t at = (trow * P.H + head) * P.D;
        T* rest = static_cast<T*>(P.rest);
        if (ni > 0) {
            mbar_wait(pv_done(i), (ni - 1) & 1, P.err, 10);
            fence_after();
            const int64_t stride = (int64_t)P.H * P.D, at0 = at - lane * stride;
            store_rows<T, DP, true>(to, base + i * TILE + q * (TILE / 4), m == -INFINITY ? 0.f : 1.0f / l, out + at0, stride,
                                    0, P.D, w.lq - (row - lane), rest ? rest + at0 : nullptr);
        } else if (live) {
            for (int d = 0; d < P.D; d += 8) {
                *reinterpret_cast<uint4*>(out + at + d) = make_uint4(0, 0, 0, 0);
                if (rest) *reinterpret_cast<uint4*>(rest + at + d) = make_uint4(0, 0, 0, 0);
            }
        }
        if (live) P.lse[(int64_t)head * P.Tq + trow] = m == -INFINITY ? -INFINITY : fmaf(m, P.scale, logf(l));
    }
done:
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        if (gave_up(bar0)) spoil_block<0, C::BARS, NBARS>(P);
        tmem_free<512>(tmem);
    }
}

// ---------------------------------------------------------------- the range of fp16
// ds = p (dp - delta) is far smaller than its sums where keys are many or
// gradients small: 4096 keys and upstream gradients of 1e-5 give 2e-9, and fp16
// ends at 6e-8.  So in fp16 p is held times 2^12 in dk / dv (exponents + 12),
// and ds times a power of two that cannot take it past 2^12 (16 times below the
// largest number): |dp| and |delta| are at most max|v| times the row's sum of
// |do|.  The factor goes by the row in dq, by the sequence and the key head's
// query heads in dk, so no other sequence has a part in it; it is never below 1,
// and the results are divided by it in fp32.  bf16 has fp32's range.
constexpr float P_LIFT = 4096.f, P_LIFT_LOG2 = 12.f;
__device__ __forceinline__ float lift(float l1, float vmax) {
    const float bound = 2.f * l1 * vmax;
    if (!(bound > 0.f && bound < 2048.f)) return 1.f;        // (NaN, infinities and zeros too)
    return __uint_as_float((uint32_t)(127 + 11 + 127) * (1u << 23) - (__float_as_uint(bound) & 0x7f800000u));
}
__device__ __forceinline__ float largest_v(const Params& P, int seq, int kvh) {       // (whole warp)
    const float* at = P.vmax + ((int64_t)seq * (P.H / P.G) + kvh) * P.chunks;
    const int lane = threadIdx.x & 31;
    return warp_maxf(lane < P.chunks ? at[lane] : 0.f);
}

// vmax, and zeros to dmax: a block takes a chunk of a sequence's keys of one
// head, 16 or 32 rows a step, eight 16-byte loads of a thread on their way.
// Reads v once more: 15 us beside 520 (8 x 2048 tokens, 16 heads of 128), 7
// beside 780 (8191 tokens, 4 key heads).
__global__ void __launch_bounds__(256) range_kernel(const __grid_constant__ Params P) {
    __shared__ float red[8];
    const int HK = P.H / P.G, c = blockIdx.x % P.chunks, kvh = blockIdx.x / P.chunks % HK, b = blockIdx.x / P.chunks / HK;
    if (c == 0)
        for (int i = threadIdx.x; i < P.G; i += 256) P.dmax[b * P.H + kvh * P.G + i] = 0;
    const int k0 = min(max(P.cuk[b], 0), P.Tk), lk = max(min(max(P.cuk[b + 1], 0), P.Tk) - k0, 0);
    const int rows = (lk + P.chunks - 1) / P.chunks, first = min((int64_t)c * rows, (int64_t)lk), left = min(rows, lk - first);
    const int wide = P.D > 64, step = wide ? 16 : 32, row = threadIdx.x >> (wide ? 4 : 3),
              col = (threadIdx.x & (wide ? 15 : 7)) * 8;
    const __half* v = static_cast<const __half*>(P.v) + ((int64_t)k0 + first + row) * P.v_ts + kvh * P.v_hs + col;
    float m = 0.f;
    if (col < P.D) {
        for (int r = row; r < left; r += 8 * step, v += 8 * step * P.v_ts) {
            uint4 u[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                u[k] = r + k * step < left ? *reinterpret_cast<const uint4*>(v + k * step * P.v_ts) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                float x[8];
                Pack16<__half>::unpack(u[k], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
            }
        }
    }
    m = warp_maxf(m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
        P.vmax[blockIdx.x] = m;
    }
}

// ---------------------------------------------------------------- backward: dq and delta
// A block owns 128 query rows of one head.  Tensor memory: S 0, dP 128, dQ
// 256, dS (16-bit pairs) 384.  S and dP of the next key block are computed as
// soon as the softmax warps have read the present ones.
// Bound by the softmax warps (1970 cycles a block, 1024 of exponentials) beside
// 1536 cycles of products.  8 x 2048, 16 heads of 128, causal: 225 us, 917
// TFLOP/s of its three products.
template <int DP> struct BwdQ {
    static constexpr int TILE = 256 * DP;
    static constexpr int KS = DP == 128 ? 3 : 4, VS = DP == 128 ? 2 : 4;
    static constexpr int K_OFF = 2 * TILE, V_OFF = K_OFF + KS * TILE;
    static constexpr int BARS = V_OFF + VS * TILE;
    static constexpr int RED = BARS + BARRIERS;                     // delta, and (fp16) the sum of |do|, of 128 rows
    static constexpr size_t SMEM = RED + 1024 + 1024;
};

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1)
    bwd_q_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                 const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo,
                 const __grid_constant__ Params P) {
    using C = BwdQ<DP>;
    constexpr int TILE = C::TILE, KS = C::KS, VS = C::VS;
    constexpr int BF = !__is_same(T, __half);
    extern __shared__ uint8_t raw[];
    uint8_t* smem = align1024(raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BARS);
    constexpr int NBARS = 2 * KS + 2 * VS + 8;
    uint32_t* slot = slot_of(bars, NBARS);
    Work* work = work_of(bars, NBARS);
    float* red = reinterpret_cast<float*>(smem + C::RED);
    const uint32_t base = smem_u32(smem), bar0 = smem_u32(bars);
    auto k_full = [&](int s) { return bar0 + 8u * s; };
    auto k_empty = [&](int s) { return bar0 + 8u * (KS + s); };
    auto v_full = [&](int s) { return bar0 + 8u * (2 * KS + s); };
    auto v_empty = [&](int s) { return bar0 + 8u * (2 * KS + VS + s); };
    const uint32_t one = bar0 + 8u * (2 * KS + 2 * VS);
    const uint32_t q_full = one, s_full = one + 8, s_free = one + 16, dp_full = one + 24, dp_free = one + 32,
                   ds_full = one + 40, ds_free = one + 48, drained = one + 56;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.x % P.H, t = blockIdx.x / P.H, kvh = head / P.G;

    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < KS; ++s) { mbar_init(k_full(s), 1); mbar_init(k_empty(s), 1); }
            for (int s = 0; s < VS; ++s) { mbar_init(v_full(s), 1); mbar_init(v_empty(s), 1); }
            mbar_init(q_full, 1);
            mbar_init(s_full, 1); mbar_init(s_free, 256);
            mbar_init(dp_full, 1); mbar_init(dp_free, 256);
            mbar_init(ds_full, 256); mbar_init(ds_free, 1);
            mbar_init(drained, 1);
            set_gave_up(bar0, 0);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        find_tile(P, false, t, gridDim.x / P.H, 128, P.causal, work);
    }
    if (warp == 1) tmem_alloc<512>(smem_u32(slot));
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *slot;
    const Work w = *work;
    const int off = w.lk - w.lq, r0 = w.tile * 128;
    int n = 0;
    if (w.tile >= 0) {
        const int last = min(r0 + 127, w.lq - 1);
        const int keys = P.causal ? min(w.lk, last + off + 1) : w.lk;
        n = keys > 0 ? (keys + 127) / 128 : 0;
    }

    if (w.tile < 0) {
        zero_uncovered(P.dq, w, P.Tq, P.H, head, P.D);
    } else if (warp == 0) {
        if (lane == 0 && n > 0) {
            auto load = [&](uint32_t dst, const CUtensorMap* m, uint32_t bar, int h, int row) {
                for (int b = 0; b < DP / 64; ++b) tma_load(dst + b * BOX, m, bar, b * 64, h, row);
            };
            mbar_expect(q_full, 2 * TILE);
            load(base, &mq, q_full, head, w.q0 + r0);
            load(base + TILE, &mdo, q_full, head, w.q0 + r0);
            int nk = 0, nv = 0;                          // tiles sent
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                const int sk = j % KS, sv = j % VS;
                if (!(ok = mbar_wait(k_empty(sk), ((j / KS) & 1) ^ 1, P.err, 21))) break;
                mbar_expect(k_full(sk), TILE);
                load(base + C::K_OFF + sk * TILE, &mk, k_full(sk), kvh, w.k0 + j * 128);
                ++nk;
                if (!(ok = mbar_wait(v_empty(sv), ((j / VS) & 1) ^ 1, P.err, 22))) break;
                mbar_expect(v_full(sv), TILE);
                load(base + C::V_OFF + sv * TILE, &mv, v_full(sv), kvh, w.k0 + j * 128);
                ++nv;
            }
            for (int x = 0; ok && x < KS && x < n; ++x)
                ok = mbar_wait(k_empty((n - 1 - x) % KS), ((n - 1 - x) / KS) & 1, P.err, 23);
            for (int x = 0; ok && x < VS && x < n; ++x)
                ok = mbar_wait(v_empty((n - 1 - x) % VS), ((n - 1 - x) / VS) & 1, P.err, 24);
            if (!ok) {
                if (ring_landed(q_full, 1, 1, P.err) && ring_landed(k_full(0), KS, nk, P.err))
                    ring_landed(v_full(0), VS, nv, P.err);
                goto done;
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t ID_S = instr_desc(BF, 128, 0), ID_Q = instr_desc(BF, DP, 1);
        const uint32_t el = elect_one(), tm = uniform(tmem), sm = uniform(base);
        const int nu = uniform(n), lk = uniform(w.lk);
        const uint64_t dq = desc_k(sm), ddo = desc_k(sm + TILE), dk = desc_k(sm + C::K_OFF), dv = desc_k(sm + C::V_OFF),
                       dkt = desc_mn(sm + C::K_OFF);
        auto dq_product = [&](int j, int s) {        // dQ += dS_j K_j
            const uint64_t b = dkt + s * (TILE >> 4);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
                mma_ts(tm + 256, tm + 384 + kk * 8, b + step_mn(kk), ID_Q, (j | kk) != 0, el);
            mma_commit(k_empty(s), el);
            mma_commit(ds_free, el);
        };
        if (nu > 0 && !warp_wait(q_full, 0, P.err, 25)) goto done;
        int sk = 0, sv = 0, before = 0;              // slots; that of the block before
        uint32_t pk = 0, pv = 0;
        for (int j = 0; j < nu; ++j) {
            if (!warp_wait(k_full(sk), pk, P.err, 26)) goto done;
            // rows of another sequence: dS is 0 there, and 0 * NaN must not reach dQ
            if (lk - j * 128 < 128) zero_rows<DP>(smem + C::K_OFF + sk * TILE, lk - j * 128);
            if (j > 0 && !warp_wait(s_free, (j - 1) & 1, P.err, 27)) goto done;
            fence_after();
            {
                const uint64_t b = dk + sk * (TILE >> 4);
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) mma_ss(tm, dq + step_k(kk), b + step_k(kk), ID_S, kk != 0, el);
                mma_commit(s_full, el);
            }
            if (!warp_wait(v_full(sv), pv, P.err, 28)) goto done;
            if (j > 0 && !warp_wait(dp_free, (j - 1) & 1, P.err, 29)) goto done;
            fence_after();
            {
                const uint64_t b = dv + sv * (TILE >> 4);
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    mma_ss(tm + 128, ddo + step_k(kk), b + step_k(kk), ID_S, kk != 0, el);
                mma_commit(dp_full, el);
                mma_commit(v_empty(sv), el);
            }
            if (j > 0) {
                if (!warp_wait(ds_full, (j - 1) & 1, P.err, 30)) goto done;
                fence_after();
                dq_product(j - 1, before);
            }
            before = sk;
            if (++sk == KS) { sk = 0; pk ^= 1; }
            if (++sv == VS) { sv = 0; pv ^= 1; }
        }
        if (nu > 0) {
            if (!warp_wait(ds_full, (nu - 1) & 1, P.err, 31)) goto done;
            fence_after();
            dq_product(nu - 1, before);
        }
    } else if (warp >= 4) {
        const int half = (warp - 4) >> 2, q = warp & 3, r = q * 32 + lane;
        const int row = r0 + r;
        const bool live = row < w.lq;
        const int64_t trow = (int64_t)w.q0 + row;
        // delta = do . o, o with its rest: o rounded to 16 bits alone makes the
        // error of dq and dk a tenth larger.  A row's 16-byte pieces go to
        // neighbouring lanes (a lane a row would touch 32 lines a load), each
        // warp takes 16 rows.
        {
            constexpr int CH = DP / 8, AT = 32 / CH, NL = 16 / AT;      // lanes of a row, rows a load, loads
            const int sub = lane / CH, c = lane % CH * 8;
            uint4 g[NL], o[NL], e[NL];                                  // all on their way at once
            const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < NL; ++k) {
                const int x = r0 + (warp - 4) * 16 + k * AT + sub;
                g[k] = o[k] = e[k] = none;
                if (x < w.lq && c < P.D) {
                    const int64_t tok = (int64_t)w.q0 + x, at = (tok * P.H + head) * P.D + c;
                    g[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(P.dout) + tok * P.do_ts +
                                                                head * P.do_hs + c));
                    o[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(P.o) + at));
                    e[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(P.rest) + at));
                }
            }
#pragma unroll
            for (int k = 0; k < NL; ++k) {
                float gv[8], ov[8], ev[8], d = 0.f, a = 0.f;
                Pack16<T>::unpack(g[k], gv);
                Pack16<T>::unpack(o[k], ov);
                Pack16<T>::unpack(e[k], ev);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    d = fmaf(gv[i], ov[i] + ev[i], d);
                    if (!BF) a += fabsf(gv[i]);
                }
#pragma unroll
                for (int i = CH / 2; i > 0; i >>= 1) {
                    d += __shfl_xor_sync(0xffffffffu, d, i);
                    if (!BF) a += __shfl_xor_sync(0xffffffffu, a, i);
                }
                if (lane % CH == 0) {
                    red[(warp - 4) * 16 + k * AT + sub] = d;
                    if (!BF) red[128 + (warp - 4) * 16 + k * AT + sub] = a;
                }
            }
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float d = red[r];
        if (live && half == 0) P.delta[(int64_t)head * P.Tq + trow] = d;
        float lse = live ? P.lse[(int64_t)head * P.Tq + trow] : 0.f;
        if (lse == -INFINITY) lse = 0.f;           // no key: everything is masked below
        float up = 1.f;                            // fp16: ds is held times this
        if (!BF) {
            const float a = red[128 + r];
            up = lift(a, largest_v(P, w.seq, kvh));
            const float most = warp_maxf(live ? a : 0.f);
            if (half == 0 && lane == 0) atomicMax(P.dmax + w.seq * P.H + head, __float_as_int(most));
        }
        const float l2 = -lse * LOG2E;
        const uint64_t c2 = f2(P.scale2, P.scale2), l22 = f2(l2, l2), nd2 = f2(-d * up, -d * up), up2 = f2(up, up);
        const int mine = (P.causal ? min(w.lk, row + off + 1) : w.lk) - half * 64;
        const int every = P.causal ? min(w.lk, r0 + off + 1) : w.lk;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        for (int j = 0; j < n; ++j) {
            // S and dP are read whole, which frees their places for the next
            // block's products, and then meet element by element: exponentials
            // and the arithmetic of ds overlap
            uint32_t u[64], v[64];
            mbar_wait(s_full, j & 1, P.err, 32);
            fence_after();
            ld32(tmem + lanes + half * 64, u);
            ld32(tmem + lanes + half * 64 + 32, u + 32);
            wait_ld();
            fence_before();
            mbar_arrive(s_free);
            mbar_wait(dp_full, j & 1, P.err, 33);
            fence_after();
            ld32(tmem + lanes + 128 + half * 64, v);
            ld32(tmem + lanes + 128 + half * 64 + 32, v + 32);
            wait_ld();
            fence_before();
            mbar_arrive(dp_free);
            const bool masked = (j + 1) * 128 > every;
            auto weigh = [&](auto with_mask) {
                constexpr bool mask = decltype(with_mask)::value;
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    float a, b;
                    unf2(fma2(f2(__uint_as_float(u[k]), __uint_as_float(u[k + 1])), c2, l22), a, b);
                    a = ex2f(a);
                    b = ex2f(b);
                    const uint64_t dp = f2(__uint_as_float(v[k]), __uint_as_float(v[k + 1]));
                    unf2(mul2(f2(a, b), BF ? add2(dp, nd2) : fma2(dp, up2, nd2)), a, b);
                    if (mask && j * 128 + k >= mine) a = 0.f;
                    if (mask && j * 128 + k + 1 >= mine) b = 0.f;
                    u[k >> 1] = pack2(a, b, T());
                }
            };
            if (masked) weigh(std::true_type());
            else weigh(std::false_type());
            if (j > 0) mbar_wait(ds_free, (j - 1) & 1, P.err, 34);
            st32(tmem + lanes + 384 + half * 32, u);
            wait_st();
            fence_before();
            mbar_arrive(ds_full);
        }
        T* dst = static_cast<T*>(P.dq) + (trow * P.H + head) * P.D;
        if (n > 0) {
            mbar_wait(ds_free, (n - 1) & 1, P.err, 35);
            fence_after();
            const int64_t stride = (int64_t)P.H * P.D;
            store_rows<T, DP / 2>(tmem + lanes + 256 + half * (DP / 2), base + half * TILE + q * (TILE / 8), P.scale / up,
                                  dst - lane * stride, stride, half * (DP / 2), P.D, w.lq - (row - lane));
        } else if (live) {
            for (int x = half * 8; x < P.D; x += 16) *reinterpret_cast<uint4*>(dst + x) = make_uint4(0, 0, 0, 0);
        }
    }
done:
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        if (gave_up(bar0)) spoil_block<1, C::BARS, NBARS>(P);
        tmem_free<512>(tmem);
    }
}

// ---------------------------------------------------------------- backward: dk and dv
// A block owns 128 keys of one key head and walks the query blocks of every
// head that shares it, or, where there are few key blocks, of some of these
// heads: the parts' sums then meet in fp32 and are added in part order.  The scores are transposed (a key is a row), so p and
// ds are the A operands of their products as they come from the softmax.
// Tensor memory: S 0, dP 128, dV 256, dK 256 + DP.  P takes half of each half
// of S (columns 0-31 and 64-95), dS the same of dP: each softmax warp writes
// only where it has read itself.  lse and delta belong to columns here: read
// per column from shared memory they met the products there (2730 cycles of
// softmax a block in place of the 1100 of its exponentials), so the products
// subtract them themselves: one more step of 16, a row of ones against the
// value in three 16-bit parts (24 bits of it).  The order of the products, dV, next S, dK,
// next dP, lets the exponentials run beside dK and dP, and ds beside dV and S.
// Bound by the chain P -> dV -> next S -> exponentials (about 2900 cycles a
// block) and by shared memory, which S and dP read at its full rate: 2048 cycles
// of products.  8 x 2048, 16 heads of 128, causal: 281 us, 979 TFLOP/s of its
// four products.
template <int DP> struct BwdK {
    static constexpr int TILE = 256 * DP;
    static constexpr int QS = DP == 128 ? 2 : 3, OS = DP == 128 ? 2 : 3;
    static constexpr int Q_OFF = 2 * TILE, O_OFF = Q_OFF + QS * TILE;
    static constexpr int BARS = O_OFF + OS * TILE;
    static constexpr int ONES = BARS + BARRIERS;                    // the row of ones, for every key
    static constexpr int STAT = ONES + THIN;                   // 2 stages of (-lse / scale, -delta), a query a row
    static constexpr size_t SMEM = STAT + 4 * THIN + 1024;
};

// A value's parts against the ones: three of 8 bits each, in bf16 for fp16
// operands too (an instruction's operands have one type, but the step of 16 that
// holds these is an instruction of its own): lse / scale is a score before
// scaling, which fp16 does not hold.  NaN comes through, an infinity as NaN.
__device__ __forceinline__ uint4 parts_ones() { return make_uint4(0x3f803f80u, 0x3f80u, 0, 0); }
__device__ __forceinline__ uint4 parts_of(float v) {
    const float a = __bfloat162float(__float2bfloat16_rn(v)), b = __bfloat162float(__float2bfloat16_rn(v - a));
    return make_uint4(pack2(a, b, __nv_bfloat16()), pack2(v - a - b, 0.f, __nv_bfloat16()), 0, 0);
}

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1)
    bwd_k_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                 const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo,
                 const __grid_constant__ Params P) {
    using C = BwdK<DP>;
    constexpr int TILE = C::TILE, QS = C::QS, OS = C::OS;
    constexpr int BF = !__is_same(T, __half);
    extern __shared__ uint8_t raw[];
    uint8_t* smem = align1024(raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BARS);
    constexpr int NBARS = 2 * QS + 2 * OS + 12;
    uint32_t* slot = slot_of(bars, NBARS);
    Work* work = work_of(bars, NBARS);
    const uint32_t base = smem_u32(smem), bar0 = smem_u32(bars);
    auto q_full = [&](int s) { return bar0 + 8u * s; };
    auto q_empty = [&](int s) { return bar0 + 8u * (QS + s); };
    auto o_full = [&](int s) { return bar0 + 8u * (2 * QS + s); };
    auto o_empty = [&](int s) { return bar0 + 8u * (2 * QS + OS + s); };
    const uint32_t one = bar0 + 8u * (2 * QS + 2 * OS);
    const uint32_t kv_full = one, s_full = one + 8, p_full = one + 16, dv_done = one + 24, dp_full = one + 32,
                   ds_full = one + 40, dk_done = one + 48;
    auto st_full = [&](int s) { return one + 56u + 8u * s; };
    auto st_empty = [&](int s) { return one + 72u + 8u * s; };
    const uint32_t drained = one + 88;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int HK = P.H / P.G;
    const int kvh = blockIdx.x % HK, part = blockIdx.x / HK % P.splits, t = blockIdx.x / HK / P.splits;
    const int head0 = kvh * P.G + part * P.per;                      // its first query head

    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < QS; ++s) { mbar_init(q_full(s), 1); mbar_init(q_empty(s), 1); }
            for (int s = 0; s < OS; ++s) { mbar_init(o_full(s), 1); mbar_init(o_empty(s), 1); }
            mbar_init(kv_full, 1);
            mbar_init(s_full, 1); mbar_init(p_full, 256); mbar_init(dv_done, 1);
            mbar_init(dp_full, 1); mbar_init(ds_full, 256); mbar_init(dk_done, 1);
            for (int s = 0; s < 2; ++s) { mbar_init(st_full(s), 64); mbar_init(st_empty(s), 1); }
            mbar_init(drained, 1);
            set_gave_up(bar0, 0);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        find_tile(P, true, t, gridDim.x / HK / P.splits, 128, false, work);
    }
    if (warp == 1) tmem_alloc<512>(smem_u32(slot));
    if (warp >= 4) {          // the ones, and zeros beside them and beside the values
        const uint4 z = make_uint4(0, 0, 0, 0);
        for (int i = threadIdx.x - 128; i < 5 * 256; i += 256) {
            const uint32_t at = base + C::ONES + (i >> 8) * THIN + (i & 255) * 16;
            sts16(at, (i < 256 && !(i & 8)) ? parts_ones() : z);
        }
        fence_async();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *slot;
    const Work w = *work;
    const int off = w.lk - w.lq, k0 = w.tile * 128;
    // query blocks [jq, jq + nq) of every head; `n` in all
    int jq = 0, nq = 0;
    if (w.tile >= 0) {
        const int first = P.causal ? max(0, k0 - off) : 0;
        if (first < w.lq) { jq = first / 128; nq = (w.lq + 127) / 128 - jq; }
    }
    const int heads = min(P.per, P.G - part * P.per), n = nq * heads;
    const int64_t all = (int64_t)P.Tk * HK * P.D;
    float* dkp = P.part + 2 * all * part;                            // splits > 1

    if (w.tile < 0) {
        // (an fp32 row is two 16-bit ones)
        const int width = P.splits > 1 ? 2 * P.D : P.D;
        zero_uncovered(P.splits > 1 ? dkp : P.dk, w, P.Tk, HK, kvh, width);
        zero_uncovered(P.splits > 1 ? dkp + all : P.dv, w, P.Tk, HK, kvh, width);
    } else if (warp == 0) {
        if (lane == 0 && n > 0) {
            auto load = [&](uint32_t dst, const CUtensorMap* m, uint32_t bar, int h, int row) {
                for (int b = 0; b < DP / 64; ++b) tma_load(dst + b * BOX, m, bar, b * 64, h, row);
            };
            mbar_expect(kv_full, 2 * TILE);
            load(base, &mk, kv_full, kvh, w.k0 + k0);
            load(base + TILE, &mv, kv_full, kvh, w.k0 + k0);
            int sent_q = 0, sent_o = 0;
            bool ok = true;
            for (int x = 0; x < n; ++x) {
                const int sq = x % QS, so = x % OS;
                const int head = head0 + x / nq, row = w.q0 + (jq + x % nq) * 128;
                if (!(ok = mbar_wait(q_empty(sq), ((x / QS) & 1) ^ 1, P.err, 41))) break;
                mbar_expect(q_full(sq), TILE);
                load(base + C::Q_OFF + sq * TILE, &mq, q_full(sq), head, row);
                ++sent_q;
                if (!(ok = mbar_wait(o_empty(so), ((x / OS) & 1) ^ 1, P.err, 42))) break;
                mbar_expect(o_full(so), TILE);
                load(base + C::O_OFF + so * TILE, &mdo, o_full(so), head, row);
                ++sent_o;
            }
            for (int x = 0; ok && x < QS && x < n; ++x)
                ok = mbar_wait(q_empty((n - 1 - x) % QS), ((n - 1 - x) / QS) & 1, P.err, 43);
            for (int x = 0; ok && x < OS && x < n; ++x)
                ok = mbar_wait(o_empty((n - 1 - x) % OS), ((n - 1 - x) / OS) & 1, P.err, 44);
            if (!ok) {
                if (ring_landed(kv_full, 1, 1, P.err) && ring_landed(q_full(0), QS, sent_q, P.err))
                    ring_landed(o_full(0), OS, sent_o, P.err);
                goto done;
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t ID_S = instr_desc(BF, 128, 0), ID_D = instr_desc(BF, DP, 1), ID_STAT = instr_desc(1, 128, 0);
        const uint32_t el = elect_one(), tm = uniform(tmem), sm = uniform(base);
        const int nu = uniform(n), per = uniform(nq), left = uniform(w.lq - jq * 128);
        const uint64_t dk = desc_k(sm), dv = desc_k(sm + TILE), dq = desc_k(sm + C::Q_OFF), ddo = desc_k(sm + C::O_OFF),
                       dqt = desc_mn(sm + C::Q_OFF), dot = desc_mn(sm + C::O_OFF);
        const uint64_t ones = desc_thin(sm + C::ONES), stat = desc_thin(sm + C::STAT);
        // rows of another sequence hold anything: p and ds are 0 there, and 0 * NaN must not reach dk and dv
        int sq = 0, so = 0, bq = 0, bo = 0;          // slots and query blocks (of their head) of the next S and dP
        uint32_t pq = 0, po = 0, ss = 0, sp = 0, ps = 0;      // ss, sp: slots of lse and delta; ps: their phase
        // the operands of the next S: waited for before its place is free
        auto s_ready = [&]() -> bool {
            if (!warp_wait(q_full(sq), pq, P.err, 45)) return false;
            if (left - bq * 128 < 128) zero_rows<DP>(smem + C::Q_OFF + sq * TILE, left - bq * 128);
            return warp_wait(st_full(ss), ps, P.err, 53);
        };
        auto s_product = [&]() {
            fence_after();
            const uint64_t b = dq + sq * (TILE >> 4);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) mma_ss(tm, dk + step_k(kk), b + step_k(kk), ID_S, kk != 0, el);
            mma_ss(tm, ones, stat + ss * (2 * THIN >> 4), ID_STAT, 1, el);
            mma_commit(s_full, el);
            ss ^= 1;
            if (ss == 0) ps ^= 1;
            if (++bq == per) bq = 0;
            if (++sq == QS) { sq = 0; pq ^= 1; }
        };
        auto dp_ready = [&]() -> bool {
            if (!warp_wait(o_full(so), po, P.err, 46)) return false;
            if (left - bo * 128 < 128) zero_rows<DP>(smem + C::O_OFF + so * TILE, left - bo * 128);
            return true;
        };
        auto dp_product = [&]() {
            fence_after();
            const uint64_t b = ddo + so * (TILE >> 4);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) mma_ss(tm + 128, dv + step_k(kk), b + step_k(kk), ID_S, kk != 0, el);
            mma_ss(tm + 128, ones, stat + (2 * sp + 1) * (THIN >> 4), ID_STAT, 1, el);
            mma_commit(dp_full, el);
            mma_commit(st_empty(sp), el);
            sp ^= 1;
            if (++bo == per) bo = 0;
            if (++so == OS) { so = 0; po ^= 1; }
        };
        if (nu > 0) {
            if (!warp_wait(kv_full, 0, P.err, 47)) goto done;
            if (!s_ready()) goto done;
            s_product();
            if (!dp_ready()) goto done;
            dp_product();
        }
        int cq = 0, co = 0;                          // slots of the present dK and dV
        for (int x = 0; x < nu; ++x) {
            if (!warp_wait(p_full, x & 1, P.err, 48)) goto done;
            fence_after();
            {
                const uint64_t b = dot + co * (TILE >> 4);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                    mma_ts(tm + 256, tm + (kk >> 2) * 64 + (kk & 3) * 8, b + step_mn(kk), ID_D, (x | kk) != 0, el);
                mma_commit(dv_done, el);
                mma_commit(o_empty(co), el);
                if (++co == OS) co = 0;
            }
            if (x + 1 < nu && !s_ready()) goto done;
            if (!warp_wait(dv_done, x & 1, P.err, 49)) goto done;      // S takes P's place
            if (x + 1 < nu) s_product();
            if (!warp_wait(ds_full, x & 1, P.err, 50)) goto done;
            fence_after();
            {
                const uint64_t b = dqt + cq * (TILE >> 4);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                    mma_ts(tm + 256 + DP, tm + 128 + (kk >> 2) * 64 + (kk & 3) * 8, b + step_mn(kk), ID_D, (x | kk) != 0,
                           el);
                mma_commit(dk_done, el);
                mma_commit(q_empty(cq), el);
                if (++cq == QS) cq = 0;
            }
            if (x + 1 < nu) {
                if (!dp_ready()) goto done;
                if (!warp_wait(dk_done, x & 1, P.err, 51)) goto done;  // dP takes dS's place
                dp_product();
            }
        }
    } else if (warp < 4) {
        // ---- lse and delta of the query rows, for the products ----
        const int i = threadIdx.x - 64;
        const float unscale = -1.0f / P.scale;
        for (int x = 0; x < n; ++x) {
            const int s = x & 1, head = head0 + x / nq, row0 = (jq + x % nq) * 128;
            float l[2], d[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int r = row0 + i + k * 64;
                l[k] = -INFINITY;
                d[k] = 0.f;
                if (r < w.lq) {
                    const int64_t at = (int64_t)head * P.Tq + w.q0 + r;
                    l[k] = P.lse[at];
                    d[k] = P.delta[at];
                }
            }
            mbar_wait(st_empty(s), ((x >> 1) & 1) ^ 1, P.err, 52);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t at = base + C::STAT + 2 * s * THIN + thin_row(i + k * 64);
                // no such row, or one without keys: far below every score, so p = 0
                sts16(at, parts_of(l[k] == -INFINITY ? -1e30f : l[k] * unscale));
                sts16(at + THIN, parts_of(-d[k]));
            }
            fence_async();
            mbar_arrive(st_full(s));
        }
        for (int x = 0; x < 2 && x < n; ++x)       // the last use of each stage
            mbar_wait(st_empty((n - 1 - x) & 1), ((n - 1 - x) >> 1) & 1, P.err, 57);
    } else {
        const int half = (warp - 4) >> 2, q = warp & 3;
        const int key = k0 + q * 32 + lane;
        const bool live = key < w.lk;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const uint64_t c2 = f2(P.scale2, P.scale2), lift2 = f2(P_LIFT_LOG2, P_LIFT_LOG2);
        float up = 1.f;                            // fp16: ds is held times this, p times P_LIFT
        if (!BF && n > 0) {
            int most = 0;
            for (int h = 0; h < heads; ++h) most = max(most, P.dmax[w.seq * P.H + head0 + h]);
            up = lift(__int_as_float(most), largest_v(P, w.seq, kvh));
        }
        const uint64_t up2 = f2(up / P_LIFT, up / P_LIFT);
        for (int x = 0; x < n; ++x) {
            const int row0 = (jq + x % nq) * 128 + half * 64;
            // the first query of this half that sees the key, as a column
            const int from = P.causal ? key - off - row0 : 0;
            const bool masked = P.causal && row0 + off < k0 + 127;
            float p[64];
            uint32_t u[64], v[32];
            mbar_wait(s_full, x & 1, P.err, 54);
            fence_after();
            ld32(tmem + lanes + half * 64, u);
            ld32(tmem + lanes + half * 64 + 32, u + 32);
            wait_ld();
#pragma unroll
            for (int k = 0; k < 64; k += 2) {
                float a, b;
                const uint64_t s = f2(__uint_as_float(u[k]), __uint_as_float(u[k + 1]));
                unf2(BF ? mul2(s, c2) : fma2(s, c2, lift2), a, b);
                p[k] = ex2f(a);
                p[k + 1] = ex2f(b);
            }
            if (masked) {
#pragma unroll
                for (int k = 0; k < 64; ++k)
                    if (k < from) p[k] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = pack2(p[2 * k], p[2 * k + 1], T());
            st32(tmem + lanes + half * 64, v);
            wait_st();
            fence_before();
            mbar_arrive(p_full);
            mbar_wait(dp_full, x & 1, P.err, 55);
            fence_after();
            ld32(tmem + lanes + 128 + half * 64, u);
            ld32(tmem + lanes + 128 + half * 64 + 32, u + 32);
            wait_ld();
#pragma unroll
            for (int k = 0; k < 64; k += 2) {
                const uint64_t ds = mul2(f2(p[k], p[k + 1]), f2(__uint_as_float(u[k]), __uint_as_float(u[k + 1])));
                unf2(BF ? ds : mul2(ds, up2), p[k], p[k + 1]);
            }
            if (masked) {
#pragma unroll
                for (int k = 0; k < 64; ++k)
                    if (k < from) p[k] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = pack2(p[2 * k], p[2 * k + 1], T());
            st32(tmem + lanes + 128 + half * 64, v);
            wait_st();
            fence_before();
            mbar_arrive(ds_full);
        }
        const int64_t at = (((int64_t)w.k0 + key - lane) * HK + kvh) * P.D, stride = (int64_t)HK * P.D;   // lane 0's row
        const int col = half * (DP / 2), rows = w.lk - (key - lane);
        auto store = [&](auto* dk, auto* dv) {
            using O = std::remove_pointer_t<decltype(dk)>;
            const uint32_t stage = base + half * TILE + q * (TILE / 16 * sizeof(O));
            store_rows<O, DP / 2>(tmem + lanes + 256 + col, stage, BF ? 1.0f : 1.0f / P_LIFT, dv + at, stride, col, P.D, rows);
            store_rows<O, DP / 2>(tmem + lanes + 256 + DP + col, stage, P.scale / up, dk + at, stride, col, P.D, rows);
        };
        auto clear = [&](auto* dk, auto* dv) {
            constexpr int E = 16 / sizeof(*dk);
            for (int d = half * E; d < P.D; d += 2 * E) {
                *reinterpret_cast<uint4*>(dk + at + lane * stride + d) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(dv + at + lane * stride + d) = make_uint4(0, 0, 0, 0);
            }
        };
        if (n > 0) {
            mbar_wait(dk_done, (n - 1) & 1, P.err, 56);      // and dV before it
            fence_after();
            if (P.splits > 1) store(dkp, dkp + all);
            else store(static_cast<T*>(P.dk), static_cast<T*>(P.dv));
        } else if (live) {
            if (P.splits > 1) clear(dkp, dkp + all);
            else clear(static_cast<T*>(P.dk), static_cast<T*>(P.dv));
        }
    }
done:
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        if (gave_up(bar0)) spoil_block<2, C::BARS, NBARS>(P);
        tmem_free<512>(tmem);
    }
}

// dk, dv from the parts' sums, in part order (8 elements a thread)
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ part, int splits, int64_t all,
                                                   T* __restrict__ dk, T* __restrict__ dv) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= 2 * all) return;
    float s[8], v[8];
    load_vec<8>(part + i, s);
    for (int k = 1; k < splits; ++k) {
        load_vec<8>(part + 2 * all * k + i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += v[e];
    }
    store_vec<8>(i < all ? dk + i : dv + (i - all), s);
}

// ---------------------------------------------------------------- host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// [rows, heads, D] with strides in elements; boxes of 128 rows x 64 columns of one head
bool make_map(CUtensorMap* m, const void* base, int bf16, int64_t rows, int64_t heads, int64_t D, int64_t ts,
              int64_t hs) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
    cuuint64_t strides[2] = {(cuuint64_t)hs * 2, (cuuint64_t)ts * 2};
    cuuint32_t box[3] = {64, 1, 128};
    cuuint32_t step[3] = {1, 1, 1};
    return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
               const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int MAX_DEVICES = 64;
__device__ int g_err;      // first wait that ran out (0: none), per device

int device_index() {
    int d = 0;
    return cudaGetDevice(&d) == cudaSuccess && d >= 0 && d < MAX_DEVICES ? d : -1;
}

// the host's error words, one a device, in memory that the kernels write to
volatile int* host_word() {
    static std::atomic<int*> words;
    static std::mutex mu;
    const int d = device_index();
    if (d < 0) return nullptr;
    int* w = words.load();
    if (!w) {
        std::lock_guard<std::mutex> g(mu);
        w = words.load();
        if (!w) {
            // (an allocation is no work on a stream: it may come first in a capture)
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
            cudaThreadExchangeStreamCaptureMode(&mode);
            void* p = nullptr;
            const cudaError_t e = cudaHostAlloc(&p, MAX_DEVICES * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
            cudaThreadExchangeStreamCaptureMode(&mode);
            if (e != cudaSuccess) {
                cudaGetLastError();
                return nullptr;
            }
            memset(p, 0, MAX_DEVICES * sizeof(int));
            words.store(w = static_cast<int*>(p));
        }
    }
    return w + d;
}

// where this device's kernels tell a wait that ran out; refuses while one is told
int error_words(int** err, int** err_host, const char* name) {
    volatile int* host = host_word();
    void* p = nullptr;
    if (!host || cudaGetSymbolAddress(&p, g_err) != cudaSuccess) return fail(CONCORD_ELAUNCH, std::string(name) + ": device set-up failed");
    if (*host)
        return fail(CONCORD_ETIMEOUT, std::string(name) + ": a wait inside an earlier attention kernel ran out (code " +
                                          std::to_string(*host) + "), its results hold NaN; concord_attention_error(1) clears this");
    *err = static_cast<int*>(p);
    if (cudaHostGetDevicePointer(&p, const_cast<int*>(host), 0) != cudaSuccess)
        return fail(CONCORD_ELAUNCH, std::string(name) + ": device set-up failed");
    *err_host = static_cast<int*>(p);
    return CONCORD_OK;
}

// a wait on a barrier that nobody arrives on, by a warp and by a thread of another
__global__ void __launch_bounds__(64) wait_check_kernel(int* err, int* err_host) {
    __shared__ __align__(BARRIERS) uint8_t bars[BARRIERS];
    const uint32_t b = smem_u32(bars);
    if (threadIdx.x == 0) {
        mbar_init(b, 1);
        set_gave_up(b, 0);
    }
    __syncthreads();
    if (threadIdx.x < 32) warp_wait(b, 0, err, 99);
    else if (threadIdx.x == 32) mbar_wait(b, 0, err, 99);
    __syncthreads();
    if (gave_up(b) && threadIdx.x == 0) {
        *reinterpret_cast<volatile int*>(err_host) = *reinterpret_cast<volatile int*>(err);
        __threadfence_system();
    }
}

template <typename T, int DP> bool raise_smem() {
    return cudaFuncSetAttribute(fwd_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)Fwd<DP>::SMEM) == cudaSuccess &&
           cudaFuncSetAttribute(bwd_q_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)BwdQ<DP>::SMEM) == cudaSuccess &&
           cudaFuncSetAttribute(bwd_k_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)BwdK<DP>::SMEM) == cudaSuccess;
}

// the kernels' shared-memory limits, once per device
bool device_ready() {
    static std::atomic<int> ready[MAX_DEVICES];
    static std::mutex mu;
    const int d = device_index();
    if (d < 0) return false;
    if (ready[d].load()) return true;
    std::lock_guard<std::mutex> g(mu);
    if (!raise_smem<__nv_bfloat16, 64>() || !raise_smem<__nv_bfloat16, 128>() || !raise_smem<__half, 64>() ||
        !raise_smem<__half, 128>()) {
        cudaGetLastError();
        return false;
    }
    ready[d].store(1);
    return true;
}

// blocks per head: enough for every tile of every sequence, and one more where a row is in none
int64_t tiles_bound(int64_t T, int64_t B, int rows) { return (T + rows - 1) / rows + B; }

int check(const char* name, const concord_attention_params* p) {
    const std::string n(name);
    if (!p) return fail(CONCORD_EINVAL, n + ": null pointer");
    if (p->type != CONCORD_BF16 && p->type != CONCORD_F16) return fail(CONCORD_EINVAL, n + ": operands must be bf16 or fp16");
    if (p->tokens_q < 0 || p->tokens_k < 0 || p->seqs < 1 || p->heads < 1 || p->kv_heads < 1 ||
        p->heads % p->kv_heads || p->tokens_q > INT32_MAX - 256 || p->tokens_k > INT32_MAX - 256)
        return fail(CONCORD_ESHAPE, n + ": bad extents, or heads not a multiple of the key heads");
    if (p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8)
        return fail(CONCORD_ESHAPE, n + ": head_dim must be a multiple of 8 up to 128");
    if (!(p->scale > 0.f) || !(p->scale < INFINITY)) return fail(CONCORD_EINVAL, n + ": scale must be positive");
    if (!p->cu_q || !p->cu_k) return fail(CONCORD_EINVAL, n + ": null pointer");
    if (tiles_bound(std::max(p->tokens_q, p->tokens_k), p->seqs, 128) * p->heads > INT32_MAX ||
        p->tokens_k * p->kv_heads * p->head_dim / 4 / 256 >= INT32_MAX)
        return fail(CONCORD_ETOOBIG, n + ": too many tiles");
    return CONCORD_OK;
}

int check_operand(const char* name, const void* x, int64_t ts, int64_t hs) {
    if (!x) return fail(CONCORD_EINVAL, std::string(name) + ": null pointer");
    if (!aligned(x, 16) || ts % 8 || hs % 8) return fail(CONCORD_EALIGN, std::string(name) + ": rows must start on 16 bytes");
    if (ts <= 0 || hs <= 0 || ts >= (1ll << 38) || hs >= (1ll << 38))
        return fail(CONCORD_ESHAPE, std::string(name) + ": strides must be positive");
    return CONCORD_OK;
}

Params make_params(const concord_attention_params* p, int* err, int* err_host) {
    Params P{};
    P.cuq = p->cu_q; P.cuk = p->cu_k; P.B = (int)p->seqs;
    P.Tq = (int)p->tokens_q; P.Tk = (int)p->tokens_k;
    P.H = (int)p->heads; P.G = (int)(p->heads / p->kv_heads); P.D = (int)p->head_dim;
    P.causal = p->causal; P.scale = p->scale; P.scale2 = p->scale * LOG2E;
    P.err = err;
    P.err_host = err_host;
    return P;
}

template <typename T, int DP>
void launch_fwd(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const Params& P, cudaStream_t st) {
    const int grid = (int)(tiles_bound(P.Tq, P.B, 256) * P.H);
    fwd_kernel<T, DP><<<grid, THREADS, Fwd<DP>::SMEM, st>>>(q, k, v, P);
}

// multiprocessors (asked for once: the sizes of workspaces go by it, so it is one number for the process)
int sm_count() {
    static const int n = [] {
        int d = 0, c = 148;
        if (cudaGetDevice(&d) == cudaSuccess) cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, d);
        return c;
    }();
    return n;
}

// Parts of a key head's query heads: with fewer key blocks than two for each
// SM, as many parts as make up two.  One key head of 16 query heads, 2048
// tokens, heads of 128: 420 us with one part, 45 us with 16 and 33 MB to join.
int splits_of(int64_t tokens_k, int64_t heads, int64_t kv_heads, int* per) {
    const int64_t G = heads / kv_heads, blocks = (tokens_k + 127) / 128 * kv_heads;
    const int64_t want = std::min<int64_t>(G, (2 * sm_count() + blocks - 1) / blocks);
    *per = (int)((G + want - 1) / want);
    return (int)((G + *per - 1) / *per);
}

// chunks of a sequence's keys in range_kernel: of about 256 keys, 32 at most (a lane each)
int chunks_of(int64_t tokens_k, int64_t seqs) {
    return (int)std::min<int64_t>(32, std::max<int64_t>(1, (tokens_k + 256 * seqs - 1) / (256 * seqs)));
}

// workspace of the backward: the parts' sums, where the query heads of a key
// head are split; in fp16 the largest |v| and rows of dout behind them
struct Space {
    size_t vmax, dmax, bytes;
    int splits, per, chunks;
    explicit Space(const concord_attention_params* p) {
        splits = splits_of(p->tokens_k, p->heads, p->kv_heads, &per);
        vmax = splits > 1 ? (size_t)splits * 2 * p->tokens_k * p->kv_heads * p->head_dim * sizeof(float) : 0;
        chunks = chunks_of(p->tokens_k, p->seqs);
        dmax = vmax + (size_t)p->seqs * p->kv_heads * chunks * sizeof(float);
        bytes = p->type == CONCORD_F16 ? dmax + (size_t)p->seqs * p->heads * sizeof(int) : vmax;
    }
};

template <typename T, int DP>
void launch_bwd(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& d,
                const Params& P, cudaStream_t st) {
    if constexpr (__is_same(T, __half)) range_kernel<<<P.B * (P.H / P.G) * P.chunks, 256, 0, st>>>(P);
    if (P.Tq > 0)
        bwd_q_kernel<T, DP><<<(int)(tiles_bound(P.Tq, P.B, 128) * P.H), THREADS, BwdQ<DP>::SMEM, st>>>(q, k, v, d, P);
    bwd_k_kernel<T, DP><<<(int)(tiles_bound(P.Tk, P.B, 128) * (P.H / P.G) * P.splits), THREADS, BwdK<DP>::SMEM, st>>>(
        q, k, v, d, P);
    if (P.splits > 1) {
        const int64_t all = (int64_t)P.Tk * (P.H / P.G) * P.D;
        join_kernel<T><<<(int)((2 * all / 8 + 255) / 256), 256, 0, st>>>(P.part, P.splits, all, static_cast<T*>(P.dk),
                                                                        static_cast<T*>(P.dv));
    }
}

}  // namespace attn
}  // namespace concord

using namespace concord;

extern "C" int concord_attention_fwd(const concord_attention_params* p, const void* q, int64_t q_ts, int64_t q_hs,
                                     const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts,
                                     int64_t v_hs, void* o, void* o_rest, float* lse, void* stream) {
    const char* name = "concord_attention_fwd";
    if (int rc = attn::check(name, p)) return rc;
    if (p->tokens_q == 0) return CONCORD_OK;
    if (p->tokens_k == 0) return fail(CONCORD_ESHAPE, "concord_attention_fwd: no keys");
    if (int rc = attn::check_operand(name, q, q_ts, q_hs)) return rc;
    if (int rc = attn::check_operand(name, k, k_ts, k_hs)) return rc;
    if (int rc = attn::check_operand(name, v, v_ts, v_hs)) return rc;
    if (!o || !lse) return fail(CONCORD_EINVAL, "concord_attention_fwd: null pointer");
    if (!aligned(o, 16) || !aligned(o_rest, 16)) return fail(CONCORD_EALIGN, "concord_attention_fwd: output must be 16-byte aligned");
    if (int rc = bind_current_context(name)) return rc;
    CUtensorMap mq, mk, mv;
    const int bf = p->type == CONCORD_BF16;
    if (!attn::make_map(&mq, q, bf, p->tokens_q, p->heads, p->head_dim, q_ts, q_hs) ||
        !attn::make_map(&mk, k, bf, p->tokens_k, p->kv_heads, p->head_dim, k_ts, k_hs) ||
        !attn::make_map(&mv, v, bf, p->tokens_k, p->kv_heads, p->head_dim, v_ts, v_hs))
        return fail(CONCORD_ELAUNCH, "concord_attention_fwd: TMA descriptor encoding failed");
    int *err, *err_host;
    if (int rc = attn::error_words(&err, &err_host, name)) return rc;
    if (!attn::device_ready()) return fail(CONCORD_ELAUNCH, "concord_attention_fwd: device set-up failed");
    attn::Params P = attn::make_params(p, err, err_host);
    P.o = o;
    P.rest = o_rest;
    P.lse = lse;
    cudaStream_t st = as_stream(stream);
    if (bf) {
        if (p->head_dim <= 64) attn::launch_fwd<__nv_bfloat16, 64>(mq, mk, mv, P, st);
        else attn::launch_fwd<__nv_bfloat16, 128>(mq, mk, mv, P, st);
    } else {
        if (p->head_dim <= 64) attn::launch_fwd<__half, 64>(mq, mk, mv, P, st);
        else attn::launch_fwd<__half, 128>(mq, mk, mv, P, st);
    }
    return check_launch(name);
}

extern "C" size_t concord_attention_bwd_workspace_bytes(const concord_attention_params* p) {
    if (attn::check("concord_attention_bwd_workspace_bytes", p) != CONCORD_OK || p->tokens_k == 0) return 0;
    return attn::Space(p).bytes;
}

extern "C" int concord_attention_bwd(const concord_attention_params* p, const void* q, int64_t q_ts, int64_t q_hs,
                                     const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts,
                                     int64_t v_hs, const void* o, const void* o_rest, const float* lse,
                                     const void* dout, int64_t do_ts, int64_t do_hs, float* delta, void* dq, void* dk, void* dv,
                                     void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "concord_attention_bwd";
    if (int rc = attn::check(name, p)) return rc;
    if (p->tokens_q == 0 || p->tokens_k == 0) return fail(CONCORD_ESHAPE, "concord_attention_bwd: no rows");
    if (int rc = attn::check_operand(name, q, q_ts, q_hs)) return rc;
    if (int rc = attn::check_operand(name, k, k_ts, k_hs)) return rc;
    if (int rc = attn::check_operand(name, v, v_ts, v_hs)) return rc;
    if (int rc = attn::check_operand(name, dout, do_ts, do_hs)) return rc;
    if (!o || !o_rest || !lse || !delta || !dq || !dk || !dv) return fail(CONCORD_EINVAL, "concord_attention_bwd: null pointer");
    if (!aligned(o, 16) || !aligned(o_rest, 16) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16))
        return fail(CONCORD_EALIGN, "concord_attention_bwd: tensors must be 16-byte aligned");
    if (workspace_bytes < concord_attention_bwd_workspace_bytes(p) || (!workspace && workspace_bytes) ||
        !aligned(workspace, 16))
        return fail(CONCORD_EWORKSPACE, "concord_attention_bwd: workspace too small or not 16-byte aligned");
    if (int rc = bind_current_context(name)) return rc;
    CUtensorMap mq, mk, mv, md;
    const int bf = p->type == CONCORD_BF16;
    if (!attn::make_map(&mq, q, bf, p->tokens_q, p->heads, p->head_dim, q_ts, q_hs) ||
        !attn::make_map(&mk, k, bf, p->tokens_k, p->kv_heads, p->head_dim, k_ts, k_hs) ||
        !attn::make_map(&mv, v, bf, p->tokens_k, p->kv_heads, p->head_dim, v_ts, v_hs) ||
        !attn::make_map(&md, dout, bf, p->tokens_q, p->heads, p->head_dim, do_ts, do_hs))
        return fail(CONCORD_ELAUNCH, "concord_attention_bwd: TMA descriptor encoding failed");
    int *err, *err_host;
    if (int rc = attn::error_words(&err, &err_host, name)) return rc;
    if (!attn::device_ready()) return fail(CONCORD_ELAUNCH, "concord_attention_bwd: device set-up failed");
    attn::Params P = attn::make_params(p, err, err_host);
    P.o = const_cast<void*>(o);
    P.rest = const_cast<void*>(o_rest);
    P.lse = const_cast<float*>(lse);
    P.dout = dout;
    P.do_ts = do_ts;
    P.do_hs = do_hs;
    P.delta = delta;
    P.dq = dq;
    P.dk = dk;
    P.dv = dv;
    const attn::Space space(p);
    P.splits = space.splits;
    P.per = space.per;
    P.chunks = space.chunks;
    P.part = static_cast<float*>(workspace);
    P.vmax = reinterpret_cast<float*>(static_cast<char*>(workspace) + space.vmax);
    P.dmax = reinterpret_cast<int*>(static_cast<char*>(workspace) + space.dmax);
    P.v = v;
    P.v_ts = v_ts;
    P.v_hs = v_hs;
    cudaStream_t st = as_stream(stream);
    if (bf) {
        if (p->head_dim <= 64) attn::launch_bwd<__nv_bfloat16, 64>(mq, mk, mv, md, P, st);
        else attn::launch_bwd<__nv_bfloat16, 128>(mq, mk, mv, md, P, st);
    } else {
        if (p->head_dim <= 64) attn::launch_bwd<__half, 64>(mq, mk, mv, md, P, st);
        else attn::launch_bwd<__half, 128>(mq, mk, mv, md, P, st);
    }
    return check_launch(name);
}

// the attention kernels' error word on the current device (0: no wait ran out)
extern "C" int concord_attention_error(int32_t reset) {
    volatile int* host = attn::host_word();
    void* p = nullptr;
    int v = 0;
    if (!host || cudaGetSymbolAddress(&p, attn::g_err) != cudaSuccess ||
        cudaMemcpy(&v, p, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess)
        return -1;
    if (!v) v = *host;
    if (reset) {
        if (cudaMemset(p, 0, sizeof(int)) != cudaSuccess) return -1;
        *host = 0;
    }
    return v;
}

extern "C" int32_t* concord_attention_error_word(void) { return const_cast<int32_t*>(attn::host_word()); }

extern "C" int concord_attention_wait_check(void* stream) {
    const char* name = "concord_attention_wait_check";
    int *err, *err_host;
    if (int rc = attn::error_words(&err, &err_host, name)) return rc;
    attn::wait_check_kernel<<<1, 64, 0, as_stream(stream)>>>(err, err_host);
    return check_launch(name);
}
