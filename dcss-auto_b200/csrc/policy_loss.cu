// Clipped policy loss with KL and entropy terms, and its gradient in the same
// pass (sm_100a).
//
//   r = e^delta, delta = logp - old     d = ref - logp
//   L = sum_i w_i ( -min(r A, clip(r) A) + kl (e^d - d - 1) - ent H )
//   dL/dlogp = w ( -r A [not cut] + kl (1 - e^d) )      dL/dH = -ent w
//
// over the tokens that the mask keeps, with w = 1 / tokens (mean over tokens) or
// 1 / (tokens of the row * rows that have any) (every row counts the same). A
// token that the mask leaves out is never looked at: its values may be anything.
//
// A token is cut where the clipped product is the smaller one: delta beyond
// log(1 + high) with A > 0, or below log(1 - low) with A < 0. Its gradient jumps
// there, so the side is that of the exact difference: where the rounded one is the rounded border itself it is
// taken in 64 bits, elsewhere rounding cannot have moved it across. e^d - d - 1 and e^delta - delta - 1 are taken from their
// series near 0, where the difference would cancel. Sums are fp64 from four
// tokens on, joined in a fixed order.
//
// The weights need the mask's counts before any token can be finished. Up to 32,768 tokens are a cluster's: each of its blocks
// counts the whole mask and takes a part of the tokens, the first one adds the blocks' sums. More have a launch ahead
// that counts (a byte a token, where the main pass reads 13 and more); without a mask it only clears the count of
// blocks that are done, by which the last one knows that it is to add the blocks' sums.
//
// Measured (one B200): 16,384 tokens 4.2 us (one block in place of eight: 10.5), 512 x 4,099 tokens by rows with a mask and the KL
// term 20 us (floor 5.4 at 6.56 TB/s), 128 x 65,536 with every term 46.6 us (37.1; 80 instructions a token fill half of the issue slots
// meanwhile).
#include <math.h>

#include "d1_common.cuh"
#include "d1_elem.cuh"
#include "d1_pdl.cuh"
#include "d1_rows.h"

namespace d1 {
namespace pl {

constexpr int SMS = 148, THREADS = 256, BLOCKS = SMS * 3, TERMS = 5;
constexpr int SMALL = 32768, SMALL_THREADS = 512, SMALL_ROWS = 2048, MOST_TOGETHER = 8;  // a cluster's batch
constexpr int PIECE = 4096, LONG = 16384;  // tokens of a row too long for one warp that a warp counts; of such a row
constexpr int TEAM = 4;  // warps that count a row of more than 1,024 tokens

struct Rows {  // fp32 [rows, length]: element (r, i) at p[r * ld + i]
    const float *p;
    int64_t ld;
};

struct Args {
    Rows logp, old, adv, ref, entropy;  // ref.p, entropy.p may be NULL
    int per_row;                        // adv is one number for each row
    const uint8_t *mask;                // may be NULL
    int64_t ld_mask;
    int64_t rows, length, count;        // count = rows * length
    double over, under;                 // log(1 + high), log(1 - low)
    float over32, under32;              // the same, rounded
    float most, least;                  // 1 + high, 1 - low
    float kl, ent;
    int by_row;                         // mean of the rows' means
    float *loss, *stats, *dlogp, *dentropy;
    double *parts;                      // [blocks][TERMS]
    int *counts;                        // tokens of row r (by_row)
    int *totals;                        // [count_blocks] tokens, or rows that have any
    unsigned *done;                     // blocks of the main pass that are done
    int blocks, count_blocks;
};

// e^v - 1 - v, given e^v. Near 0 from the series v^2 (1/2! + v/3! + ...), whose first term left out is below
// 2^-25 of the sum.
__device__ __forceinline__ float beyond_linear(float v, float grown) {
    float s = 1.f / 362880.f;
    s = fmaf(s, v, 1.f / 40320.f);
    s = fmaf(s, v, 1.f / 5040.f);
    s = fmaf(s, v, 1.f / 720.f);
    s = fmaf(s, v, 1.f / 120.f);
    s = fmaf(s, v, 1.f / 24.f);
    s = fmaf(s, v, 1.f / 6.f);
    s = fmaf(s, v, 0.5f);
    return fabsf(v) < 0.5f ? s * v * v : grown - 1.f - v;
}

struct Sums {
    float t[TERMS];
};

// One token of weight w: its share of the five terms (times w) and its gradient.
__device__ __forceinline__ float token(const Args &a, float logp, float old, float adv, float ref, float h, float w, Sums &s) {
    const float delta = logp - old, r = expf(delta);
    bool over = delta > a.over32, under = delta < a.under32;
    if (delta == a.over32 || delta == a.under32) {  // rounding is monotonic: only here may the exact difference lie on the other side
        const double wide = (double)logp - (double)old;
        over = wide > a.over, under = wide < a.under;
    }
    const bool cut = (over && adv > 0.f) || (under && adv < 0.f);
    // an advantage or a coefficient of 0 is 0 beside a finite difference whose power passes fp32
    const float gain = adv == 0.f && delta < INFINITY ? 0.f : r * adv;
    s.t[0] -= w * (cut ? (over ? a.most : a.least) * adv : gain);
    float g = cut ? 0.f : -gain;
    if (a.ref.p) {
        const float d = ref - logp, grown = expf(d), k = beyond_linear(d, grown);
        s.t[1] += w * k;
        if (a.kl != 0.f) g = fmaf(-a.kl, fabsf(d) < 0.5f ? d + k : grown - 1.f, g);  // e^d - 1
    }
    if (a.entropy.p) s.t[2] += w * h;
    if (cut) s.t[3] += w;
    s.t[4] += w * beyond_linear(delta, r);
    return g * w;
}

__device__ __forceinline__ float weight_of(const Args &a, const int *row_counts, int64_t row, float flat, float rows_inv) {
    if (!a.by_row) return flat;
    const int n = a.mask ? row_counts[row] : (int)min(a.length, (int64_t)INT32_MAX);
    return n ? rows_inv / (float)n : 0.f;
}

// V tokens as they are read.
template <int V> struct Held {
    Elems<float, V> logp, old, adv, ref, h;
    Elems<uint8_t, V> keep;
};
template <int V> __device__ __forceinline__ int64_t row_of(const Args &a, int64_t i) {
    return a.count <= INT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)a.length) : i / a.length;
}
template <int V> __device__ __forceinline__ void load(const Args &a, int64_t i, Held<V> &t) {
    if constexpr (V > 1) {
        t.logp = *reinterpret_cast<const Elems<float, V> *>(a.logp.p + i);
        t.old = *reinterpret_cast<const Elems<float, V> *>(a.old.p + i);
        if (!a.per_row) t.adv = *reinterpret_cast<const Elems<float, V> *>(a.adv.p + i);
        if (a.ref.p) t.ref = *reinterpret_cast<const Elems<float, V> *>(a.ref.p + i);
        if (a.entropy.p) t.h = *reinterpret_cast<const Elems<float, V> *>(a.entropy.p + i);
        if (a.mask) t.keep = *reinterpret_cast<const Elems<uint8_t, V> *>(a.mask + i);
    } else {
        const int64_t row = row_of<V>(a, i), col = i - row * a.length;
        t.logp.v[0] = a.logp.p[row * a.logp.ld + col];
        t.old.v[0] = a.old.p[row * a.old.ld + col];
        if (!a.per_row) t.adv.v[0] = a.adv.p[row * a.adv.ld + col];
        if (a.ref.p) t.ref.v[0] = a.ref.p[row * a.ref.ld + col];
        if (a.entropy.p) t.h.v[0] = a.entropy.p[row * a.entropy.ld + col];
        if (a.mask) t.keep.v[0] = a.mask[row * a.ld_mask + col];
    }
}

// Everything of V tokens from i on.
template <int V>
__device__ __forceinline__ void work(const Args &a, const int *row_counts, float flat, float rows_inv, int64_t i, const Held<V> &t, double (&total)[TERMS]) {
    int64_t row = 0, col = 0;
    if (a.by_row || a.per_row) row = row_of<V>(a, i), col = i - row * a.length;
    float row_adv = a.per_row ? a.adv.p[row * a.adv.ld] : 0.f, w = weight_of(a, row_counts, row, flat, rows_inv);
    Sums s = {};
    Elems<float, V> g, dh;
#pragma unroll
    for (int v = 0; v < V; v++) {
        if (V > 1 && v && (a.by_row || a.per_row) && ++col == a.length) {  // the next token is the next row's first
            col = 0;
            row++;
            if (a.per_row) row_adv = a.adv.p[row * a.adv.ld];
            w = weight_of(a, row_counts, row, flat, rows_inv);
        }
        g.v[v] = dh.v[v] = 0.f;
        if (!a.mask || t.keep.v[v]) {
            g.v[v] = token(a, t.logp.v[v], t.old.v[v], a.per_row ? row_adv : t.adv.v[v], t.ref.v[v], t.h.v[v], w, s);
            dh.v[v] = -a.ent * w;
        }
    }
    if (a.dlogp) *reinterpret_cast<Elems<float, V> *>(a.dlogp + i) = g;
    if (a.dentropy) *reinterpret_cast<Elems<float, V> *>(a.dentropy + i) = dh;
#pragma unroll
    for (int k = 0; k < TERMS; k++) total[k] += (double)s.t[k];
}

// The tokens first, first + stride, ..., V at a time along the flat index (V > 1: every operand's rows lie end to
// end). The first ones' loads are under way before the weights are known. (Loads of the next ones during the arithmetic of
// these took 20 registers a thread more, and 57 us in place of 46 for 128 x 65,536 tokens: spills, or fewer warps.)
template <int V> struct Pass {
    int64_t i, step;
    Held<V> now;

    __device__ __forceinline__ Pass(const Args &a, int64_t first, int64_t stride) : i(first * V), step(stride * V) {
        if (i < a.count) load<V>(a, i, now);
    }
    __device__ __forceinline__ void run(const Args &a, const int *row_counts, float flat, float rows_inv, double (&total)[TERMS]) {
        while (i < a.count) {
            work<V>(a, row_counts, flat, rows_inv, i, now, total);
            i += step;
            if (i < a.count) load<V>(a, i, now);
        }
    }
};

// The block's sums in thread 0, added in a fixed order.
template <int N> __device__ __forceinline__ void join(double (&total)[TERMS], double (*shared)[TERMS]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < TERMS; k++) {
#pragma unroll
        for (int o = 16; o; o >>= 1) total[k] += __shfl_xor_sync(0xffffffffu, total[k], o);
        if (lane == 0) shared[warp][k] = total[k];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int k = 0; k < TERMS; k++) {
            total[k] = lane < N / 32 ? shared[lane][k] : 0.;
#pragma unroll
            for (int o = 16; o; o >>= 1) total[k] += __shfl_xor_sync(0xffffffffu, total[k], o);
        }
    }
}

__device__ __forceinline__ void finish(const Args &a, const double (&t)[TERMS]) {
    if (a.loss) *a.loss = (float)(t[0] + (a.kl != 0.f ? (double)a.kl * t[1] : 0.) - (a.ent != 0.f ? (double)a.ent * t[2] : 0.));
    if (a.stats)
        for (int k = 0; k < TERMS; k++) a.stats[k] = (float)t[k];
}

// Weight of a token in the mean over tokens, and 1 / rows that have any.
__device__ __forceinline__ float inverse(int64_t n) { return n > 0 ? (float)(1. / (double)n) : 0.f; }

// How many of `n` bytes are not 0, by the threads k, k + stride, ... of those that count them. Whole 16-byte pieces are read
// as such, wherever the row begins.
__device__ __forceinline__ int count_bytes(const uint8_t *p, int64_t n, int k, int stride) {
    const int64_t head = min(n, (int64_t)(-(intptr_t)p & 15)), pieces = (n - head) / 16, tail = head + pieces * 16;
    int sum = 0;
    for (int64_t i = k; i < head; i += stride) sum += p[i] != 0;
    const uint4 *const q = reinterpret_cast<const uint4 *>(p + head);
#pragma unroll 4
    for (int64_t i = k; i < pieces; i += stride) {
        const uint4 w = q[i];
        sum += __popc(__vcmpne4(w.x, 0) & 0x01010101u) + __popc(__vcmpne4(w.y, 0) & 0x01010101u) + __popc(__vcmpne4(w.z, 0) & 0x01010101u) +
               __popc(__vcmpne4(w.w, 0) & 0x01010101u);
    }
    for (int64_t i = tail + k; i < n; i += stride) sum += p[i] != 0;
    return sum;
}

// Sum over the block of whole numbers, in every thread.
template <int N> __device__ __forceinline__ int block_sum(int x, int *shared) {
    x = __reduce_add_sync(0xffffffffu, x);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < N / 32; w++) x += shared[w];
    __syncthreads();
    return x;
}

// The tokens that the mask keeps: of a flat batch, of rows by a warp each, of long ones by the blocks (into counts that are 0
// then), and what totals[] says of them.
__global__ void __launch_bounds__(THREADS) count_kernel(Args a) {
    __shared__ int shared[THREADS / 32];
    pdl_launch();
    pdl_wait();
    const int lane = threadIdx.x & 31, warps = (int)gridDim.x * (THREADS / 32), at = (int)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    int sum = 0;
    if (!a.mask) {
    } else if (!a.by_row) {
        if (a.ld_mask == a.length || a.rows == 1) {
            sum = count_bytes(a.mask, a.count, (int)blockIdx.x * THREADS + threadIdx.x, (int)gridDim.x * THREADS);
        } else
            for (int64_t row = at; row < a.rows; row += warps) sum += count_bytes(a.mask + row * a.ld_mask, a.length, lane, 32);
    } else if (a.length <= 1024) {
        for (int64_t row = at; row < a.rows; row += warps) {
            const int n = __reduce_add_sync(0xffffffffu, count_bytes(a.mask + row * a.ld_mask, a.length, lane, 32));
            if (lane == 0) a.counts[row] = n;
            sum += lane == 0 && n;
        }
    } else if (a.length <= LONG) {  // TEAM warps a row, two rows a block
        const int team = threadIdx.x / (32 * TEAM);
        for (int64_t row = (int64_t)blockIdx.x * 2; row < a.rows; row += (int64_t)gridDim.x * 2) {
            int n = 0;
            if (row + team < a.rows) n = __reduce_add_sync(0xffffffffu, count_bytes(a.mask + (row + team) * a.ld_mask, a.length, threadIdx.x % (32 * TEAM), 32 * TEAM));
            __syncthreads();
            if (lane == 0) shared[threadIdx.x >> 5] = n;
            __syncthreads();
            if (threadIdx.x % (32 * TEAM) == 0 && row + team < a.rows) {
                n = shared[TEAM * team] + shared[TEAM * team + 1] + shared[TEAM * team + 2] + shared[TEAM * team + 3];
                a.counts[row + team] = n;
                sum += n > 0;
            }
        }
        __syncthreads();
    } else {
        const int64_t pieces = (a.length + PIECE - 1) / PIECE;
        for (int64_t p = at; p < a.rows * pieces; p += warps) {
            const int64_t row = p / pieces, c0 = (p - row * pieces) * PIECE;
            const int n = __reduce_add_sync(0xffffffffu, count_bytes(a.mask + row * a.ld_mask + c0, min((int64_t)PIECE, a.length - c0), lane, 32));
            // whoever adds the row's first tokens counts the row
            if (lane == 0 && n && atomicAdd(a.counts + row, n) == 0) sum++;
        }
    }
    sum = block_sum<THREADS>(sum, shared);
    if (threadIdx.x == 0) a.totals[blockIdx.x] = sum;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.done = 0;
}

template <int V> __global__ void __launch_bounds__(THREADS, 3) loss_kernel(Args a) {
    __shared__ double shared[THREADS / 32][TERMS];
    __shared__ int counted[THREADS / 32];
    pdl_launch();
    Pass<V> pass(a, (int64_t)blockIdx.x * THREADS + threadIdx.x, (int64_t)gridDim.x * THREADS);  // not what the launch before this writes
    pdl_wait();
    int n = 0;
    if (a.mask) {
        for (int b = threadIdx.x; b < a.count_blocks; b += THREADS) n += a.totals[b];
        n = block_sum<THREADS>(n, counted);
    }
    double total[TERMS] = {};
    pass.run(a, a.counts, inverse(a.mask ? n : a.count), inverse(a.mask ? n : a.rows), total);
    join<THREADS>(total, shared);
    __shared__ bool last;
    if (threadIdx.x == 0) {
        for (int k = 0; k < TERMS; k++) a.parts[(int64_t)blockIdx.x * TERMS + k] = total[k];
        __threadfence();
        last = atomicAdd(a.done, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    for (int k = 0; k < TERMS; k++) total[k] = 0.;
    for (int b = threadIdx.x; b < a.blocks; b += THREADS)
        for (int k = 0; k < TERMS; k++) total[k] += __ldcg(a.parts + (int64_t)b * TERMS + k);
    join<THREADS>(total, shared);
    if (threadIdx.x == 0) finish(a, total);
}

// All of a small batch by one cluster.
template <int V> __global__ void __launch_bounds__(SMALL_THREADS) small_kernel(Args a) {
    __shared__ double shared[SMALL_THREADS / 32][TERMS], blocks[MOST_TOGETHER][TERMS];
    __shared__ int counts[SMALL_ROWS], counted[SMALL_THREADS / 32];
    uint32_t rank, together;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(together));
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // all blocks have begun before one writes to the first
    Pass<V> pass(a, rank * SMALL_THREADS + threadIdx.x, together * SMALL_THREADS);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int n = 0;
    if (a.mask) {
        if (!a.by_row && (a.ld_mask == a.length || a.rows == 1)) {
            n = count_bytes(a.mask, a.count, threadIdx.x, SMALL_THREADS);
        } else {
            for (int row = warp; row < (int)a.rows; row += SMALL_THREADS / 32) {
                const int k = __reduce_add_sync(0xffffffffu, count_bytes(a.mask + row * a.ld_mask, a.length, lane, 32));
                if (lane == 0) {
                    counts[row] = k;
                    n += a.by_row ? k > 0 : k;
                }
            }
        }
        n = block_sum<SMALL_THREADS>(n, counted);  // and the rows' counts are there
    }
    double total[TERMS] = {};
    pass.run(a, counts, inverse(a.mask ? n : a.count), inverse(a.mask ? n : a.rows), total);
    join<SMALL_THREADS>(total, shared);
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (threadIdx.x == 0) {
        uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(blocks[rank])), to;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(at));
        for (int k = 0; k < TERMS; k++) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to + 8 * k), "d"(total[k]) : "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0 && threadIdx.x == 0) {
        for (int k = 0; k < TERMS; k++) {
            total[k] = 0.;
            for (uint32_t b = 0; b < together; b++) total[k] += blocks[b][k];
        }
        finish(a, total);
    }
}

static bool is_small(int64_t rows, int64_t count) { return count <= SMALL && (rows <= SMALL_ROWS || !count); }
constexpr int64_t PART_BYTES = (int64_t)BLOCKS * TERMS * 8;

static bool rows_ok(const void *p, int64_t ld, int64_t rows, int64_t length, bool needed) {
    if (!p) return !needed;
    return ld >= 0 && ld <= ((int64_t)1 << 42) && aligned_to(4, p);
}

}  // namespace pl
}  // namespace d1

extern "C" int64_t d1_policy_loss_work_bytes(int64_t rows, int64_t length) {
    if (rows < 0 || length < 0 || length > INT32_MAX || (length && rows > ((int64_t)1 << 40) / length)) return -1;
    if (d1::pl::is_small(rows, rows * length)) return 0;
    return d1::pl::PART_BYTES + 4 * (1 + d1::pl::BLOCKS + rows);
}

extern "C" int d1_policy_loss(const float *logp, int64_t ld_logp, const float *old_logp, int64_t ld_old,
                              const float *advantage, int64_t ld_advantage, int per_row, const float *ref_logp,
                              int64_t ld_ref, const float *entropy, int64_t ld_entropy, const uint8_t *mask,
                              int64_t ld_mask, int64_t rows, int64_t length, double clip_low, double clip_high,
                              double kl_coef, double ent_coef, int by_row, float *loss, float *stats, float *dlogp,
                              float *dentropy, void *work, void *stream) {
    using namespace d1;
    using namespace d1::pl;
    const int64_t bytes = d1_policy_loss_work_bytes(rows, length);
    const int64_t count = bytes < 0 ? 0 : rows * length;
    if (bytes < 0 || !rows_ok(logp, ld_logp, rows, length, count > 0) || !rows_ok(old_logp, ld_old, rows, length, count > 0) ||
        !rows_ok(advantage, ld_advantage, rows, length, count > 0) || !rows_ok(ref_logp, ld_ref, rows, length, false) ||
        !rows_ok(entropy, ld_entropy, rows, length, false) || ld_mask < 0 || ld_mask > ((int64_t)1 << 42) ||
        !(clip_low >= 0.) || !(clip_high >= 0.) || !(kl_coef == kl_coef) || !(ent_coef == ent_coef) ||
        !aligned_to(4, loss, stats, dlogp, dentropy) || (bytes && !work) || !aligned_to(8, work) || (mask && count > INT32_MAX))
        return D1_ERR_BAD_ARGUMENT;
    // the gradients are contiguous and share no memory with what the call reads
    const RowSpan d[2] = {{(uintptr_t)dlogp, dlogp ? 1 : 0, 4 * count, 0}, {(uintptr_t)dentropy, dentropy ? 1 : 0, 4 * count, 0}};
    const RowSpan in[6] = {{(uintptr_t)logp, rows, 4 * length, 4 * ld_logp},
                           {(uintptr_t)old_logp, rows, 4 * length, 4 * ld_old},
                           {(uintptr_t)advantage, rows, per_row ? 4 : 4 * length, 4 * ld_advantage},
                           {(uintptr_t)ref_logp, ref_logp ? rows : 0, 4 * length, 4 * ld_ref},
                           {(uintptr_t)entropy, entropy ? rows : 0, 4 * length, 4 * ld_entropy},
                           {(uintptr_t)mask, mask ? rows : 0, length, ld_mask}};
    for (const RowSpan &o : d)
        for (const RowSpan &i : in)
            if (rows_overlap(o, i)) return D1_ERR_BAD_ARGUMENT;
    if (rows_overlap(d[0], d[1])) return D1_ERR_BAD_ARGUMENT;
    Args a{};
    a.logp = {logp, ld_logp}, a.old = {old_logp, ld_old}, a.adv = {advantage, ld_advantage}, a.ref = {ref_logp, ld_ref};
    a.entropy = {entropy, ld_entropy};
    a.per_row = per_row != 0, a.mask = mask, a.ld_mask = ld_mask;
    a.rows = count ? rows : 0, a.length = length, a.count = count;  // no rows without a token: their counts need no room
    a.over = log1p(clip_high), a.under = clip_low < 1. ? log1p(-clip_low) : -INFINITY;
    a.over32 = (float)a.over, a.under32 = (float)a.under;
    a.most = (float)(1. + clip_high), a.least = (float)(1. - clip_low);
    a.kl = (float)kl_coef, a.ent = (float)ent_coef, a.by_row = by_row != 0;
    a.loss = loss, a.stats = stats, a.dlogp = dlogp, a.dentropy = dentropy;
    a.parts = (double *)work;
    a.done = work ? (unsigned *)((char *)work + PART_BYTES) : nullptr;
    a.totals = work ? (int *)a.done + 1 : nullptr;
    a.counts = work ? a.totals + BLOCKS : nullptr;
    const cudaStream_t s = (cudaStream_t)stream;
    const auto flat = [&](const void *p, int64_t ld, int align) { return !p || (ld == length || rows == 1) && aligned_to(align, p); };
    const bool four = count % 4 == 0 && flat(logp, ld_logp, 16) && flat(old_logp, ld_old, 16) &&
                      (per_row || flat(advantage, ld_advantage, 16)) && flat(ref_logp, ld_ref, 16) &&
                      flat(entropy, ld_entropy, 16) && flat(mask, ld_mask, 4) && aligned_to(16, dlogp, dentropy);
    cudaLaunchAttribute attr;
    if (is_small(rows, count)) {
        int together = 1;
        while (together < MOST_TOGETHER && together * SMALL_THREADS * 4 < count) together *= 2;
        cudaLaunchConfig_t cfg = pdl_config(dim3(together), dim3(SMALL_THREADS), 0, s, &attr);
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = together;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        return (int)cudaLaunchKernelEx(&cfg, four ? small_kernel<4> : small_kernel<1>, a);
    }
    const int64_t want = (count + THREADS * 4 - 1) / (THREADS * 4);
    a.blocks = (int)(want < BLOCKS ? want : BLOCKS);
    cudaLaunchConfig_t cfg = pdl_config(dim3(a.blocks), dim3(THREADS), 0, s, &attr);
    if (mask && by_row && length > LONG)
        if (cudaError_t e = cudaMemsetAsync(a.counts, 0, (size_t)(4 * rows), s)) return (int)e;
    // 16 bytes a thread; a row a warp, or two a block; a piece a warp
    const int64_t blocks = !mask ? 1
                           : !by_row ? (flat(mask, ld_mask, 1) ? (count + THREADS * 16 - 1) / (THREADS * 16) : (rows + 7) / 8)
                           : length <= 1024 ? (rows + 7) / 8
                           : length <= LONG ? (rows + 1) / 2
                                            : (rows * ((length + PIECE - 1) / PIECE) + 7) / 8;
    a.count_blocks = (int)(blocks < BLOCKS ? blocks : BLOCKS);
    cudaLaunchConfig_t before = cfg;
    before.gridDim = dim3(a.count_blocks);
    before.numAttrs = 0;
    if (cudaError_t e = cudaLaunchKernelEx(&before, count_kernel, a)) return (int)e;
    return (int)cudaLaunchKernelEx(&cfg, four ? loss_kernel<4> : loss_kernel<1>, a);
}
