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
// there, so the side is decided in 64 bits, where the difference of two fp32
// numbers is exact. e^d - d - 1 and e^delta - delta - 1 are taken from their
// series near 0, where the difference would cancel. Sums are fp64 from four
// tokens on, joined in a fixed order.
//
// The weights need the mask's counts before any token can be finished. Small
// batches count in the one block that does the rest; larger ones clear and fill
// integer counts in a launch ahead (whole numbers: the order does not matter),
// which reads a byte a token where the main pass reads 13 and more.
#include <math.h>

#include "d1_common.cuh"
#include "d1_elem.cuh"
#include "d1_pdl.cuh"
#include "d1_rows.h"

namespace d1 {
namespace pl {

constexpr int SMS = 148, THREADS = 256, BLOCKS = SMS * 4, SMALL = 16384, SMALL_THREADS = 1024, SMALL_ROWS = 2048, TERMS = 5;

struct Rows {  // fp32 [rows, length]: element (r, i) at p[r * ld + i * step]
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
    float most, least;                  // 1 + high, 1 - low
    float kl, ent;
    int by_row;                         // mean of the rows' means
    float *loss, *stats, *dlogp, *dentropy;
    double *parts;                      // [blocks][TERMS]
    int *counts;                        // [0] tokens or rows that have any; [1 + r] tokens of row r
    int blocks;
};

// e^v - 1 - v.
__device__ __forceinline__ float beyond_linear(float v, float e1) {
    if (fabsf(v) >= 0.5f) return e1 - v;
    // v^2 (1/2! + v/3! + ...): the first term left out is below 2^-25 of the sum
    float s = 1.f / 362880.f;
    s = fmaf(s, v, 1.f / 40320.f);
    s = fmaf(s, v, 1.f / 5040.f);
    s = fmaf(s, v, 1.f / 720.f);
    s = fmaf(s, v, 1.f / 120.f);
    s = fmaf(s, v, 1.f / 24.f);
    s = fmaf(s, v, 1.f / 6.f);
    s = fmaf(s, v, 0.5f);
    return s * v * v;
}

struct Sums {
    float t[TERMS];
};

// One token of weight w: its share of the five terms (times w) and its gradient.
__device__ __forceinline__ float token(const Args &a, float logp, float old, float adv, float ref, float h, float w, Sums &s) {
    const double wide = (double)logp - (double)old;
    const bool over = wide > a.over, under = wide < a.under;
    const bool cut = (over && adv > 0.f) || (under && adv < 0.f);
    const float delta = logp - old, r = expf(delta);
    s.t[0] -= w * ((cut ? (over ? a.most : a.least) : r) * adv);
    float g = cut ? 0.f : -adv * r;
    if (a.ref.p) {
        const float d = ref - logp, e1 = expm1f(d);
        s.t[1] += w * beyond_linear(d, e1);
        g = fmaf(-a.kl, e1, g);
    }
    if (a.entropy.p) s.t[2] += w * h;
    if (cut) s.t[3] += w;
    s.t[4] += w * beyond_linear(delta, r - 1.f);
    return g * w;
}

__device__ __forceinline__ float weight_of(const Args &a, const int *row_counts, int64_t row, float flat, float rows_inv) {
    if (!a.by_row) return flat;
    const int n = a.mask ? row_counts[row] : (int)min(a.length, (int64_t)INT32_MAX);
    return n ? rows_inv / (float)n : 0.f;
}

// Everything of the tokens first, first + stride, ..., V at a time along the flat index (V > 1: every
// operand's rows lie end to end).
template <int V>
__device__ __forceinline__ void pass(const Args &a, const int *row_counts, float flat, float rows_inv, int64_t first, int64_t stride, double (&total)[TERMS]) {
    const bool small = a.count <= INT32_MAX;
    for (int64_t i = first * V; i < a.count; i += stride * V) {
        int64_t row = small ? (int64_t)((uint32_t)i / (uint32_t)a.length) : i / a.length, col = i - row * a.length;
        Sums s = {};
        Elems<float, V> lp, old, adv, ref = {}, h = {}, g, dh;
        Elems<uint8_t, V> keep;
        if constexpr (V > 1) {
            lp = *reinterpret_cast<const Elems<float, V> *>(a.logp.p + i);
            old = *reinterpret_cast<const Elems<float, V> *>(a.old.p + i);
            if (!a.per_row) adv = *reinterpret_cast<const Elems<float, V> *>(a.adv.p + i);
            if (a.ref.p) ref = *reinterpret_cast<const Elems<float, V> *>(a.ref.p + i);
            if (a.entropy.p) h = *reinterpret_cast<const Elems<float, V> *>(a.entropy.p + i);
            if (a.mask) keep = *reinterpret_cast<const Elems<uint8_t, V> *>(a.mask + i);
        } else {
            lp.v[0] = a.logp.p[row * a.logp.ld + col];
            old.v[0] = a.old.p[row * a.old.ld + col];
            if (!a.per_row) adv.v[0] = a.adv.p[row * a.adv.ld + col];
            if (a.ref.p) ref.v[0] = a.ref.p[row * a.ref.ld + col];
            if (a.entropy.p) h.v[0] = a.entropy.p[row * a.entropy.ld + col];
            if (a.mask) keep.v[0] = a.mask[row * a.ld_mask + col];
        }
        float row_adv = a.per_row ? a.adv.p[row * a.adv.ld] : 0.f, w = weight_of(a, row_counts, row, flat, rows_inv);
#pragma unroll
        for (int v = 0; v < V; v++) {
            if (V > 1 && v && ++col == a.length) {  // the next token is the next row's first
                col = 0;
                row++;
                if (a.per_row) row_adv = a.adv.p[row * a.adv.ld];
                w = weight_of(a, row_counts, row, flat, rows_inv);
            }
            g.v[v] = dh.v[v] = 0.f;
            if (!a.mask || keep.v[v]) {
                g.v[v] = token(a, lp.v[v], old.v[v], a.per_row ? row_adv : adv.v[v], ref.v[v], h.v[v], w, s);
                dh.v[v] = -a.ent * w;
            }
        }
        if (a.dlogp) *reinterpret_cast<Elems<float, V> *>(a.dlogp + i) = g;
        if (a.dentropy) *reinterpret_cast<Elems<float, V> *>(a.dentropy + i) = dh;
#pragma unroll
        for (int k = 0; k < TERMS; k++) total[k] += (double)s.t[k];
    }
}

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
    if (a.loss) *a.loss = (float)(t[0] + (double)a.kl * t[1] - (double)a.ent * t[2]);
    if (a.stats)
        for (int k = 0; k < TERMS; k++) a.stats[k] = (float)t[k];
}

// Weight of a token in the mean over tokens, and 1 / rows that have any.
__device__ __forceinline__ float inverse(int64_t n) { return n > 0 ? (float)(1. / (double)n) : 0.f; }

// The tokens of every row that the mask keeps, and counts[0].
__global__ void __launch_bounds__(THREADS) count_kernel(Args a) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (THREADS / 32), at = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    // a warp takes 1024 tokens of a row at a time
    const int64_t pieces = (a.length + 1023) / 1024;
    int sum = 0;
    for (int64_t p = at; p < a.rows * pieces; p += warps) {
        const int64_t row = p / pieces, c0 = (p - row * pieces) * 1024;
        const uint8_t *m = a.mask + row * a.ld_mask + c0;
        const int n = (int)min((int64_t)1024, a.length - c0);
        int k = 0;
#pragma unroll 8
        for (int i = lane; i < n; i += 32) k += m[i] != 0;
        if (a.by_row) {
            k = __reduce_add_sync(0xffffffffu, k);
            // whoever adds the row's first tokens counts the row
            if (lane == 0 && k && atomicAdd(a.counts + 1 + row, k) == 0) atomicAdd(a.counts, 1);
        } else
            sum += k;
    }
    if (!a.by_row) {
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0 && sum) atomicAdd(a.counts, sum);
    }
}

template <int V> __global__ void __launch_bounds__(THREADS) loss_kernel(Args a) {
    __shared__ double shared[THREADS / 32][TERMS];
    pdl_wait();
    const float flat = inverse(a.mask ? a.counts[0] : a.count), rows_inv = inverse(a.mask ? a.counts[0] : a.rows);
    double total[TERMS] = {};
    pass<V>(a, a.counts + 1, flat, rows_inv, (int64_t)blockIdx.x * THREADS + threadIdx.x, (int64_t)gridDim.x * THREADS, total);
    join<THREADS>(total, shared);
    if (threadIdx.x == 0)
        for (int k = 0; k < TERMS; k++) a.parts[(int64_t)blockIdx.x * TERMS + k] = total[k];
}

__global__ void __launch_bounds__(1024) finish_kernel(Args a) {
    __shared__ double shared[32][TERMS];
    pdl_wait();
    double total[TERMS] = {};
    for (int b = threadIdx.x; b < a.blocks; b += 1024)
        for (int k = 0; k < TERMS; k++) total[k] += a.parts[(int64_t)b * TERMS + k];
    join<1024>(total, shared);
    if (threadIdx.x == 0) finish(a, total);
}

// All of a small batch in one block.
template <int V> __global__ void __launch_bounds__(SMALL_THREADS) small_kernel(Args a) {
    __shared__ double shared[SMALL_THREADS / 32][TERMS];
    __shared__ int counts[1 + SMALL_ROWS];
    if (a.mask) {
        for (int i = threadIdx.x; i < 1 + (a.by_row ? (int)a.rows : 0); i += SMALL_THREADS) counts[i] = 0;
        __syncthreads();
        int sum = 0;
        for (int i = threadIdx.x; i < (int)a.count; i += SMALL_THREADS) {
            const int row = i / (int)a.length;
            if (a.mask[row * a.ld_mask + (i - row * (int)a.length)]) {
                if (!a.by_row)
                    sum++;
                else if (atomicAdd(counts + 1 + row, 1) == 0)
                    atomicAdd(counts, 1);
            }
        }
        if (!a.by_row) {
            sum = __reduce_add_sync(0xffffffffu, sum);
            if ((threadIdx.x & 31) == 0 && sum) atomicAdd(counts, sum);
        }
        __syncthreads();
    }
    const float flat = inverse(a.mask ? counts[0] : a.count), rows_inv = inverse(a.mask ? counts[0] : a.rows);
    double total[TERMS] = {};
    pass<V>(a, counts + 1, flat, rows_inv, threadIdx.x, SMALL_THREADS, total);
    join<SMALL_THREADS>(total, shared);
    if (threadIdx.x == 0) finish(a, total);
}

static bool is_small(int64_t rows, int64_t count) { return count <= SMALL && rows <= SMALL_ROWS; }
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
    return d1::pl::PART_BYTES + 4 * (1 + rows);
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
    a.rows = rows, a.length = length, a.count = count;
    a.over = log1p(clip_high), a.under = clip_low < 1. ? log1p(-clip_low) : -INFINITY;
    a.most = (float)(1. + clip_high), a.least = (float)(1. - clip_low);
    a.kl = (float)kl_coef, a.ent = (float)ent_coef, a.by_row = by_row != 0;
    a.loss = loss, a.stats = stats, a.dlogp = dlogp, a.dentropy = dentropy;
    a.parts = (double *)work;
    a.counts = work ? (int *)((char *)work + PART_BYTES) : nullptr;
    const cudaStream_t s = (cudaStream_t)stream;
    const auto flat = [&](const void *p, int64_t ld, int align) { return !p || (ld == length || rows == 1) && aligned_to(align, p); };
    const bool four = count % 4 == 0 && flat(logp, ld_logp, 16) && flat(old_logp, ld_old, 16) &&
                      (per_row || flat(advantage, ld_advantage, 16)) && flat(ref_logp, ld_ref, 16) &&
                      flat(entropy, ld_entropy, 16) && flat(mask, ld_mask, 4) && aligned_to(16, dlogp, dentropy);
    if (is_small(rows, count)) {
        if (four)
            small_kernel<4><<<1, SMALL_THREADS, 0, s>>>(a);
        else
            small_kernel<1><<<1, SMALL_THREADS, 0, s>>>(a);
        return (int)cudaGetLastError();
    }
    const int64_t want = (count + THREADS * 4 - 1) / (THREADS * 4);
    a.blocks = (int)(want < BLOCKS ? want : BLOCKS);
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = pdl_config(dim3(a.blocks), dim3(THREADS), 0, s, &attr);
    if (mask) {
        if (cudaError_t e = cudaMemsetAsync(a.counts, 0, (size_t)(4 * (by_row ? 1 + rows : 1)), s)) return (int)e;
        const int64_t pieces = rows * ((length + 1023) / 1024), blocks = (pieces + 7) / 8;
        count_kernel<<<(unsigned)(blocks < SMS * 8 ? blocks : SMS * 8), THREADS, 0, s>>>(a);
        if (cudaError_t e = cudaGetLastError()) return (int)e;
    } else
        cfg.numAttrs = 0;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, four ? loss_kernel<4> : loss_kernel<1>, a)) return (int)e;
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(1024);
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, finish_kernel, a);
}
