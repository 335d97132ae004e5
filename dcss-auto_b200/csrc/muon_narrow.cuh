// Newton-Schulz steps of narrow matrices (a side of at most 64), part of muon.cu.
//
// Every step multiplies X by a polynomial of X X^T, so that all of them commute and the steps need no X:
//
//   A_0 = X X^T     F_k = a I + b A_k + c A_k^2     Q_{k+1} = F_k Q_k     A_{k+1} = F_k A_k F_k     result = Q X
//
// X is read twice instead of twice a step, and what lies between is 64 x 64 at most: one launch for momentum and A_0 over all of
// X, one for the steps (a block a matrix), one for the result. Its price is precision: an error of A_0 is multiplied by a^2 = 11.9
// a step where A_k should vanish. In fp32 that would leave 2e-3 of the result after five steps; A, F and Q are fp64 (the fp64
// form of mma.sync: tcgen05 has none), Q X is fp32. |u| is the root of the trace of u u^T, and A_0 is divided by the trace.
//
// The sums of A_0 are one partial result for each part of X, 18 KB of fp64 each, which a cluster of eight blocks adds up where there
// are many (one block took 17 us for 128 of them, its share of the L2's rate), in a fixed order.
#pragma once

namespace narrow {

constexpr int MOST = 64, TILES = 36, WARPS = 12, THREADS_SUM = 32 * WARPS, THREADS_APPLY = 256;
constexpr int WIDTH = MOST + 4;  // fp64 of a row in shared memory: eight rows of four meet no bank twice
constexpr int MATRIX_BYTES = MOST * WIDTH * 8, STEP_BYTES = 5 * MATRIX_BYTES, PART_BYTES = 3 * BLOCK_BYTES;
constexpr int FEW = 8, TOGETHER = 8;  // partial sums that one block adds; blocks for more

static_assert(TILES * 64 * 8 <= PART_BYTES, "a part's sums lie in place of its blocks of X");

// Where a matrix's sums, Q (fp32 [64][64]) and 1 / |u| lie in the work buffer: its blocks are not used otherwise.
__device__ __forceinline__ double2 *sums_of(const Job &o, const Matrix &m, int part) {
    return reinterpret_cast<double2 *>(o.work + (int64_t)m.hi[0] * BLOCK_BYTES + (int64_t)part * PART_BYTES);
}
__device__ __forceinline__ float *q_of(const Job &o, const Matrix &m) { return reinterpret_cast<float *>(o.work + (int64_t)m.gram * BLOCK_BYTES); }
__device__ __forceinline__ double *inverse_of(const Job &o, const Matrix &m) { return reinterpret_cast<double *>(o.work + (int64_t)m.quad * BLOCK_BYTES); }

// Eights of the smaller side.
__device__ __forceinline__ int eights(const Matrix &m) { return (min(m.rows, m.cols) + 7) / 8; }

__device__ __forceinline__ Part part_of_block(const Job &o) {
    if (o.matrices) return o.parts[blockIdx.x];
    return Part{(int)blockIdx.x / o.one.parts, (int)blockIdx.x % o.one.parts};
}

// put(i, l, u) for u at i along the smaller side (up to the next multiple of 8) and l < 64 along the larger one, from 64 * chunk on; zeros past the edges.
// UPDATE: the momentum is brought up to date first.
template <bool UPDATE, int THREADS, class Put> __device__ __forceinline__ void each_u(const Job &o, const Matrix &m, int chunk, Put put) {
    const int padded = 8 * eights(m);
    for (int e = threadIdx.x; e < MOST * 8; e += THREADS) {
        // eight elements of a row of the matrix: along the larger side, or (tall) along the smaller one, a row a lane
        const int row = m.tall ? e & 63 : e >> 3, col = (m.tall ? e >> 6 : e & 7) * 8;
        if ((m.tall ? col : row) >= padded) continue;
        const int i = m.tall ? chunk * MOST + row : row, j = m.tall ? col : chunk * MOST + col;
        const int n = i < m.rows ? min(8, max(0, m.cols - j)) : 0;
        float u[8] = {};
        if (n) momentum8<UPDATE>(o, m, i, j, n, u);
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (m.tall)
                put(col + k, row, u[k]);
            else
                put(row, col + k, u[k]);
    }
}

// One 8 x 8 tile: c += a b over four columns of a and rows of b. A lane holds a[lane / 4][lane % 4], b[lane % 4][lane / 4] and
// c[lane / 4][2 (lane % 4) + (0, 1)].
__device__ __forceinline__ void mma64(double2 &c, double a, double b) {
    asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(c.x), "+d"(c.y) : "d"(a), "d"(b));
}

// The tiles on and below the diagonal of a symmetric product of rows of `a` and rows of `b`, over 4 * fours columns: tiles
// warp, warp + 12, warp + 24.
struct Lower {
    int i[3], j[3], count;  // first row and column of a tile for this lane: its element of c, but for the column's second one

    __device__ __forceinline__ explicit Lower(int eights) : count(0) {
        const int tiles = eights * (eights + 1) / 2;
#pragma unroll
        for (int q = 0; q < 3; q++) {
            const int t = (threadIdx.x >> 5) + WARPS * q;
            symmetric_tile(t, i[q], j[q]);
            i[q] *= 8, j[q] *= 8;
            if (t < tiles) count = q + 1;
        }
    }
    __device__ __forceinline__ void add(double2 (&c)[3], const double *a, const double *b, int fours) const {
        const int lane = threadIdx.x & 31, at = (lane >> 2) * WIDTH + (lane & 3);
        const double *const pa = a + at, *const pb = b + at;
#pragma unroll 4
        for (int k = 0; k < fours; k++)
#pragma unroll
            for (int q = 0; q < 3; q++)
                if (q < count) mma64(c[q], pa[i[q] * WIDTH + 4 * k], pb[j[q] * WIDTH + 4 * k]);
    }
    // each(i, j, value) for this lane's elements of the lower tiles; those of the diagonal's are whole
    template <class Each> __device__ __forceinline__ void each(const double2 (&c)[3], Each each) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int q = 0; q < 3; q++)
            if (q < count) {
                const int r = i[q] + (lane >> 2), s = j[q] + 2 * (lane & 3);
                each(r, s, c[q].x, i[q] != j[q]);
                each(r, s + 1, c[q].y, i[q] != j[q]);
            }
    }
};

// The momentum, and a part's share of u u^T (u^T u).
__global__ void __launch_bounds__(THREADS_SUM) sums_kernel(Job o) {
    __shared__ double u[MOST * WIDTH];
    pdl_launch();
    const Part part = part_of_block(o);
    const Matrix m = matrix_of(o, part.matrix);
    const int chunks = max(m.rb, m.cb), side = eights(m);
    const Lower lower(side);
    double2 c[3] = {};
    for (int k = part.k; k < chunks; k += m.parts) {
        __syncthreads();
        each_u<true, THREADS_SUM>(o, m, k, [&](int i, int l, float x) { u[i * WIDTH + l] = (double)x; });
        __syncthreads();
        lower.add(c, u, u, MOST / 4);
    }
    double2 *const to = sums_of(o, m, part.k) + (threadIdx.x & 31);
#pragma unroll
    for (int q = 0; q < 3; q++)
        if (q < lower.count) to[((threadIdx.x >> 5) + WARPS * q) * 32] = c[q];
}

// The steps: a block a matrix, or a cluster whose other blocks only help to add the sums.
__global__ void __launch_bounds__(THREADS_SUM) steps_kernel(Job o) {
    extern __shared__ __align__(16) double space[];
    double *a = space, *f = a + MOST * WIDTH, *q = f + MOST * WIDTH, *g = q + MOST * WIDTH, *next = g + MOST * WIDTH;
    const int together = (int)cluster_size(), rank = (int)cluster_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch();
    pdl_wait();
    const Matrix m = matrix_of(o, blockIdx.x / together);
    const int side = eights(m), all = side * (side + 1) / 2 * 32;  // pairs of sums
    const auto join = [](double2 &s, const double2 v) { s.x += v.x, s.y += v.y; };
    double2 *const sums = reinterpret_cast<double2 *>(g);  // the first block's
    if (together == 1) {
        for (int e = threadIdx.x; e < all; e += THREADS_SUM) {
            double2 s = {};
#pragma unroll 8
            for (int p = 0; p < m.parts; p++) join(s, __ldcg(sums_of(o, m, p) + e));
            sums[e] = s;
        }
        __syncthreads();
    } else {
        // this block's pairs; a warp adds every twelfth part
        const int from = all * rank / together, n = all * (rank + 1) / together - from;
        double2 *const share = reinterpret_cast<double2 *>(f);  // [12][n], n <= 144
        cluster_sync();
        for (int e = lane; e < n; e += 32) {
            double2 s = {};
#pragma unroll 8
            for (int p = warp; p < m.parts; p += WARPS) join(s, __ldcg(sums_of(o, m, p) + from + e));
            share[warp * n + e] = s;
        }
        __syncthreads();
        const uint32_t to = mapa(smem_u32(sums + from), 0);
        for (int e = threadIdx.x; e < n; e += THREADS_SUM) {
            double2 s = share[e];
#pragma unroll
            for (int w = 1; w < WARPS; w++) join(s, share[w * n + e]);
            asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(to + 16 * e), "d"(s.x), "d"(s.y) : "memory");
        }
        cluster_sync();
        if (rank) return;
    }
    const Lower lower(side);
    const auto both = [](double *to, int i, int j, double v, bool mirror) {
        to[i * WIDTH + j] = v;
        if (mirror) to[j * WIDTH + i] = v;
    };
    double trace = 0.;
    for (int i = lane; i < 8 * side; i += 32) {  // every warp adds the diagonal: element (r, r) of diagonal tile t
        const int t = i >> 3, r = i & 7;
        const double2 d = sums[(t * (t + 3) / 2) * 32 + 4 * r + (r >> 1)];
        trace += r & 1 ? d.y : d.x;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) trace += __shfl_xor_sync(0xffffffffu, trace, d);
    double2 c[3];
#pragma unroll
    for (int k = 0; k < 3; k++)
        if (k < lower.count) {
            c[k] = sums[(warp + WARPS * k) * 32 + lane];
            c[k].x = trace == 0. ? 0. : c[k].x / trace, c[k].y = trace == 0. ? 0. : c[k].y / trace;
        }
    lower.each(c, [&](int i, int j, double v, bool mirror) { both(a, i, j, v, mirror); });
    if (threadIdx.x == 0) *inverse_of(o, m) = trace == 0. ? 0. : 1. / sqrt(trace);
    __syncthreads();
    const auto product = [&](const double *x, const double *y) {
#pragma unroll
        for (int k = 0; k < 3; k++) c[k] = double2{0., 0.};
        lower.add(c, x, y, 2 * side);
    };
    float *const out = q_of(o, m);
    const auto result = [&](int i, int j, double v, bool mirror) {
        out[i * MOST + j] = (float)v;
        if (mirror) out[j * MOST + i] = (float)v;
    };
    for (int k = 0;; k++) {
        const bool last = k + 1 == o.steps;
        product(a, a);
        lower.each(c, [&](int i, int j, double v, bool mirror) {
            v = fma((double)NS_C, v, fma((double)NS_B, a[i * WIDTH + j], i == j ? (double)NS_A : 0.));
            if (last && k == 0)
                result(i, j, v, mirror);
            else
                both(f, i, j, v, mirror);
        });
        if (last && k == 0) break;
        __syncthreads();
        if (k) {
            product(f, q);
            if (last) {
                lower.each(c, result);
                break;
            }
            lower.each(c, [&](int i, int j, double v, bool mirror) { both(next, i, j, v, mirror); });
        }
        product(f, a);
        lower.each(c, [&](int i, int j, double v, bool mirror) { both(g, i, j, v, mirror); });
        __syncthreads();
        product(g, f);
        lower.each(c, [&](int i, int j, double v, bool mirror) { both(a, i, j, v, mirror); });
        __syncthreads();
        double *const was = q;
        if (k)
            q = next, next = was;
        else  // Q_1 = F_0
            q = f, f = was;
    }
}

// The result Q X, and the step with it: 64 positions of the larger side at a time, 4 x 4 elements a thread.
__global__ void __launch_bounds__(THREADS_APPLY) apply_kernel(Job o) {
    __shared__ __align__(16) float q[MOST * MOST], x[MOST * WIDTH];
    pdl_launch();
    pdl_wait();
    const Part part = part_of_block(o);
    const Matrix m = matrix_of(o, part.matrix);
    const int chunks = max(m.rb, m.cb), padded = 8 * eights(m), narrow = threadIdx.x & 15, wide = threadIdx.x >> 4;
    const int i0 = 4 * (m.tall ? narrow : wide), l0 = 4 * (m.tall ? wide : narrow);  // neighbours along a row of the matrix
    const double inverse = *inverse_of(o, m);
    const float keep = (float)(1. - o.lr * (double)m.keep_decay), rate = (float)(-o.lr * (double)m.rate);
    const float4 *const from = reinterpret_cast<const float4 *>(q_of(o, m));
    for (int e = threadIdx.x; e < padded * (MOST / 4); e += THREADS_APPLY) reinterpret_cast<float4 *>(q)[e] = from[e];
    for (int k = part.k; k < chunks; k += m.parts) {
        __syncthreads();
        each_u<false, THREADS_APPLY>(o, m, k, [&](int i, int l, float u) { x[i * WIDTH + l] = (float)((double)u * inverse); });
        __syncthreads();
        if (i0 >= padded) continue;
        float y[4][4] = {};
#pragma unroll 4
        for (int s = 0; s < padded; s++) {
            const float4 f = *reinterpret_cast<const float4 *>(q + s * MOST + i0), v = *reinterpret_cast<const float4 *>(x + s * WIDTH + l0);
            const float fs[4] = {f.x, f.y, f.z, f.w}, vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int l = 0; l < 4; l++) y[r][l] = fmaf(fs[r], vs[l], y[r][l]);
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int l = 0; l < 4; l++) {
                const int i = m.tall ? k * MOST + l0 + l : i0 + r, j = m.tall ? i0 + r : k * MOST + l0 + l;
                if (i >= m.rows || j >= m.cols) continue;
                const int64_t at = (int64_t)i * m.cols + j;
                if (m.param) {
                    const float p = fmaf(rate, y[r][l], m.param[at] * keep);
                    m.param[at] = p;
                    if (m.out) ((__nv_bfloat16 *)m.out)[at] = __float2bfloat16_rn(p);
                } else if (m.out_type == D1_TYPE_BF16)
                    ((__nv_bfloat16 *)m.out)[at] = __float2bfloat16_rn(y[r][l]);
                else
                    ((__half *)m.out)[at] = __float2half_rn(y[r][l]);
            }
    }
}

}  // namespace narrow
