// Newton-Schulz steps of narrow matrices (a side of at most 64), part of muon.cu.
//
// Every step multiplies X by a polynomial of X X^T, so that all of them commute and the steps need no X:
//
//   A_0 = X X^T     F_k = a I + b A_k + c A_k^2     Q_{k+1} = F_k Q_k     A_{k+1} = F_k A_k F_k     result = Q X
//
// X is read twice instead of twice a step, and what lies between is 64 x 64 at most. Its price is precision: an error of A_0 is
// multiplied by a^2 = 11.9 a step where A_k should vanish, 2^-24 by 20,000 before the last of five. So A, F and Q are fp64 (the
// fp64 form of mma.sync: tcgen05 has none), Q X is fp32. And its end are five steps: A_k may be a little below 0, where F_k pulls nothing back,
// so that an error of 2^-56 of a matrix of low rank has passed 1 in 16 steps (and is NaN in 20); before that, fp32's rounding of X passes 2^-12 with
// Q, a factor of 3.4 a step. More steps go through the products of muon.cu, which take A from X each time
// (64 x 64 with six steps 80 us, in place of the 49 that it would take here, 64 x 8,192 198 in place of 60). |u| is the root of the trace of u u^T, and A_0 is divided by the trace.
//
// Up to 8 or 16 blocks of X a matrix, a cluster does all of it in one launch, and its first block takes the steps. Longer ones have one launch for
// momentum and A_0, one for the steps (a block a matrix) and one for the result. The sums of A_0 are a partial result of 18 KB of fp64 for
// each block of threads; where they are many a cluster adds them (128 are 2.4 MB, 19 us at an SM's 64 bytes a cycle), always in
// the same order.
//
// Measured (one B200, bf16, five steps; in brackets through the products of muon.cu). 1 x 8: 9 us (65). 28 x 512: 16 (80).
// 64 x 64: 41 (68). 64 x 8,192: 50 (164). 16 x 64 x 4,096: 91 (215). With a side of 64 the steps are 33 of it: 17 products of 2,900 cycles,
// 2,300 of them the fp64 rate's (64 products and sums a cycle), the rest the way through shared memory.
#pragma once

namespace narrow {

constexpr int MOST = 64, TILES = 36, WARPS = 12, THREADS_SUM = 32 * WARPS, THREADS_APPLY = 256;
constexpr int WIDTH = MOST + 4;  // fp64 of a row in shared memory: eight rows of four meet no bank twice
constexpr int PART_BYTES = 3 * BLOCK_BYTES;
constexpr int FEW = 8;  // partial sums that one block adds
constexpr int MOST_STEPS = 5;

static_assert(TILES * 64 * 8 <= PART_BYTES, "a part's sums lie in place of its blocks of X");

// Shared memory of the steps (of the whole) for a smaller side of `eights` eights.
constexpr int step_bytes(int eights) { return 5 * eights * 8 * WIDTH * 8; }
constexpr int whole_bytes(int eights) { return 6 * eights * 8 * WIDTH * 8; }

// Where a matrix's sums, Q (fp32 [64][64]) and 1 / |u| lie in the work buffer: its blocks are not used otherwise.
__device__ __forceinline__ double2 *sums_of(const Job &o, const Matrix &m, int part) {
    return reinterpret_cast<double2 *>(o.work + (int64_t)m.hi[0] * BLOCK_BYTES + (int64_t)part * PART_BYTES);
}
__device__ __forceinline__ float *q_of(const Job &o, const Matrix &m) { return reinterpret_cast<float *>(o.work + (int64_t)m.gram * BLOCK_BYTES); }
__device__ __forceinline__ double *inverse_of(const Job &o, const Matrix &m) { return reinterpret_cast<double *>(o.work + (int64_t)m.quad * BLOCK_BYTES); }

// Eights of the smaller side.
__device__ __forceinline__ int eights(const Matrix &m) { return (min(m.rows, m.cols) + 7) / 8; }

// Blocks that add a matrix's sums: two an SM in all, a part each at most (18 KB of sums a block are read again).
__device__ __forceinline__ int adders(const Job &o, const Matrix &m) { return min(m.parts, o.adders); }

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

// The tiles on and below the diagonal of a symmetric product of rows of one matrix and rows of another one: tiles warp, warp + 12,
// warp + 24. All places are 32-bit offsets into one array in shared memory, and a warp without a tile skips the product: with
// pointers of the five matrices a product was 26 instructions an mma, and took three times as long.
struct Lower {
    int count;
    int row[3], col[3];    // this lane's elements of the tiles' rows, of either operand
    int at[3], turned[3];  // its pair of the product, and the pair's first element across the diagonal (the second is a row on)
    uint32_t mirrored;     // tiles that are off the diagonal, a bit each
    uint32_t first, second;  // tiles in which its first (second) element is on the diagonal

    __device__ __forceinline__ explicit Lower(int eights) : count(0), mirrored(0), first(0), second(0) {
        const int tiles = eights * (eights + 1) / 2, lane = threadIdx.x & 31, r = lane >> 2, s = lane & 3;
#pragma unroll
        for (int q = 0; q < 3; q++) {
            const int t = (threadIdx.x >> 5) + WARPS * q;
            int i, j;
            symmetric_tile(t, i, j);
            row[q] = (8 * i + r) * WIDTH + s, col[q] = (8 * j + r) * WIDTH + s;
            at[q] = (8 * i + r) * WIDTH + 8 * j + 2 * s, turned[q] = (8 * j + 2 * s) * WIDTH + 8 * i + r;
            if (t < tiles) count = q + 1;
            if (i != j)
                mirrored |= 1u << q;
            else if (r == 2 * s)
                first |= 1u << q;
            else if (r == 2 * s + 1)
                second |= 1u << q;
        }
    }
    template <int N> __device__ __forceinline__ void add(double2 (&c)[3], const double *m, int x, int y, int fours) const {
#pragma unroll 2
        for (int k = 0; k < fours; k += 2, x += 8, y += 8) {  // (fours is even)
            double a[N][2], b[N][2];
#pragma unroll
            for (int q = 0; q < N; q++)
#pragma unroll
                for (int h = 0; h < 2; h++) a[q][h] = m[x + row[q] + 4 * h], b[q][h] = m[y + col[q] + 4 * h];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int q = 0; q < N; q++) mma64(c[q], a[q][h], b[q][h]);
        }
    }
    // work(std::integral_constant<int, N>) for the N tiles that this warp has, if any: code for N tiles is a third of that for up to
    // three, which mattered where a warp's instructions are what is waited for (1 x 8: 13.2 us with the latter)
    template <class Work> __device__ __forceinline__ void with_count(Work work) const {
        if (count == 3)
            work(std::integral_constant<int, 3>());
        else if (count == 2)
            work(std::integral_constant<int, 2>());
        else if (count == 1)
            work(std::integral_constant<int, 1>());
    }
    __device__ __forceinline__ void put(const double2 &c, double *m, int to, int q) const {
        *reinterpret_cast<double2 *>(m + to + at[q]) = c;
        if (mirrored >> q & 1u) m[to + turned[q]] = c.x, m[to + turned[q] + WIDTH] = c.y;
    }
};

// A share of u u^T (u^T u): the chunks from, from + step, ..., and the momentum brought up to date.
__device__ __forceinline__ void add_sums(const Job &o, const Matrix &m, const Lower &lower, double *u, int from, int step, double2 (&c)[3]) {
    const int chunks = max(m.rb, m.cb);
    for (int k = from; k < chunks; k += step) {
        __syncthreads();
        each_u<true, THREADS_SUM>(o, m, k, [&](int i, int l, float x) { u[i * WIDTH + l] = (double)x; });
        __syncthreads();
        lower.with_count([&](auto n) { lower.add<decltype(n)::value>(c, u, 0, 0, MOST / 4); });
    }
}

// The steps, by a block, from the sums (tile after tile, a pair a lane); Q and 1 / |u| go to the work buffer. `space`: five
// matrices of side * 8 rows, `sums` outside the first of them.
__device__ __forceinline__ void take_steps(const Job &o, const Matrix &m, const Lower &lower, int side, double *space, const double2 *sums) {
    const int size = 8 * side * WIDTH, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int a = 0, f = size, q = 2 * size, g = 3 * size, next = 4 * size;  // where they lie in `space`
    double trace = 0.;
    for (int i = lane; i < 8 * side; i += 32) {  // every warp adds the diagonal: element (r, r) of diagonal tile t
        const int t = i >> 3, r = i & 7;
        const double2 d = sums[(t * (t + 3) / 2) * 32 + 4 * r + (r >> 1)];
        trace += r & 1 ? d.y : d.x;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) trace += __shfl_xor_sync(0xffffffffu, trace, d);
    const double scale = trace == 0. ? 0. : 1. / trace;
    lower.with_count([&](auto n) {
#pragma unroll
        for (int h = 0; h < decltype(n)::value; h++) {
            double2 c = sums[(warp + WARPS * h) * 32 + lane];
            c.x *= scale, c.y *= scale;
            lower.put(c, space, a, h);
        }
    });
    if (threadIdx.x == 0) *inverse_of(o, m) = sqrt(scale);
    __syncthreads();
    float *const out = q_of(o, m);
    // the products of all steps by the same instructions: a kernel that runs once waits for most of its code to come
#pragma unroll 1
    for (int k = 0;; k++) {
#pragma unroll 1
        for (int p = k ? 0 : 1; p < 4; p++) {
            // F = polynomial of a a;  next = F q (in the first step q is F);  g = F a;  a = g F
            const bool poly = k ? p == 0 : p == 1, last = k + 1 == o.steps && p == 1;
            const int x = poly ? a : p == 3 ? g : f, y = poly ? a : p == 1 ? q : p == 2 ? a : f, to = poly ? f : p == 1 ? next : p == 2 ? g : a;
            lower.with_count([&](auto n) {
                constexpr int N = decltype(n)::value;
                double2 c[3] = {};
                lower.add<N>(c, space, x, y, 2 * side);
                if (poly)
#pragma unroll
                    for (int h = 0; h < N; h++) {
                        const double2 v = *reinterpret_cast<const double2 *>(space + a + lower.at[h]);
                        c[h].x = fma((double)NS_C, c[h].x, fma((double)NS_B, v.x, lower.first >> h & 1u ? (double)NS_A : 0.));
                        c[h].y = fma((double)NS_C, c[h].y, fma((double)NS_B, v.y, lower.second >> h & 1u ? (double)NS_A : 0.));
                    }
                if (!last) {
#pragma unroll
                    for (int h = 0; h < N; h++) lower.put(c[h], space, to, h);
                } else
#pragma unroll
                    for (int h = 0; h < N; h++) {
                        const int i = lower.at[h] / WIDTH, j = lower.at[h] % WIDTH;
                        *reinterpret_cast<float2 *>(out + i * MOST + j) = make_float2((float)c[h].x, (float)c[h].y);
                        if (lower.mirrored >> h & 1u) out[j * MOST + i] = (float)c[h].x, out[(j + 1) * MOST + i] = (float)c[h].y;
                    }
            });
            if (last) return;
            if (poly || p > 1) __syncthreads();
        }
        const int was = q;
        if (k)
            q = next, next = was;
        else  // Q_1 = F_0
            q = f, f = was;
    }
}

template <class T> __device__ __forceinline__ void store4(T *to, const float (&v)[4]) {
    Elems<T, 4> e;
#pragma unroll
    for (int c = 0; c < 4; c++) e.v[c] = from_f32<T>(v[c]);
    *reinterpret_cast<Elems<T, 4> *>(to) = e;
}

// The result Q X of the chunks from, from + step, ..., and the step with it: 4 x 4 elements a thread of the first 256. q and x:
// MOST x MOST and MOST x WIDTH in shared memory.
template <int THREADS> __device__ __forceinline__ void apply(const Job &o, const Matrix &m, float *q, float *x, int from, int step) {
    const int chunks = max(m.rb, m.cb), padded = 8 * eights(m), narrow = threadIdx.x & 15, wide = threadIdx.x >> 4;
    const int i0 = 4 * (m.tall ? narrow : wide), l0 = 4 * (m.tall ? wide : narrow);  // neighbours along a row of the matrix
    const double inverse = __ldcg(inverse_of(o, m));
    const float keep = (float)(1. - o.lr * (double)m.keep_decay), rate = (float)(-o.lr * (double)m.rate);
    const bool fours = m.cols % 4 == 0 && ((uintptr_t)m.param & 15) == 0 && ((uintptr_t)m.out & 7) == 0;
    const float4 *const q_from = reinterpret_cast<const float4 *>(q_of(o, m));
    for (int e = threadIdx.x; e < padded * (MOST / 4); e += THREADS) reinterpret_cast<float4 *>(q)[e] = __ldcg(q_from + e);
    for (int k = from; k < chunks; k += step) {
        __syncthreads();
        each_u<false, THREADS>(o, m, k, [&](int i, int l, float u) { x[i * WIDTH + l] = (float)((double)u * inverse); });
        __syncthreads();
        if (i0 >= padded || wide >= 16) continue;
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
        // four elements of a row at a time
        const int row = m.tall ? k * MOST + l0 : i0, col = m.tall ? i0 : k * MOST + l0;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (row + r >= m.rows || col >= m.cols) continue;
            float v[4];
#pragma unroll
            for (int c = 0; c < 4; c++) v[c] = m.tall ? y[c][r] : y[r][c];
            const int64_t at = (int64_t)(row + r) * m.cols + col;
            if (fours) {
                if (m.param) {
                    const float4 p = *reinterpret_cast<const float4 *>(m.param + at);
                    v[0] = fmaf(rate, v[0], p.x * keep), v[1] = fmaf(rate, v[1], p.y * keep), v[2] = fmaf(rate, v[2], p.z * keep), v[3] = fmaf(rate, v[3], p.w * keep);
                    *reinterpret_cast<float4 *>(m.param + at) = make_float4(v[0], v[1], v[2], v[3]);
                }
                if (m.out && m.out_type == D1_TYPE_BF16)
                    store4((__nv_bfloat16 *)m.out + at, v);
                else if (m.out)
                    store4((__half *)m.out + at, v);
            } else
                for (int c = 0; c < 4 && col + c < m.cols; c++) {
                    float x = c == 0 ? v[0] : c == 1 ? v[1] : c == 2 ? v[2] : v[3];
                    if (m.param) m.param[at + c] = x = fmaf(rate, x, m.param[at + c] * keep);
                    if (m.out && m.out_type == D1_TYPE_BF16)
                        ((__nv_bfloat16 *)m.out)[at + c] = __float2bfloat16_rn(x);
                    else if (m.out)
                        ((__half *)m.out)[at + c] = __float2half_rn(x);
                }
        }
    }
}

__device__ __forceinline__ void join(double2 &s, const double2 v) { s.x += v.x, s.y += v.y; }

// ---- three launches: sums by parts, steps, result by parts

__global__ void __launch_bounds__(THREADS_SUM) sums_kernel(Job o) {
    __shared__ double u[MOST * WIDTH];
    pdl_launch();
    const Part part = part_of_block(o);
    const Matrix m = matrix_of(o, part.matrix);
    if (part.k >= adders(o, m)) return;
    const Lower lower(eights(m));
    double2 c[3] = {};
    add_sums(o, m, lower, u, part.k, adders(o, m), c);
    double2 *const to = sums_of(o, m, part.k) + (threadIdx.x & 31);
#pragma unroll
    for (int q = 0; q < 3; q++)
        if (q < lower.count) to[((threadIdx.x >> 5) + WARPS * q) * 32] = c[q];
}

// A block a matrix, or a cluster whose other blocks only help to add the sums.
__global__ void __launch_bounds__(THREADS_SUM) steps_kernel(Job o) {
    extern __shared__ __align__(16) double space[];
    const int together = (int)cluster_size(), rank = (int)cluster_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch();
    pdl_wait();
    const Matrix m = matrix_of(o, blockIdx.x / together);
    const int side = eights(m), size = 8 * side * WIDTH, all = side * (side + 1) / 2 * 32, parts = adders(o, m);  // (pairs of sums)
    double2 *const sums = reinterpret_cast<double2 *>(space + 3 * size);  // the first block's
    if (together == 1) {
        for (int e = threadIdx.x; e < all; e += THREADS_SUM) {
            double2 s = {};
#pragma unroll 8
            for (int p = 0; p < parts; p++) join(s, __ldcg(sums_of(o, m, p) + e));
            sums[e] = s;
        }
        __syncthreads();
    } else {
        // this block's pairs; a warp adds every twelfth part (two warps every sixth, of half of them)
        const int from = all * rank / together, n = all * (rank + 1) / together - from, groups = together == 2 ? WARPS / 2 : WARPS;
        double2 *const share = reinterpret_cast<double2 *>(space + size);  // [groups][n]: two of the matrices' room at most
        cluster_sync();
        for (int e = lane + warp / groups * 32; e < n; e += WARPS / groups * 32) {
            double2 s = {};
#pragma unroll 8
            for (int p = warp % groups; p < parts; p += groups) join(s, __ldcg(sums_of(o, m, p) + from + e));
            share[warp % groups * n + e] = s;
        }
        __syncthreads();
        const uint32_t to = mapa(smem_u32(sums + from), 0);
        for (int e = threadIdx.x; e < n; e += THREADS_SUM) {
            double2 s = share[e];
            for (int w = 1; w < groups; w++) join(s, share[w * n + e]);
            asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(to + 16 * e), "d"(s.x), "d"(s.y) : "memory");
        }
        cluster_sync();
        if (rank) return;
    }
    take_steps(o, m, Lower(side), side, space, sums);
}

__global__ void __launch_bounds__(THREADS_APPLY) apply_kernel(Job o) {
    __shared__ __align__(16) float q[MOST * MOST], x[MOST * WIDTH];
    pdl_launch();
    pdl_wait();
    const Part part = part_of_block(o);
    const Matrix m = matrix_of(o, part.matrix);
    apply<THREADS_APPLY>(o, m, q, x, part.k, m.parts);
}

// ---- one launch for short ones: a cluster a matrix, its first block takes the steps

__global__ void __launch_bounds__(THREADS_SUM) whole_kernel(Job o) {
    extern __shared__ __align__(16) double space[];
    const int together = (int)cluster_size(), rank = (int)cluster_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Matrix m = matrix_of(o, blockIdx.x / together);
    const int side = eights(m), size = 8 * side * WIDTH, all = side * (side + 1) / 2 * 32;
    const auto meet = [&] {
        if (together > 1)
            cluster_sync();
        else
            __syncthreads();  // (of a cluster of one it took 0.7 us)
    };
    double *const u = space + 5 * size;  // then the sums of all blocks
    const Lower lower(side);
    double2 c[3] = {};
    add_sums(o, m, lower, u, rank, together, c);
    meet();  // all blocks have begun
    // the blocks' sums one after another in the first one's room for the steps
    const uint32_t to = mapa(smem_u32(space), 0) + (rank * all + lane) * 16;
#pragma unroll
    for (int q = 0; q < 3; q++)
        if (q < lower.count) asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(to + (warp + WARPS * q) * 512), "d"(c[q].x), "d"(c[q].y) : "memory");
    meet();
    if (rank == 0) {
        double2 *const sums = reinterpret_cast<double2 *>(u);
        const double2 *const shares = reinterpret_cast<const double2 *>(space);
        for (int e = threadIdx.x; e < all; e += THREADS_SUM) {
            double2 s = shares[e];
            for (int r = 1; r < together; r++) join(s, shares[r * all + e]);
            sums[e] = s;
        }
        __syncthreads();
        take_steps(o, m, lower, side, space, sums);
    }
    meet();
    float *const q = reinterpret_cast<float *>(space);
    apply<THREADS_SUM>(o, m, q, q + 8 * side * MOST, rank, together);
}

}  // namespace narrow
