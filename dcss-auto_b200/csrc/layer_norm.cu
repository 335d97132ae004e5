// Layer norm over the last dimension, forward and backward (sm_100a).
//
//   mean = sum(x) / n          rstd = 1 / sqrt(sum((x - mean)^2) / n + eps)
//   xhat = (x - mean) rstd     y = xhat w + b
//   g = dy w                   dx = rstd (g - mean_j(g) - xhat mean_j(g xhat))
//   dw_j = sum_r dy xhat       db_j = sum_r dy
//
// Both passes are bound by memory. A row is read once and held in registers, P
// elements a thread, by 8 or 32 lanes (short rows, joined by shuffles) or by a
// block (joined through shared memory); the variance is the mean square of the
// held x - mean, not a difference of sums. A block keeps taking rows, and loads
// the next one before it joins the sums of this one, so that loads are in
// flight all the time. In the backward pass a thread owns the same columns in
// every row, so that the weights' gradients are sums in its registers; a block
// writes one partial sum for each column, and a second, small launch adds the
// blocks' in a fixed order.
//
// Rows are read as 16-byte vectors where base, pitch and n allow, else element
// by element (still coalesced).
#include "d1_elem.cuh"
#include "d1_pdl.cuh"

namespace d1 {
namespace ln {

constexpr int SMS = 148;
constexpr int HELD_FORWARD = 32768, HELD_BACKWARD = 8192;  // longest rows held in registers

// P elements of a row as P / VEC vectors, `threads` apart.
template <class T, int VEC, int P> struct Held {
    Elems<T, VEC> v[P / VEC];
    __device__ __forceinline__ void load(const T *row, int t, int threads, int n) {
#pragma unroll
        for (int i = 0; i < P / VEC; i++) {
            const int j = (t + i * threads) * VEC;
            if (j < n)
                v[i] = *reinterpret_cast<const Elems<T, VEC> *>(row + j);
            else
#pragma unroll
                for (int e = 0; e < VEC; e++) v[i].v[e] = from_f32<T>(0.f);
        }
    }
    __device__ __forceinline__ float at(int k) const { return to_f32(v[k / VEC].v[k % VEC]); }
};
template <class T, int VEC, int P>
__device__ __forceinline__ void store_row(T *row, int t, int threads, int n, const float (&y)[P]) {
#pragma unroll
    for (int i = 0; i < P / VEC; i++) {
        const int j = (t + i * threads) * VEC;
        if (j < n) {
            Elems<T, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; e++) o.v[e] = from_f32<T>(y[i * VEC + e]);
            *reinterpret_cast<Elems<T, VEC> *>(row + j) = o;
        }
    }
}
// The columns' weights (`other` where there are none, 0 past the row).
template <int VEC, int P>
__device__ __forceinline__ void load_weights(const float *w, int t, int threads, int n, float other, float (&x)[P]) {
#pragma unroll
    for (int k = 0; k < P; k++) {
        const int j = (t + k / VEC * threads) * VEC + k % VEC;
        x[k] = j < n ? (w ? __ldg(w + j) : other) : 0.f;
    }
}

// Sums over the G threads of a row, which all get them: by shuffles (G <= 32),
// or over the block (G = 0) through `part`, of which calls in turn take turns.
template <int G, int K> __device__ __forceinline__ void row_sums(float (&s)[K], float (*part)[32]) {
#pragma unroll
    for (int o = (G ? G : 32) / 2; o; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; k++) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
    if (G) return;
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; k++) part[k][threadIdx.x >> 5] = s[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
        s[k] = lane < warps ? part[k][lane] : 0.f;
        s[k] = warp_sum(s[k]);
    }
}

template <class T, int VEC, int P, int G>
__global__ void __launch_bounds__(G ? 256 : P == 32 ? 1024 : 512)
    forward_kernel(const T *__restrict__ x, int64_t ldx, int64_t rows, int n, const float *__restrict__ w,
                   const float *__restrict__ b, float eps, T *__restrict__ y, int64_t ldy, float *__restrict__ mean,
                   float *__restrict__ rstd) {
    constexpr bool KEEP = P <= 16;  // the weights stay in registers too
    __shared__ float part[4][1][32];
    const int threads = G ? G : blockDim.x, t = G ? threadIdx.x % G : threadIdx.x;
    const int per_block = G ? 256 / (G ? G : 1) : 1;
    const int64_t step = (int64_t)gridDim.x * per_block;
    const int64_t base = (int64_t)blockIdx.x * per_block, mine = G ? threadIdx.x / (G ? G : 1) : 0;
    float wk[KEEP ? P : 1], bk[KEEP ? P : 1];
    if (KEEP) {
        load_weights<VEC>(w, t, threads, n, 1.f, wk);
        load_weights<VEC>(b, t, threads, n, 0.f, bk);
    }
    const float inv_n = 1.f / n;
    Held<T, VEC, P> now, next;
    if (base + mine < rows) now.load(x + (base + mine) * ldx, t, threads, n);
    int turn = 0;
    for (int64_t first = base; first < rows; first += step) {  // the lanes of a warp stay together
        const int64_t r = first + mine;
        const bool live = r < rows;
        if (r + step < rows) next.load(x + (r + step) * ldx, t, threads, n);
        float s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < P; k++) s[0] += now.at(k);  // zeros past the row
        row_sums<G>(s, part[turn]);
        const float mu = s[0] * inv_n;
        s[0] = 0.f;
#pragma unroll
        for (int k = 0; k < P; k++) {
            const float c = now.at(k) - mu;
            if ((t + k / VEC * threads) * VEC < n) s[0] += c * c;
        }
        row_sums<G>(s, part[turn + 1]);
        turn ^= 2;
        const float rs = 1.f / sqrtf(s[0] * inv_n + eps);
        if (live) {
            float o[P];
            if (KEEP) {
#pragma unroll
                for (int k = 0; k < P; k++) o[k] = (now.at(k) - mu) * rs * wk[k] + bk[k];
            } else {
#pragma unroll
                for (int k = 0; k < P; k++) {
                    const int j = (t + k / VEC * threads) * VEC + k % VEC;
                    o[k] = (now.at(k) - mu) * rs;
                    if (j < n) o[k] = o[k] * (w ? __ldg(w + j) : 1.f) + (b ? __ldg(b + j) : 0.f);
                }
            }
            store_row<T, VEC, P>(y + r * ldy, t, threads, n, o);
            if (t == 0) {
                if (mean) mean[r] = mu;
                if (rstd) rstd[r] = rs;
            }
        }
        now = next;
    }
}

// dx of the rows that a block takes, and its partial sums of dw and db in work[blockIdx.x].
template <class T, int VEC, int P, int G>
__global__ void __launch_bounds__(G ? 256 : 512)
    backward_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, int64_t rows, int n,
                    const float *__restrict__ w, const float *__restrict__ mean, const float *__restrict__ rstd,
                    T *__restrict__ dx, int64_t lddx, float *__restrict__ work) {
    constexpr bool KEEP = P <= 16;
    constexpr int GROUPS = G ? 256 / (G ? G : 1) : 1;
    __shared__ float part[2][2][32];
    __shared__ float joined[G ? 256 * P : 1];
    const int threads = G ? G : blockDim.x, t = G ? threadIdx.x % G : threadIdx.x;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    const int64_t base = (int64_t)blockIdx.x * GROUPS, mine = G ? threadIdx.x / (G ? G : 1) : 0;
    float wk[KEEP ? P : 1], aw[P], ab[P];
    if (KEEP) load_weights<VEC>(w, t, threads, n, 1.f, wk);
#pragma unroll
    for (int k = 0; k < P; k++) aw[k] = ab[k] = 0.f;
    const float inv_n = 1.f / n;
    Held<T, VEC, P> xv, dv, xn, dn;
    float mu = 0.f, rs = 0.f, mun = 0.f, rsn = 0.f;
    auto fetch = [&](int64_t r, Held<T, VEC, P> &a, Held<T, VEC, P> &d, float &m, float &s) {
        a.load(x + r * ldx, t, threads, n);
        d.load(dy + r * lddy, t, threads, n);
        m = __ldg(mean + r);
        s = __ldg(rstd + r);
    };
    if (base + mine < rows) fetch(base + mine, xv, dv, mu, rs);
    int turn = 0;
    for (int64_t first = base; first < rows; first += step) {
        const int64_t r = first + mine;
        const bool live = r < rows;
        if (r + step < rows) fetch(r + step, xn, dn, mun, rsn);
        float s[2] = {0.f, 0.f};
        if (live) {
#pragma unroll
            for (int k = 0; k < P; k++) {
                const int j = (t + k / VEC * threads) * VEC + k % VEC;
                const float d = dv.at(k), xhat = (xv.at(k) - mu) * rs;
                const float g = d * (KEEP ? wk[KEEP ? k : 0] : w && j < n ? __ldg(w + j) : 1.f);  // d is zero past the row
                s[0] += g;
                s[1] += g * xhat;
                aw[k] += d * xhat;
                ab[k] += d;
            }
        }
        row_sums<G>(s, part[turn]);
        turn ^= 1;
        if (live && dx) {
            const float s1 = s[0] * inv_n, s2 = s[1] * inv_n;
            float o[P];
#pragma unroll
            for (int k = 0; k < P; k++) {
                const int j = (t + k / VEC * threads) * VEC + k % VEC;
                const float g = dv.at(k) * (KEEP ? wk[KEEP ? k : 0] : w && j < n ? __ldg(w + j) : 1.f);
                o[k] = rs * (g - s1 - (xv.at(k) - mu) * rs * s2);
            }
            store_row<T, VEC, P>(dx + r * lddx, t, threads, n, o);
        }
        xv = xn;
        dv = dn;
        mu = mun;
        rs = rsn;
    }
    if (!work) return;
    float *out = work + (int64_t)blockIdx.x * 2 * n;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        float(&a)[P] = half ? ab : aw;
        if (G) {  // the groups' sums, added in their order
            __syncthreads();
#pragma unroll
            for (int k = 0; k < P; k++) joined[threadIdx.x * P + k] = a[k];
            __syncthreads();
            if (mine == 0)
#pragma unroll
                for (int k = 0; k < P; k++) {
                    a[k] = 0.f;
                    for (int g = 0; g < GROUPS; g++) a[k] += joined[(g * threads + t) * P + k];
                }
        }
        if (mine == 0)
#pragma unroll
            for (int k = 0; k < P; k++) {
                const int j = (t + k / VEC * threads) * VEC + k % VEC;
                if (j < n) out[half * n + j] = a[k];
            }
    }
}

// dw and db from the blocks' partial sums: 32 columns a block, in 8 slices of the parts.
__global__ void __launch_bounds__(256)
    reduce_kernel(const float *__restrict__ work, int parts, int n, float *__restrict__ dw, float *__restrict__ db) {
    __shared__ float sums[8][32];
    pdl_wait();
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (j < 2 * n) {
#pragma unroll 8
        for (int p = slice; p < parts; p += 8) s += work[(int64_t)p * 2 * n + j];
    }
    sums[slice][lane] = s;
    __syncthreads();
    if (slice || j >= 2 * n) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) s += sums[i][lane];
    if (j < n) {
        if (dw) dw[j] = s;
    } else if (db)
        db[j - n] = s;
}

// ---------------------------------------------------------------- rows too long for registers

constexpr int WIDE = 1024;

template <class T>
__global__ void __launch_bounds__(WIDE)
    wide_forward_kernel(const T *__restrict__ x, int64_t ldx, int64_t rows, int n, const float *__restrict__ w,
                        const float *__restrict__ b, float eps, T *__restrict__ y, int64_t ldy,
                        float *__restrict__ mean, float *__restrict__ rstd) {
    __shared__ float part[2][1][32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + r * ldx;
        float s[1] = {0.f};
        for (int j = threadIdx.x; j < n; j += WIDE) s[0] += to_f32(xr[j]);
        row_sums<0>(s, part[0]);
        const float mu = s[0] / n;
        s[0] = 0.f;
        for (int j = threadIdx.x; j < n; j += WIDE) {
            const float c = to_f32(xr[j]) - mu;
            s[0] += c * c;
        }
        row_sums<0>(s, part[1]);
        const float rs = 1.f / sqrtf(s[0] / n + eps);
        for (int j = threadIdx.x; j < n; j += WIDE)
            y[r * ldy + j] = from_f32<T>((to_f32(xr[j]) - mu) * rs * (w ? w[j] : 1.f) + (b ? b[j] : 0.f));
        if (threadIdx.x == 0) {
            if (mean) mean[r] = mu;
            if (rstd) rstd[r] = rs;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(WIDE)
    wide_rows_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, int64_t rows, int n,
                     const float *__restrict__ w, const float *__restrict__ mean, const float *__restrict__ rstd,
                     T *__restrict__ dx, int64_t lddx) {
    __shared__ float part[2][2][32];
    int turn = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float mu = mean[r], rs = rstd[r];
        float s[2] = {0.f, 0.f};
        for (int j = threadIdx.x; j < n; j += WIDE) {
            const float g = to_f32(dy[r * lddy + j]) * (w ? w[j] : 1.f);
            s[0] += g;
            s[1] += g * ((to_f32(x[r * ldx + j]) - mu) * rs);
        }
        row_sums<0>(s, part[turn]);
        turn ^= 1;
        const float s1 = s[0] / n, s2 = s[1] / n;
        for (int j = threadIdx.x; j < n; j += WIDE) {
            const float g = to_f32(dy[r * lddy + j]) * (w ? w[j] : 1.f);
            dx[r * lddx + j] = from_f32<T>(rs * (g - s1 - (to_f32(x[r * ldx + j]) - mu) * rs * s2));
        }
    }
}

// Column sums over the rows of one part: a thread owns a column.
template <class T>
__global__ void __launch_bounds__(256)
    wide_columns_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, int64_t rows,
                        int n, const float *__restrict__ mean, const float *__restrict__ rstd,
                        float *__restrict__ work) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= n) return;
    const int64_t lo = rows * blockIdx.y / gridDim.y, hi = rows * (blockIdx.y + 1) / gridDim.y;
    float sw = 0.f, sb = 0.f;
#pragma unroll 4
    for (int64_t r = lo; r < hi; r++) {
        const float d = to_f32(dy[r * lddy + j]);
        sw += d * ((to_f32(x[r * ldx + j]) - mean[r]) * rstd[r]);
        sb += d;
    }
    work[(int64_t)blockIdx.y * 2 * n + j] = sw;
    work[(int64_t)blockIdx.y * 2 * n + n + j] = sb;
}

// ---------------------------------------------------------------- launches

// Threads of a block that holds rows of n, P elements each.
static int block_threads(int n, int p) { return ((n + p - 1) / p + 31) / 32 * 32; }

// Rows at a time and blocks of the backward pass. More blocks hide more latency
// but write more partial sums: about 768 threads an SM.
static void backward_shape(int64_t rows, int n, int *threads, int *grid) {
    int per_block = 1;
    if (n <= 64)
        *threads = 256, per_block = 32;
    else if (n <= 512)
        *threads = 256, per_block = 8;
    else
        *threads = block_threads(n, n <= 2048 ? 8 : 16);
    const int64_t want = (rows + per_block - 1) / per_block;
    const int full = SMS * (*threads >= 384 ? 2 : 768 / *threads);
    *grid = (int)(want < 1 ? 1 : want < full ? want : full);
}
static int parts_of(int64_t rows, int n) {
    if (n > HELD_BACKWARD) return (int)(rows < 1 ? 1 : rows < 16 ? rows : 16);
    int threads, grid;
    backward_shape(rows, n, &threads, &grid);
    return grid;
}

template <class T> static bool vectors_of(const void *p, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * (int64_t)sizeof(T) % 16 == 0;
}

template <class T, int VEC>
static int forward(const T *x, int64_t ldx, int64_t rows, int n, const float *w, const float *b, float eps, T *y,
                   int64_t ldy, float *mean, float *rstd, cudaStream_t s) {
#define D1_LN_FORWARD(P, G, threads, per_block, resident)                                                             \
    forward_kernel<T, VEC, P, G>                                                                                      \
        <<<(int)((rows + per_block - 1) / per_block < SMS * (resident) ? (rows + per_block - 1) / per_block           \
                                                                       : SMS * (resident)),                          \
           threads, 0, s>>>(x, ldx, rows, n, w, b, eps, y, ldy, mean, rstd)
    if (n <= 64)
        D1_LN_FORWARD(8, 8, 256, 32, 6);
    else if (n <= 256)
        D1_LN_FORWARD(8, 32, 256, 8, 6);
    else if (n <= 512)
        D1_LN_FORWARD(16, 32, 256, 8, 4);
    else if (n <= 1024)
        D1_LN_FORWARD(32, 32, 256, 8, 4);
    else if (n <= 8192) {
        const int threads = block_threads(n, 16);
        D1_LN_FORWARD(16, 0, threads, 1, 1024 / threads);
    } else {
        const int threads = block_threads(n, 32);
        D1_LN_FORWARD(32, 0, threads, 1, threads <= 512 ? 2 : 1);
    }
    return (int)cudaGetLastError();
}

template <class T>
static int forward_any(const void *x, int64_t ldx, int64_t rows, int n, const float *w, const float *b, float eps,
                       void *y, int64_t ldy, float *mean, float *rstd, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    if (n > HELD_FORWARD) {
        wide_forward_kernel<T><<<(int)(rows < SMS * 2 ? rows : SMS * 2), WIDE, 0, s>>>(
            (const T *)x, ldx, rows, n, w, b, eps, (T *)y, ldy, mean, rstd);
        return (int)cudaGetLastError();
    }
    if (n % VEC == 0 && vectors_of<T>(x, ldx) && vectors_of<T>(y, ldy))
        return forward<T, VEC>((const T *)x, ldx, rows, n, w, b, eps, (T *)y, ldy, mean, rstd, s);
    return forward<T, 1>((const T *)x, ldx, rows, n, w, b, eps, (T *)y, ldy, mean, rstd, s);
}

template <class T, int VEC>
static int backward(const T *dy, int64_t lddy, const T *x, int64_t ldx, int64_t rows, int n, const float *w,
                    const float *mean, const float *rstd, T *dx, int64_t lddx, float *work, cudaStream_t s) {
    int threads, grid;
    backward_shape(rows, n, &threads, &grid);
#define D1_LN_BACKWARD(P, G) \
    backward_kernel<T, VEC, P, G><<<grid, threads, 0, s>>>(dy, lddy, x, ldx, rows, n, w, mean, rstd, dx, lddx, work)
    if (n <= 64)
        D1_LN_BACKWARD(8, 8);
    else if (n <= 256)
        D1_LN_BACKWARD(8, 32);
    else if (n <= 512)
        D1_LN_BACKWARD(16, 32);
    else if (n <= 2048)
        D1_LN_BACKWARD(8, 0);
    else
        D1_LN_BACKWARD(16, 0);
    return (int)cudaGetLastError();
}

template <class T>
static int backward_any(const void *dy, int64_t lddy, const void *x, int64_t ldx, int64_t rows, int n, const float *w,
                        const float *mean, const float *rstd, void *dx, int64_t lddx, float *dw, float *db,
                        float *work, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    const int parts = parts_of(rows, n);
    const bool sums = dw || db;
    int e = 0;
    if (n > HELD_BACKWARD) {
        if (dx && rows)
            wide_rows_kernel<T><<<(int)(rows < SMS * 2 ? rows : SMS * 2), WIDE, 0, s>>>(
                (const T *)dy, lddy, (const T *)x, ldx, rows, n, w, mean, rstd, (T *)dx, lddx);
        if ((e = (int)cudaGetLastError())) return e;
        if (sums)
            wide_columns_kernel<T><<<dim3((n + 255) / 256, parts), 256, 0, s>>>((const T *)dy, lddy, (const T *)x, ldx,
                                                                                rows, n, mean, rstd, work);
        e = (int)cudaGetLastError();
    } else if (n % VEC == 0 && vectors_of<T>(x, ldx) && vectors_of<T>(dy, lddy) && (!dx || vectors_of<T>(dx, lddx)))
        e = backward<T, VEC>((const T *)dy, lddy, (const T *)x, ldx, rows, n, w, mean, rstd, (T *)dx, lddx,
                             sums ? work : nullptr, s);
    else
        e = backward<T, 1>((const T *)dy, lddy, (const T *)x, ldx, rows, n, w, mean, rstd, (T *)dx, lddx,
                           sums ? work : nullptr, s);
    if (e || !sums) return e;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = pdl_config(dim3((2 * n + 31) / 32), dim3(256), 0, s, &attr);
    return (int)cudaLaunchKernelEx(&cfg, reduce_kernel, (const float *)work, parts, n, dw, db);
}

}  // namespace ln
}  // namespace d1

extern "C" int d1_layer_norm(const void *x, int64_t ldx, int type, int64_t rows, int n, const float *weight,
                             const float *bias, float eps, void *y, int64_t ldy, float *mean, float *rstd,
                             void *stream) {
    using namespace d1;
    if (!type_ok(type) || rows < 0 || n < 1 || (rows && (!x || !y)) || !(eps >= 0.f) || ldx < 0 || ldy < 0 ||
        (rows > 1 && ldy < n) || !element_aligned(x, type) || !element_aligned(y, type))
        return D1_ERR_BAD_ARGUMENT;
    if (rows == 0) return 0;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == D1_TYPE_F32) return ln::forward_any<float>(x, ldx, rows, n, weight, bias, eps, y, ldy, mean, rstd, s);
    if (type == D1_TYPE_BF16)
        return ln::forward_any<__nv_bfloat16>(x, ldx, rows, n, weight, bias, eps, y, ldy, mean, rstd, s);
    return ln::forward_any<__half>(x, ldx, rows, n, weight, bias, eps, y, ldy, mean, rstd, s);
}

extern "C" int d1_layer_norm_parts(int64_t rows, int n) {
    if (rows < 0 || n < 1) return D1_ERR_BAD_ARGUMENT;
    return d1::ln::parts_of(rows, n);
}

extern "C" int d1_layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, int type, int64_t rows,
                                      int n, const float *weight, const float *mean, const float *rstd, void *dx,
                                      int64_t lddx, float *dweight, float *dbias, float *work, void *stream) {
    using namespace d1;
    if (!type_ok(type) || rows < 0 || n < 1 || (rows && (!dy || !x || !mean || !rstd)) || lddy < 0 || ldx < 0 ||
        lddx < 0 || (dx && rows > 1 && lddx < n) || ((dweight || dbias) && !work) || !element_aligned(x, type) ||
        !element_aligned(dy, type) || !element_aligned(dx, type))
        return D1_ERR_BAD_ARGUMENT;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == D1_TYPE_F32)
        return ln::backward_any<float>(dy, lddy, x, ldx, rows, n, weight, mean, rstd, dx, lddx, dweight, dbias, work, s);
    if (type == D1_TYPE_BF16)
        return ln::backward_any<__nv_bfloat16>(dy, lddy, x, ldx, rows, n, weight, mean, rstd, dx, lddx, dweight, dbias,
                                               work, s);
    return ln::backward_any<__half>(dy, lddy, x, ldx, rows, n, weight, mean, rstd, dx, lddx, dweight, dbias, work, s);
}
