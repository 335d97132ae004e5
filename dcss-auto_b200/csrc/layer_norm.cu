// Layer norm over the last dimension, forward and backward (sm_100a).
//
//   mean = sum(x) / n          rstd = 1 / sqrt(sum((x - mean)^2) / n + eps)
//   xhat = (x - mean) rstd     y = xhat w + b
//   g = dy w                   dx = rstd (g - mean_j(g) - xhat mean_j(g xhat))
//   dw_j = sum_r dy xhat       db_j = sum_r dy
#include "d1_elem.cuh"

namespace d1 {
namespace ln {

constexpr int THREADS = 256;

__device__ __forceinline__ float block_sum(float x, float *part) {
    x = warp_sum(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; i++) s += part[i];
    return s;
}

template <class T>
__global__ void __launch_bounds__(THREADS)
    forward_kernel(const T *__restrict__ x, int64_t ldx, int64_t rows, int n, const float *__restrict__ w,
                   const float *__restrict__ b, float eps, T *__restrict__ y, int64_t ldy, float *__restrict__ mean,
                   float *__restrict__ rstd) {
    __shared__ float part[THREADS / 32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + r * ldx;
        float s = 0.f;
        for (int j = threadIdx.x; j < n; j += THREADS) s += to_f32(xr[j]);
        const float mu = block_sum(s, part) / n;
        s = 0.f;
        for (int j = threadIdx.x; j < n; j += THREADS) {
            const float c = to_f32(xr[j]) - mu;
            s += c * c;
        }
        const float rs = 1.f / sqrtf(block_sum(s, part) / n + eps);
        for (int j = threadIdx.x; j < n; j += THREADS)
            y[r * ldy + j] = from_f32<T>((to_f32(xr[j]) - mu) * rs * (w ? w[j] : 1.f) + (b ? b[j] : 0.f));
        if (threadIdx.x == 0) {
            if (mean) mean[r] = mu;
            if (rstd) rstd[r] = rs;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(THREADS)
    backward_rows_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, int64_t rows,
                         int n, const float *__restrict__ w, const float *__restrict__ mean,
                         const float *__restrict__ rstd, T *__restrict__ dx, int64_t lddx) {
    __shared__ float part[THREADS / 32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float mu = mean[r], rs = rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int j = threadIdx.x; j < n; j += THREADS) {
            const float g = to_f32(dy[r * lddy + j]) * (w ? w[j] : 1.f);
            s1 += g;
            s2 += g * ((to_f32(x[r * ldx + j]) - mu) * rs);
        }
        s1 = block_sum(s1, part) / n;
        s2 = block_sum(s2, part) / n;
        for (int j = threadIdx.x; j < n; j += THREADS) {
            const float g = to_f32(dy[r * lddy + j]) * (w ? w[j] : 1.f);
            const float xhat = (to_f32(x[r * ldx + j]) - mu) * rs;
            dx[r * lddx + j] = from_f32<T>(rs * (g - s1 - xhat * s2));
        }
    }
}

// Column sums over the rows of one part: a thread owns a column.
template <class T>
__global__ void __launch_bounds__(THREADS)
    backward_columns_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, int64_t rows,
                            int n, const float *__restrict__ mean, const float *__restrict__ rstd,
                            float *__restrict__ work) {
    const int j = blockIdx.x * THREADS + threadIdx.x;
    if (j >= n) return;
    const int64_t lo = rows * blockIdx.y / gridDim.y, hi = rows * (blockIdx.y + 1) / gridDim.y;
    float sw = 0.f, sb = 0.f;
    for (int64_t r = lo; r < hi; r++) {
        const float d = to_f32(dy[r * lddy + j]);
        sw += d * ((to_f32(x[r * ldx + j]) - mean[r]) * rstd[r]);
        sb += d;
    }
    work[(int64_t)blockIdx.y * 2 * n + j] = sw;
    work[(int64_t)blockIdx.y * 2 * n + n + j] = sb;
}

__global__ void __launch_bounds__(THREADS)
    reduce_kernel(const float *__restrict__ work, int parts, int n, float *__restrict__ dw, float *__restrict__ db) {
    const int j = blockIdx.x * THREADS + threadIdx.x;
    if (j >= 2 * n) return;
    float s = 0.f;
    for (int p = 0; p < parts; p++) s += work[(int64_t)p * 2 * n + j];
    if (j < n) {
        if (dw) dw[j] = s;
    } else if (db)
        db[j - n] = s;
}

static int parts_of(int64_t rows, int n) {
    (void)n;
    return (int)(rows < 1 ? 1 : rows < 148 ? rows : 148);
}

template <class T>
static int forward(const void *x, int64_t ldx, int64_t rows, int n, const float *w, const float *b, float eps, void *y,
                   int64_t ldy, float *mean, float *rstd, cudaStream_t s) {
    const int grid = (int)(rows < 148 * 8 ? rows : 148 * 8);
    forward_kernel<T><<<grid, THREADS, 0, s>>>((const T *)x, ldx, rows, n, w, b, eps, (T *)y, ldy, mean, rstd);
    return (int)cudaGetLastError();
}

template <class T>
static int backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, int64_t rows, int n, const float *w,
                    const float *mean, const float *rstd, void *dx, int64_t lddx, float *dw, float *db, float *work,
                    cudaStream_t s) {
    const int grid = (int)(rows < 148 * 8 ? rows : 148 * 8), parts = parts_of(rows, n);
    if (dx && rows) {
        backward_rows_kernel<T><<<grid, THREADS, 0, s>>>((const T *)dy, lddy, (const T *)x, ldx, rows, n, w, mean,
                                                         rstd, (T *)dx, lddx);
        if (cudaError_t e = cudaGetLastError()) return (int)e;
    }
    if (dw || db) {
        const dim3 cols((n + THREADS - 1) / THREADS, parts);
        backward_columns_kernel<T><<<cols, THREADS, 0, s>>>((const T *)dy, lddy, (const T *)x, ldx, rows, n, mean,
                                                            rstd, work);
        if (cudaError_t e = cudaGetLastError()) return (int)e;
        reduce_kernel<<<(2 * n + THREADS - 1) / THREADS, THREADS, 0, s>>>(work, parts, n, dw, db);
    }
    return (int)cudaGetLastError();
}

}  // namespace ln
}  // namespace d1

extern "C" int d1_layer_norm(const void *x, int64_t ldx, int type, int64_t rows, int n, const float *weight,
                             const float *bias, float eps, void *y, int64_t ldy, float *mean, float *rstd,
                             void *stream) {
    using namespace d1::ln;
    if (!d1::type_ok(type) || rows < 0 || n < 1 || !x || !y || !(eps >= 0.f) || ldx < 0 || ldy < 0 ||
        (rows > 1 && ldy < n))
        return D1_ERR_BAD_ARGUMENT;
    if (rows == 0) return 0;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == D1_TYPE_F32) return forward<float>(x, ldx, rows, n, weight, bias, eps, y, ldy, mean, rstd, s);
    if (type == D1_TYPE_BF16) return forward<__nv_bfloat16>(x, ldx, rows, n, weight, bias, eps, y, ldy, mean, rstd, s);
    return forward<__half>(x, ldx, rows, n, weight, bias, eps, y, ldy, mean, rstd, s);
}

extern "C" int d1_layer_norm_parts(int64_t rows, int n) {
    if (rows < 0 || n < 1) return D1_ERR_BAD_ARGUMENT;
    return d1::ln::parts_of(rows, n);
}

extern "C" int d1_layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, int type, int64_t rows,
                                      int n, const float *weight, const float *mean, const float *rstd, void *dx,
                                      int64_t lddx, float *dweight, float *dbias, float *work, void *stream) {
    using namespace d1::ln;
    if (!d1::type_ok(type) || rows < 0 || n < 1 || (rows && (!dy || !x || !mean || !rstd)) || lddy < 0 || ldx < 0 ||
        lddx < 0 || (dx && rows > 1 && lddx < n) || ((dweight || dbias) && !work))
        return D1_ERR_BAD_ARGUMENT;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == D1_TYPE_F32)
        return backward<float>(dy, lddy, x, ldx, rows, n, weight, mean, rstd, dx, lddx, dweight, dbias, work, s);
    if (type == D1_TYPE_BF16)
        return backward<__nv_bfloat16>(dy, lddy, x, ldx, rows, n, weight, mean, rstd, dx, lddx, dweight, dbias, work, s);
    return backward<__half>(dy, lddy, x, ldx, rows, n, weight, mean, rstd, dx, lddx, dweight, dbias, work, s);
}
