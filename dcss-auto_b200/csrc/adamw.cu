// One AdamW step over many parameter tensors in one launch (two with clipping),
// moments held in 32 or in 8 bits (sm_100a).
//
//   g' = g min(1, max_norm / (||g|| + 1e-6))             (all tensors' norm)
//   m' = b1 m + (1 - b1) g'       v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr decay) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// The tensors are laid end to end in blocks of 128 elements (the last block of
// a tensor is padded), and the moments are flat arrays over those blocks. A
// warp takes one block at a time, four elements a lane, so that every load of
// an aligned tensor is one vector per lane.
//
// 8-bit moments. A block of m is 128 e4m3 codes and a power-of-two scale that
// brings the largest |m| to [2^7, 2^8); a block of v is 128 e5m2 codes with the
// largest v at [2^14, 2^15); neither rounding up at the top nor a power of two
// loses bits, so a decoded code is exact. With b2 = 0.999 a step moves v by a
// thousandth of its distance to g^2, far below the spacing of any 8-bit code:
// rounded to nearest, v would never move again. So codes are rounded up with
// the probability of the distance to the code below (unbiased in m and in v),
// from 16 random bits per element that are a function of (seed, step, element)
// alone: a step is reproducible. v > 0 never becomes the code zero (m / eps
// would explode); it stays at the smallest code. A block that meets an infinity
// or a NaN gets a NaN scale.
#include "d1_common.cuh"
#include "d1_elem.cuh"

namespace d1 {
namespace adamw {

constexpr int BLOCK = 128, THREADS = 256, WARPS = THREADS / 32, GRID = 148 * 4;

struct Args {
    const D1AdamWTensor *tensors;
    int ntensors;
    int64_t nblocks;
    void *m, *v;
    float *m_scale, *v_scale;
    double lr, beta1, beta2, log2_beta1, log2_beta2;
    float b1, c1, b2, c2, eps, max_norm;
    int64_t *step;
    uint64_t seed;
    double *partials;       // GRID sums of squares, then the arrival count
    unsigned *arrived;
    float *grad_norm;
};

// The tensor that holds block `b`: the last one that starts at or before it.
__device__ __forceinline__ int tensor_of(const Args &a, int64_t b) {
    int lo = 0, hi = a.ntensors - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.tensors[mid].first_block <= b)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// Four elements of a tensor from element i (those beyond `count` are zero), as
// one vector where the base is aligned.
template <class T> __device__ __forceinline__ void load4(const T *p, int64_t i, int64_t count, bool wide, float (&x)[4]) {
    if (wide && i + 4 <= count) {
        const Elems<T, 4> e = *reinterpret_cast<const Elems<T, 4> *>(p + i);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = to_f32(e.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = i + k < count ? to_f32(p[i + k]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store4(T *p, int64_t i, int64_t count, bool wide, const float (&x)[4]) {
    if (wide && i + 4 <= count) {
        Elems<T, 4> e;
#pragma unroll
        for (int k = 0; k < 4; k++) e.v[k] = from_f32<T>(x[k]);
        *reinterpret_cast<Elems<T, 4> *>(p + i) = e;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (i + k < count) p[i + k] = from_f32<T>(x[k]);
    }
}
template <class T> __device__ __forceinline__ bool aligned4(const T *p) {
    return (reinterpret_cast<uintptr_t>(p) & (sizeof(T) * 4 - 1)) == 0;
}

__device__ __forceinline__ void load_grad(const D1AdamWTensor &t, int64_t i, float (&g)[4]) {
    if (t.grad_type == D1_TYPE_F32)
        load4((const float *)t.grad, i, t.count, aligned4((const float *)t.grad), g);
    else
        load4((const __nv_bfloat16 *)t.grad, i, t.count, aligned4((const __nv_bfloat16 *)t.grad), g);
}

__global__ void __launch_bounds__(THREADS) norm_kernel(Args a) {
    __shared__ double part[WARPS];
    float s = 0.f;
    for (int64_t b = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); b < a.nblocks; b += (int64_t)gridDim.x * WARPS) {
        const D1AdamWTensor &t = a.tensors[tensor_of(a, b)];
        float g[4];
        load_grad(t, (b - t.first_block) * BLOCK + 4 * (threadIdx.x & 31), g);
        s += (g[0] * g[0] + g[1] * g[1]) + (g[2] * g[2] + g[3] * g[3]);
    }
    double d = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = d;
    __syncthreads();
    if (threadIdx.x == 0) {
        d = 0.;
        for (int i = 0; i < WARPS; i++) d += part[i];
        a.partials[blockIdx.x] = d;
    }
}

// 2^e for -149 <= e <= 127.
__device__ __forceinline__ float pow2(int e) { return e >= -126 ? __int_as_float((e + 127) << 23) : __int_as_float(1 << (e + 149)); }

// The block's exponent for a largest magnitude `top` (its bits), never below
// -100; the scale then is 2^(exponent - field).
__device__ __forceinline__ int block_exponent(uint32_t top) { return imax((int)(top >> 23) - 127, -100); }

__device__ __forceinline__ uint32_t warp_max(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }

template <int BITS> __global__ void __launch_bounds__(THREADS) step_kernel(Args a, int norm_parts) {
    __shared__ double part[WARPS];
    __shared__ float coef[3];
    __shared__ int64_t now;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float clip = 1.f;
    if (a.max_norm > 0.f) {
        double d = 0.;
        for (int i = threadIdx.x; i < norm_parts; i += THREADS) d += a.partials[i];
#pragma unroll
        for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        if (lane == 0) part[warp] = d;
    }
    if (threadIdx.x == 0) {
        const int64_t t = *a.step + 1;
        now = t;
        coef[0] = (float)(a.lr / (1. - exp2((double)t * a.log2_beta1)));
        coef[1] = (float)sqrt(1. - exp2((double)t * a.log2_beta2));
    }
    __syncthreads();
    if (a.max_norm > 0.f) {
        double d = 0.;
        for (int i = 0; i < WARPS; i++) d += part[i];
        const float norm = (float)sqrt(d);
        clip = fminf(1.f, __fdiv_rn(a.max_norm, norm + 1e-6f));
        if (norm != norm) clip = norm;
        if (blockIdx.x == 0 && threadIdx.x == 0 && a.grad_norm) *a.grad_norm = norm;
    }
    const float rate = coef[0], bc2 = coef[1];
    const uint64_t key = mix64(mix64(a.seed) + (uint64_t)now);
    // the step was read before each block's arrival: the last one advances it
    if (threadIdx.x == 0) __threadfence();
    if (threadIdx.x == 0 && atomicAdd(a.arrived, 1u) == gridDim.x - 1) {
        *a.arrived = 0u;
        *a.step = now;
    }
    for (int64_t b = (int64_t)blockIdx.x * WARPS + warp; b < a.nblocks; b += (int64_t)gridDim.x * WARPS) {
        const D1AdamWTensor t = a.tensors[tensor_of(a, b)];
        const int64_t i = (b - t.first_block) * BLOCK + 4 * lane, at = b * BLOCK + 4 * lane;
        const bool wide = aligned4(t.param);
        const float keep = (float)(1. - a.lr * t.decay);
        float g[4], p[4], m[4], v[4];
        load_grad(t, i, g);
        load4(t.param, i, t.count, wide, p);
        if (BITS == 32) {
            load4((const float *)a.m, at, at + 4, true, m);
            load4((const float *)a.v, at, at + 4, true, v);
        } else {
            const uint32_t mc = ((const uint32_t *)a.m)[at >> 2], vc = ((const uint32_t *)a.v)[at >> 2];
            const float ms = a.m_scale[b], vs = a.v_scale[b];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t cm = mc >> (8 * k), cv = vc >> (8 * k);
                // the code's bits at an fp32 number's exponent, then the difference of the biases
                m[k] = __uint_as_float((cm & 0x80u) << 24 | (cm & 0x7fu) << 20) * pow2(120) * ms;
                v[k] = __uint_as_float((cv & 0x7fu) << 21) * pow2(112) * vs;
            }
        }
        uint32_t mtop = 0u, vtop = 0u;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float gk = __fmul_rn(g[k], clip);
            m[k] = __fadd_rn(__fmul_rn(m[k], a.b1), __fmul_rn(gk, a.c1));
            v[k] = __fadd_rn(__fmul_rn(v[k], a.b2), __fmul_rn(__fmul_rn(gk, gk), a.c2));
            p[k] = p[k] * keep - rate * (m[k] / (sqrtf(v[k]) / bc2 + a.eps));
            mtop = max(mtop, __float_as_uint(m[k]) & 0x7fffffffu);
            vtop = max(vtop, __float_as_uint(v[k]) & 0x7fffffffu);
        }
        store4(t.param, i, t.count, wide, p);
        if (t.copy) store4((__nv_bfloat16 *)t.copy, i, t.count, aligned4((__nv_bfloat16 *)t.copy), p);
        if (BITS == 32) {
            store4((float *)a.m, at, at + 4, true, m);
            store4((float *)a.v, at, at + 4, true, v);
        } else {
            mtop = warp_max(mtop);
            vtop = warp_max(vtop);
            const int em = block_exponent(mtop), ev = block_exponent(vtop);
            const uint64_t word = mix64(key + (uint64_t)(b * 32 + lane));
            uint32_t mc = 0u, vc = 0u;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t d = (uint32_t)(word >> (16 * k)) & 0xffffu;
                const float ym = __fmul_rn(__fmul_rn(fabsf(m[k]), pow2(7 - em)), pow2(-120));
                const float yv = __fmul_rn(__fmul_rn(v[k], pow2(14 - ev)), pow2(-112));
                const uint32_t cm = (__float_as_uint(ym) + (d << 4 | 8u)) >> 20 | (m[k] < 0.f ? 0x80u : 0u);
                uint32_t cv = (__float_as_uint(yv) + (d << 5 | 16u)) >> 21;
                if (v[k] > 0.f && cv == 0u) cv = 1u;
                mc |= cm << (8 * k);
                vc |= cv << (8 * k);
            }
            const bool mbad = mtop >= 0x7f800000u, vbad = vtop >= 0x7f800000u;
            ((uint32_t *)a.m)[at >> 2] = mbad ? 0u : mc;
            ((uint32_t *)a.v)[at >> 2] = vbad ? 0u : vc;
            if (lane == 0) {
                a.m_scale[b] = mbad ? __uint_as_float(0x7fc00000u) : pow2(em - 7);
                a.v_scale[b] = vbad ? __uint_as_float(0x7fc00000u) : pow2(ev - 14);
            }
        }
    }
}

}  // namespace adamw
}  // namespace d1

extern "C" int d1_adamw_work_bytes(void) { return d1::adamw::GRID * (int)sizeof(double) + 16; }

extern "C" int d1_adamw(const D1AdamWTensor *tensors, int ntensors, int64_t nblocks, int state_bits, void *m, void *v,
                        float *m_scale, float *v_scale, double lr, double beta1, double beta2, double eps,
                        double max_norm, int64_t *step, uint64_t seed, void *work, float *grad_norm, void *stream) {
    using namespace d1::adamw;
    if (!tensors || ntensors < 1 || nblocks < 1 || (state_bits != 32 && state_bits != 8) || !m || !v || !step ||
        !work || (state_bits == 8 && (!m_scale || !v_scale)) || !(beta1 >= 0. && beta1 < 1.) ||
        !(beta2 >= 0. && beta2 < 1.) || !(eps >= 0.) || (reinterpret_cast<uintptr_t>(m) & 15) ||
        (reinterpret_cast<uintptr_t>(v) & 15) || (reinterpret_cast<uintptr_t>(work) & 15))
        return D1_ERR_BAD_ARGUMENT;
    Args a{tensors, ntensors, nblocks, m, v, m_scale, v_scale, lr, beta1, beta2, log2(beta1), log2(beta2),
           (float)beta1, (float)(1. - beta1), (float)beta2, (float)(1. - beta2), (float)eps, (float)max_norm, step,
           seed, (double *)work, (unsigned *)((double *)work + GRID), grad_norm};
    const int64_t want = (nblocks + WARPS - 1) / WARPS;
    const int grid = (int)(want < GRID ? want : GRID);
    const cudaStream_t s = (cudaStream_t)stream;
    if (a.max_norm > 0.f) {
        norm_kernel<<<grid, THREADS, 0, s>>>(a);
        if (cudaError_t e = cudaGetLastError()) return (int)e;
    }
    if (state_bits == 32)
        step_kernel<32><<<grid, THREADS, 0, s>>>(a, grid);
    else
        step_kernel<8><<<grid, THREADS, 0, s>>>(a, grid);
    return (int)cudaGetLastError();
}
