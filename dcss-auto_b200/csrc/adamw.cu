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
#include <cuda_fp8.h>

#include "d1_common.cuh"
#include "d1_elem.cuh"
#include "d1_pdl.cuh"

namespace d1 {
namespace adamw {

__device__ __forceinline__ int64_t imin64(int64_t a, int64_t b) { return a < b ? a : b; }

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

// A warp's place in the tensor list (the same in every lane): a tensor's
// addresses, moved so that element i of all blocks is at index i.
struct Place {
    uintptr_t param, grad, copy;  // copy 0: none
    int64_t stop, end;            // first element past the tensor; first block past its blocks
    float keep;                   // 1 - lr decay
    int grad_shift;               // 2: fp32, 1: bf16
    bool wide;                    // every address allows vectors of four
};

// The place of block `b`: the last tensor that starts at or before it, found by
// the whole warp (32 tensors looked at in one round trip).
__device__ __forceinline__ Place locate(const Args &a, int64_t b) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = a.ntensors;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t before = __ballot_sync(FULL, at < hi && a.tensors[at < hi ? at : lo].first_block <= b);
        lo += (31 - __clz(before)) * step;
        hi = imin(lo + step, hi);
    }
    const D1AdamWTensor t = a.tensors[lo];
    const int64_t start = t.first_block * BLOCK;
    Place p;
    p.grad_shift = t.grad_type == D1_TYPE_F32 ? 2 : 1;
    p.param = reinterpret_cast<uintptr_t>(t.param) - 4 * start;
    p.grad = reinterpret_cast<uintptr_t>(t.grad) - (start << p.grad_shift);
    p.copy = t.copy ? reinterpret_cast<uintptr_t>(t.copy) - 2 * start : 0;
    p.stop = start + t.count;
    p.end = lo + 1 < a.ntensors ? a.tensors[lo + 1].first_block : a.nblocks;
    p.keep = (float)(1. - a.lr * t.decay);
    const uintptr_t odd = (reinterpret_cast<uintptr_t>(t.param) & 15) | (reinterpret_cast<uintptr_t>(t.copy) & 7) |
                          (reinterpret_cast<uintptr_t>(t.grad) & ((4 << p.grad_shift) - 1));
    p.wide = odd == 0;
    return p;
}

// Four elements from element i of a tensor; those at `left` and beyond are zero.
template <class T, bool WIDE> __device__ __forceinline__ void load4(const T *p, int left, float (&x)[4]) {
    if (WIDE) {
        const Elems<T, 4> e = *reinterpret_cast<const Elems<T, 4> *>(p);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = to_f32(e.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = k < left ? to_f32(p[k]) : 0.f;
    }
}
template <class T, bool WIDE> __device__ __forceinline__ void store4(T *p, int left, const float (&x)[4]) {
    if (WIDE) {
        Elems<T, 4> e;
#pragma unroll
        for (int k = 0; k < 4; k++) e.v[k] = from_f32<T>(x[k]);
        *reinterpret_cast<Elems<T, 4> *>(p) = e;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (k < left) p[k] = from_f32<T>(x[k]);
    }
}
template <bool WIDE> __device__ __forceinline__ void load_grad(const Place &t, int64_t i, int left, float (&g)[4]) {
    const uintptr_t at = t.grad + (i << t.grad_shift);
    if (t.grad_shift == 2)
        load4<float, WIDE>(reinterpret_cast<const float *>(at), left, g);
    else
        load4<__nv_bfloat16, WIDE>(reinterpret_cast<const __nv_bfloat16 *>(at), left, g);
}

// Blocks [lo, hi) of block `blockIdx.x`'s share; its warps take pairs of blocks
// in turn. f(place, b, two): blocks b and b + 1 whole and in vectors of one
// tensor (two), or block b alone.
template <class F> __device__ __forceinline__ void for_blocks(const Args &a, F f) {
    const int64_t lo = a.nblocks * blockIdx.x / gridDim.x, hi = a.nblocks * (blockIdx.x + 1) / gridDim.x;
    int64_t b = lo + 2 * (threadIdx.x >> 5);
    if (b >= hi) return;
    Place p = locate(a, b);
    for (; b < hi; b += 2 * WARPS) {
        if (b >= p.end) p = locate(a, b);
        if (b + 1 < hi && p.wide && (b + 2) * BLOCK <= p.stop) {
            f(p, b, true);
        } else {
            f(p, b, false);
            if (b + 1 < hi) {
                if (b + 1 >= p.end) p = locate(a, b + 1);
                f(p, b + 1, false);
            }
        }
    }
}

__global__ void __launch_bounds__(THREADS) norm_kernel(Args a) {
    __shared__ double part[WARPS];
    pdl_launch();
    const int lane = threadIdx.x & 31;
    float s = 0.f;
    for_blocks(a, [&](const Place &t, int64_t b, bool two) {
        const int64_t i = b * BLOCK + 4 * lane;
        float g[4], h[4] = {0.f, 0.f, 0.f, 0.f};
        if (two) {
            load_grad<true>(t, i, 4, g);
            load_grad<true>(t, i + BLOCK, 4, h);
        } else
            load_grad<false>(t, i, (int)imin64(t.stop - i, 4), g);
        s += (g[0] * g[0] + g[1] * g[1]) + (g[2] * g[2] + g[3] * g[3]);
        s += (h[0] * h[0] + h[1] * h[1]) + (h[2] * h[2] + h[3] * h[3]);
    });
    double d = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(FULL, d, o);
    if (lane == 0) part[threadIdx.x >> 5] = d;
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

__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float sqrt_approx(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four codes as numbers (exact: both formats are within fp16), before their scale.
template <bool E4M3> __device__ __forceinline__ void decode4(uint32_t codes, float (&x)[4]) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * h)), E4M3 ? __NV_E4M3 : __NV_E5M2);
        const float2 f = __half22float2(__half2(r));
        x[2 * h] = f.x;
        x[2 * h + 1] = f.y;
    }
}

// x times a power of two that brings the block's top to `field` of an 8-bit
// float of bias `bias`, at the exponent where an fp32 number's bits from
// position 23 - mantissa on are that float's. One product where the factor is a
// normal number, else two: both exact but for the last, subnormal rounding.
__device__ __forceinline__ void code_factors(int exponent, int field, int bias, float &first, float &second) {
    const int e = field - exponent + bias - 127;
    first = e >= -126 ? pow2(e) : pow2(field - exponent);
    second = e >= -126 ? 1.f : pow2(bias - 127);
}

struct Step {
    float clip, rate, inv_bc2, eps, b1, c1, b2, c2;
    uint64_t key;
};

// One block of 128: p and both moments, four elements a lane.
template <int BITS> struct Held {
    float p[4], g[4];
    float m32[BITS == 32 ? 4 : 1], v32[BITS == 32 ? 4 : 1];
    uint32_t mc, vc;
    float ms, vs;
};
template <int BITS, bool WIDE>
__device__ __forceinline__ void load_block(const Args &a, const Place &t, int64_t b, Held<BITS> &h) {
    const int lane = threadIdx.x & 31;
    const int64_t at = b * BLOCK + 4 * lane;
    const int left = WIDE ? 4 : (int)imin64(t.stop - at, 4);
    load4<float, WIDE>(reinterpret_cast<const float *>(t.param) + at, left, h.p);
    load_grad<WIDE>(t, at, left, h.g);
    if constexpr (BITS == 32) {
        load4<float, true>((const float *)a.m + at, 4, h.m32);
        load4<float, true>((const float *)a.v + at, 4, h.v32);
    } else {
        h.mc = ((const uint32_t *)a.m)[at >> 2];
        h.vc = ((const uint32_t *)a.v)[at >> 2];
        h.ms = a.m_scale[b];
        h.vs = a.v_scale[b];
    }
}
template <int BITS, bool WIDE>
__device__ __forceinline__ void step_block(const Args &a, const Step &s, const Place &t, int64_t b, Held<BITS> &h) {
    const int lane = threadIdx.x & 31;
    const int64_t at = b * BLOCK + 4 * lane;
    const int left = WIDE ? 4 : (int)imin64(t.stop - at, 4);
    float m[4], v[4];
    if constexpr (BITS == 32) {
#pragma unroll
        for (int k = 0; k < 4; k++) m[k] = h.m32[k], v[k] = h.v32[k];
    } else {
        decode4<true>(h.mc, m);
        decode4<false>(h.vc, v);
#pragma unroll
        for (int k = 0; k < 4; k++) m[k] *= h.ms, v[k] *= h.vs;
    }
    float mtop = 0.f, vtop = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float g = __fmul_rn(h.g[k], s.clip);
        m[k] = __fadd_rn(__fmul_rn(m[k], s.b1), __fmul_rn(g, s.c1));
        v[k] = __fadd_rn(__fmul_rn(v[k], s.b2), __fmul_rn(__fmul_rn(g, g), s.c2));
        h.p[k] = fmaf(-s.rate, __fdividef(m[k], fmaf(sqrt_approx(v[k]), s.inv_bc2, s.eps)), h.p[k] * t.keep);
        mtop = max_nan(mtop, fabsf(m[k]));
        vtop = max_nan(vtop, v[k]);
    }
    store4<float, WIDE>(reinterpret_cast<float *>(t.param) + at, left, h.p);
    if (t.copy) store4<__nv_bfloat16, WIDE>(reinterpret_cast<__nv_bfloat16 *>(t.copy) + at, left, h.p);
    if constexpr (BITS == 32) {
        store4<float, true>((float *)a.m + at, 4, m);
        store4<float, true>((float *)a.v + at, 4, v);
    } else {
        const uint32_t mbits = __reduce_max_sync(FULL, __float_as_uint(mtop));
        const uint32_t vbits = __reduce_max_sync(FULL, __float_as_uint(vtop));
        const int em = block_exponent(mbits), ev = block_exponent(vbits);
        float mf, mg, vf, vg;
        code_factors(em, 7, 7, mf, mg);
        code_factors(ev, 14, 15, vf, vg);
        const uint64_t word = mix64(s.key + (uint64_t)(b * 32 + lane));
        uint32_t mc[4], vc[4];  // the codes in the top byte
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t w = (uint32_t)(word >> (k < 2 ? 0 : 32)), d = k & 1 ? w >> 16 : w & 0xffffu;
            const float ym = __fmul_rn(__fmul_rn(fabsf(m[k]), mf), mg), yv = __fmul_rn(__fmul_rn(v[k], vf), vg);
            mc[k] = ((__float_as_uint(ym) + (d << 4 | 8u)) << 4 & 0x7f000000u) | (__float_as_uint(m[k]) & 0x80000000u);
            vc[k] = max(__float_as_uint(yv) + (d << 5 | 16u), v[k] > 0.f ? 1u << 21 : 0u) << 3;
        }
        const uint32_t mw = __byte_perm(__byte_perm(mc[0], mc[1], 0x0073), __byte_perm(mc[2], mc[3], 0x0073), 0x5410);
        const uint32_t vw = __byte_perm(__byte_perm(vc[0], vc[1], 0x0073), __byte_perm(vc[2], vc[3], 0x0073), 0x5410);
        const bool mbad = mbits >= 0x7f800000u, vbad = vbits >= 0x7f800000u;
        ((uint32_t *)a.m)[at >> 2] = mbad ? 0u : mw;
        ((uint32_t *)a.v)[at >> 2] = vbad ? 0u : vw;
        if (lane == 0) {
            a.m_scale[b] = mbad ? __uint_as_float(0x7fc00000u) : pow2(em - 7);
            a.v_scale[b] = vbad ? __uint_as_float(0x7fc00000u) : pow2(ev - 14);
        }
    }
}

template <int BITS> __global__ void __launch_bounds__(THREADS, 4) step_kernel(Args a) {
    __shared__ double part[WARPS];
    __shared__ float coef[2];
    __shared__ int64_t now;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < 2) {  // the two bias corrections, side by side
        const int64_t t = *a.step + 1;
        const double left = 1. - exp2((double)t * (lane ? a.log2_beta2 : a.log2_beta1));
        coef[lane] = lane ? (float)(1. / sqrt(left)) : (float)(a.lr / left);
        now = t;
    }
    Step s{1.f, 0.f, 0.f, a.eps, a.b1, a.c1, a.b2, a.c2, 0u};
    if (a.max_norm > 0.f) {
        pdl_wait();  // for the norm's partial sums
        double d = 0.;
        for (int i = threadIdx.x; i < gridDim.x; i += THREADS) d += a.partials[i];
#pragma unroll
        for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(FULL, d, o);
        if (lane == 0) part[warp] = d;
        __syncthreads();
        d = 0.;
        for (int i = 0; i < WARPS; i++) d += part[i];
        const float norm = (float)sqrt(d);
        s.clip = norm == norm ? fminf(1.f, __fdiv_rn(a.max_norm, norm + 1e-6f)) : norm;
        if (blockIdx.x == 0 && threadIdx.x == 0 && a.grad_norm) *a.grad_norm = norm;
    } else
        __syncthreads();
    s.rate = coef[0];
    s.inv_bc2 = coef[1];
    s.key = mix64(mix64(a.seed) + (uint64_t)now);
    // the step was read before each block's arrival: the last one advances it
    if (threadIdx.x == 0) {
        __threadfence();
        if (atomicAdd(a.arrived, 1u) == gridDim.x - 1) {
            *a.arrived = 0u;
            *a.step = now;
        }
    }
    for_blocks(a, [&](const Place &t, int64_t b, bool two) {
        if (two) {
            Held<BITS> h, k;
            load_block<BITS, true>(a, t, b, h);
            load_block<BITS, true>(a, t, b + 1, k);
            step_block<BITS, true>(a, s, t, b, h);
            step_block<BITS, true>(a, s, t, b + 1, k);
        } else {
            Held<BITS> h;
            load_block<BITS, false>(a, t, b, h);
            step_block<BITS, false>(a, s, t, b, h);
        }
    });
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
    const int64_t want = (nblocks + 2 * WARPS - 1) / (2 * WARPS);
    const int grid = (int)(want < GRID ? want : GRID);
    const cudaStream_t s = (cudaStream_t)stream;
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = d1::pdl_config(dim3(grid), dim3(THREADS), 0, s, &attr);
    if (a.max_norm > 0.f) {
        norm_kernel<<<grid, THREADS, 0, s>>>(a);
        if (cudaError_t e = cudaGetLastError()) return (int)e;
    } else
        cfg.numAttrs = 0;
    return (int)(state_bits == 32 ? cudaLaunchKernelEx(&cfg, step_kernel<32>, a)
                                  : cudaLaunchKernelEx(&cfg, step_kernel<8>, a));
}
